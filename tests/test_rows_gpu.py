"""The operators of long conversations, each against its definition in 64 bits: norms of the
query and key heads with their rotation, K/V rows of a batch, a cache in 4 bits, and
attention under a window and first tokens that stay visible; then all of them together as a
host's own layer runs them.

EPS below is half a step of fp32, 2^-24."""
import math

import numpy as np
import pytest

from test_verify_gpu import EPS, f32, frequencies, i32, make_ctx, rope64, torch_

pytestmark = pytest.mark.gpu


def bf16(ctx, a):
    return ctx.loadWeightBf16((np.ascontiguousarray(a, np.float32).view(np.uint32) >> 16).astype(np.uint16))


def cut(a):
    """fp32 values cut to bf16, as fp32."""
    return (np.ascontiguousarray(a, np.float32).view(np.uint32) & np.uint32(0xFFFF0000)).view(np.float32)


# ---- norms of the heads with the rotation -------------------------------------------------------
def norm64(x, w, eps):
    x = x.astype(np.float64)
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w.astype(np.float64)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("hd,rd", [(64, 64), (64, 2), (64, 22), (64, 56), (128, 128), (128, 96), (128, 34), (128, 126)])
def test_norm_rope_at(dllm, layout, hd, rd):
    nq, kvh = 6, 2
    ctx = make_ctx(dllm, nq, kvh, hd)
    plan = ctx.ropePlan(layout=layout, rotary_dim=rd, theta=1e6)
    f, factor = frequencies(rd, 1e6, None)
    rng = np.random.default_rng(rd)
    qn, kn = (cut(1 + 0.3 * rng.standard_normal(hd)) for _ in range(2))
    for n in (1, 3, 37, 700):
        pos = rng.integers(0, 1 << 24, n)
        # rows of very different sizes, one of them next to eps, and a head of zeros
        size = np.float32(10.0) ** rng.integers(-4, 5, (n, 1, 1)).astype(np.float32)
        q, k = (rng.standard_normal((n, h, hd), np.float32) * size for h in (nq, kvh))
        k[0, 0] = 0
        qb, kb, pb, qw, kw = f32(ctx, q), f32(ctx, k), i32(ctx, pos), bf16(ctx, qn), bf16(ctx, kn)
        qo, ko = ctx.createF32(q.size), ctx.createF32(k.size)
        ctx.normRopeAt(plan, pb, n, qb, kb, qw, kw, qo, ko)
        outs = [ctx.readF32(b, b.n) for b in (qo, ko)]
        assert np.array_equal(ctx.readF32(qb, qb.n), q.reshape(-1))  # inputs untouched
        ctx.normRopeAt(plan, pb, n, qb, kb, qw, kw)  # in place
        inplace = [ctx.readF32(b, b.n) for b in (qb, kb)]
        for x, w, o, ip in ((q, qn, outs[0], inplace[0]), (k, kn, outs[1], inplace[1])):
            y = norm64(x, w, 1e-6)
            want, mag = rope64(y, pos, rd, layout, f, factor)
            # a sum of squares in at most 8 + 5 rounded steps, halved by the root, the mean: 8 eps; the
            # root's reciprocal 4; three rounded products 3: 15 eps of y. The rotation: 9 eps (|y1| + |y2|).
            bound = 24 * EPS * np.maximum(mag, np.abs(y))
            err = np.abs(o.reshape(x.shape) - want)
            assert (err <= bound).all(), (n, float((err / np.maximum(bound, 1e-30)).max()))
            assert np.array_equal(o, ip)
    ctx.close()


def test_norm_rope_at_one_of_q_and_k(dllm):
    ctx = make_ctx(dllm, 4, 2, 64)
    plan, rng = ctx.ropePlan(), np.random.default_rng(0)
    q, k = rng.standard_normal((5, 4, 64)).astype(np.float32), rng.standard_normal((5, 2, 64)).astype(np.float32)
    pos, w = i32(ctx, [5, 0, 2 ** 31 - 1, -7, 9]), bf16(ctx, np.ones(64))
    both = [ctx.createF32(q.size), ctx.createF32(k.size)]
    ctx.normRopeAt(plan, pos, 5, f32(ctx, q), f32(ctx, k), w, w, *both)
    qb, kb = f32(ctx, q), f32(ctx, k)
    ctx.normRopeAt(plan, pos, 5, qBuf=qb, qNorm=w)
    ctx.normRopeAt(plan, pos, 5, kBuf=kb, kNorm=w)
    for one, b in zip((qb, kb), both):
        assert np.array_equal(ctx.readF32(one, one.n), ctx.readF32(b, b.n))
    # rows behind the n given stay as they are
    qb = f32(ctx, q)
    ctx.normRopeAt(plan, pos, 3, qBuf=qb, qNorm=w)
    assert np.array_equal(ctx.readF32(qb, qb.n)[3 * 256:], q.reshape(-1)[3 * 256:])


def test_norm_rope_at_refusals(dllm):
    ctx = make_ctx(dllm, 4, 2, 64)
    plan, pos = ctx.ropePlan(), i32(ctx, [0, 1])
    q, k, w = ctx.createF32(2 * 256), ctx.createF32(2 * 128), bf16(ctx, np.ones(64))
    short, other = bf16(ctx, np.ones(63)), make_ctx(dllm, 4, 2, 64)
    for args, kw in (((plan, pos, 0, q, k, w, w), {}), ((plan, pos, 3, q, k, w, w), {}), ((plan, pos, 2, q, k, w, None), {}),
                     ((plan, pos, 2, q, None, w, w), {}), ((plan, pos, 2), {}), ((plan, pos, 2, q, k, short, w), {}),
                     ((plan, pos, 2, q, k, q, w), {}), ((plan, pos, 2, q, q, w, w), {}), ((plan, pos, 2, k, k, w, w), {}),
                     ((plan, pos, 2, q, None, w, None), {"kOut": k}), ((plan, q, 2, q, k, w, w), {}),
                     ((plan, pos, 2, q, k, w, w), {"qOut": k}), ((other.ropePlan(), pos, 2, q, k, w, w), {})):
        with pytest.raises(dllm.DllmError):
            ctx.normRopeAt(*args, **kw)


# ---- caches and their rows --------------------------------------------------------------------
def codes64(x):
    """The values that 4-bit rows stand for, by the definition, 64 bits: [..., hd] fp32 in."""
    z = np.ascontiguousarray(x, np.float32).reshape(*x.shape[:-1], x.shape[-1] // 32, 32)

    def down(a):  # to bf16: 8 significant bits, or multiples of the smallest number, 2^-133
        ex = np.maximum(np.frexp(a.astype(np.float64))[1] - 8, -133)
        return np.ldexp(np.floor(np.ldexp(a.astype(np.float64), -ex)), ex)
    low = down(z.min(-1, keepdims=True)).astype(np.float32)
    span = (z.max(-1, keepdims=True) - low).astype(np.float32)
    scale = -down(-(span.astype(np.float64) / 15).astype(np.float32))
    c = np.rint((z - low).astype(np.float64) / np.where(scale > 0, scale, 1)).clip(0, 15)
    return (low + c * scale).reshape(x.shape), np.broadcast_to(scale, z.shape).reshape(x.shape)


class Rows:
    """A paged cache ("f32", "bf16" or "4") filled through the operators under shuffled pages,
    and its values in 64 bits on the GPU, [sequence][which] -> [slots, KVH, HD]."""

    def __init__(self, dllm, nq, kvh, hd, kind, lens, counts, page=64, seqs=None, seed=0, layers=1, max_pos=None, edit=None):
        torch = torch_()
        self.lens, self.counts, self.kind, self.hd, self.nq, self.kvh = lens, counts, kind, hd, nq, kvh
        self.seqs = seqs or list(range(len(lens)))
        max_pos = max_pos or max(t + c for t, c in zip(lens, counts))
        self.ctx = make_ctx(dllm, nq, kvh, hd, kv_dtype="f32" if kind == "f32" else "bf16", kv_page_size=page,
                            max_pos=max_pos, max_seqs=max(self.seqs) + 1, num_layers=layers)
        self.cache = dllm.Cache4(self.ctx, 0, layers) if kind == "4" else dllm.Stage(self.ctx, 0, layers)
        self.layer = layers - 1
        rng = np.random.default_rng(seed)
        per = self.cache.pages_per_seq()
        table = rng.permutation((max(self.seqs) + 1) * per).reshape(-1, per)
        for s in range(max(self.seqs) + 1):
            self.cache.set_page_table(s, table[s])
        # slots behind the batch hold other data (NaN in the pages' own memory, where it can be reached)
        if kind != "4":
            for which in ("k", "v"):
                torch.as_tensor(self.cache.kv_pool(which), device="cuda").fill_(-1 if kind == "bf16" else float("nan"))
            torch.cuda.synchronize()
        self.values, bufs = [], []
        for t, c in zip(lens, counts):
            kv = [rng.standard_normal((t + c, kvh, hd)).astype(np.float32) + rng.standard_normal((kvh, hd)).astype(np.float32)
                  for _ in range(2)]
            if edit:
                edit(len(bufs), kv)
            bufs.append(kv)
            self.values.append([torch.from_numpy(self.held(x)).cuda() for x in kv])
        at = [i for i, (t, c) in enumerate(zip(lens, counts)) if t + c]
        rows = self.ctx.rowBatch([lens[i] + counts[i] for i in at], [self.seqs[i] for i in at])
        self.append(rows, *(f32(self.ctx, np.concatenate([bufs[i][w] for i in at])) for w in (0, 1)))
        for s, t in zip(self.seqs, lens):
            self.cache.set_t0(s, t)
        self.rows = self.ctx.rowBatch(counts, self.seqs)

    def held(self, x):
        if self.kind == "4":
            return codes64(x)[0]
        if self.kind == "bf16":
            return torch_().from_numpy(x).bfloat16().double().numpy()
        return x.astype(np.float64)

    def append(self, rows, k, v):
        (self.cache.append if self.kind == "4" else self.cache.append_rows)(self.layer, rows, k, v)

    def attend(self, q, window=0, sinks=0, rows=None, out=None):
        fn = self.cache.attention if self.kind == "4" else self.cache.window_attention
        return fn(self.layer, rows or self.rows, q, out, window=window, sinks=sinks)

    def close(self):
        self.cache.close()
        self.ctx.close()


def attend64(R, q, window, sinks):
    """The definition, with per row the largest visible |v| and the largest visible sum of |q_i k_i|
    in powers of two (what the error bound is made of), each [n, NQ, ...]."""
    torch = torch_()
    G, outs, vmax, amax, row = R.nq // R.kvh, [], [], [], 0
    for (k, v), t0, m in zip(R.values, R.lens, R.counts):
        if not m:
            continue
        qq = torch.from_numpy(q[row:row + m]).cuda().double()
        row += m
        slot, at = torch.arange(t0, t0 + m, device="cuda")[:, None], torch.arange(t0 + m, device="cuda")[None]
        see = at <= slot
        if window:
            see &= (at > slot - window) | (at < sinks)
        for h0 in range(0, R.kvh):
            kk, vv = torch.nan_to_num(k[:, h0]), torch.nan_to_num(v[:, h0])
            z = torch.einsum("mgd,td->mgt", qq[:, h0 * G:(h0 + 1) * G], kk) / math.sqrt(R.hd)
            p = torch.softmax(torch.where(see[:, None], z, -math.inf), -1)
            outs.append(torch.einsum("mgt,td->mgd", p, vv))
            a = torch.einsum("mgd,td->mgt", qq[:, h0 * G:(h0 + 1) * G].abs(), kk.abs())
            amax.append(torch.where(see[:, None], a, 0).amax(-1) * (math.log2(math.e) / math.sqrt(R.hd)))
            vm = torch.where(see[..., None], vv.abs()[None], 0).amax((1, 2)) if m * vv.numel() < 1e8 else vv.abs().max().expand(m)
            vmax.append(vm[:, None].expand(m, G))
    group = lambda xs: np.concatenate([np.concatenate([x.cpu().numpy() for x in xs[i:i + R.kvh]], 1)  # noqa: E731
                                       for i in range(0, len(xs), R.kvh)])
    return group(outs), group(vmax), group(amax)


def attention_bound(R, vmax, amax):
    """A score sums hd products in at most hd / 8 + 6 truncated steps of 2^-23 of the sum of
    magnitudes (operands cut to 22 bits or more count as two of the six; 4-bit rows add codes and
    minima, each at most three times the value they make up): e. Every p is off by e ln 2 and the
    exponential's 2^-21 relative, which counts twice (numerator and sum); a block's product adds up
    to 20 truncated steps of 2^-23, the blocks one rounding each, the join and the quotient a few."""
    e = (R.hd / 8 + 6) * 2.0 ** -23 * amax * (3 if R.kind == "4" else 1)
    slots = max(t + c for t, c in zip(R.lens, R.counts))
    return (vmax * (2 * (0.7 * e + 2.0 ** -21) + (28 + slots / 64) * 2.0 ** -23 * (3 if R.kind == "4" else 1)))[:, :, None]


def check_attention(R, window=0, sinks=0, seed=1, scale=1.5):
    n = sum(R.counts)
    q = np.random.default_rng(seed).standard_normal((n, R.nq, R.hd)).astype(np.float32) * np.float32(scale)
    out = R.attend(f32(R.ctx, q), window, sinks)
    got = R.ctx.readF32(out, out.n).reshape(n, R.nq, R.hd)
    want, vmax, amax = attend64(R, q, window, sinks)
    err, bound = np.abs(got - want), attention_bound(R, vmax, amax)
    assert np.isfinite(got).all()
    assert (err <= bound).all(), f"worst {float((err / bound).max())} of the bound, {float(err.max())}"
    # on average the errors are far inside the worst case; fp32 level
    assert np.linalg.norm(got - want) <= 4e-6 * np.linalg.norm(want)
    return got


KINDS = ["bf16", "f32", "4"]
HEAD_SHAPES = [(4, 2, 64), (7, 1, 64), (8, 1, 128), (6, 2, 128), (3, 3, 128)]


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("page", [32, 64, 256])
def test_cache4_rows(dllm, hd, page):
    """The values are the definition's, bit for bit, and each is within half a scale of its own."""
    rng = np.random.default_rng(hd)
    ctx = make_ctx(dllm, 6, 3, hd, max_pos=600, max_seqs=4, num_layers=2, kv_page_size=page)
    cache = dllm.Cache4(ctx, 0, 2)
    per = cache.pages_per_seq()
    table = rng.permutation(4 * per).reshape(4, per)
    for s in range(4):
        cache.set_page_table(s, table[s])
        cache.set_t0(s, [0, 59, 31, 300][s])
    assert cache.size == 2 * 2 * 4 * per * page * 3 * hd * 5 // 8
    rows = ctx.rowBatch([3, 0, 130, 1], [2, 0, 3, 1])
    n = rows.n
    kv = []
    for w in range(2):
        x = rng.standard_normal((n, 3, hd)).astype(np.float32) * np.float32(10.0) ** rng.integers(-6, 7, (n, 3, 1)).astype(np.float32)
        x[0, 0, :32] = 0  # a group of zeros, of one value, of negative values, of bf16 values, with an offset
        x[1, 0, :32] = np.float32(1 / 3)
        x[2, 0, :32] = -np.abs(x[2, 0, :32])
        x[3, 1, :32] = cut(x[3, 1, :32])
        x[4, 1] += np.float32(1000)
        x[5, 2, :32] = np.arange(32) % 16  # codes with nothing to round
        x[6, 2, :32] = np.float32(1e-41) * np.arange(32)  # subnormal
        kv.append(x)
    other = [f32(ctx, np.full((n, 3, hd), 7)) for _ in range(2)]
    cache.append(0, rows, *other)
    cache.append(1, rows, *(f32(ctx, x) for x in kv))
    for got, x in zip(cache.read_rows(1, rows), kv):
        got = ctx.readF32(got, got.n).reshape(x.shape)
        want, scale = codes64(x)
        assert np.array_equal(got, want.astype(np.float32))
        assert (np.abs(got.astype(np.float64) - x) <= scale / 2 * (1 + 2.0 ** -20) + np.abs(x) * 2.0 ** -22).all()
    for got in cache.read_rows(0, rows):
        assert (ctx.readF32(got, got.n) == 7).all()
    # one of the two only; rows behind the batch stay as they are
    only = f32(ctx, np.full((n + 2) * 3 * hd, 5))
    cache.read_rows(1, rows, vOut=only)
    got = ctx.readF32(only, only.n).reshape(n + 2, 3, hd)
    assert np.array_equal(got[:n], codes64(kv[1])[0].astype(np.float32)) and (got[n:] == 5).all()
    ctx.close()


def test_cache4_without_a_number(dllm):
    """NaN, infinities and ranges of 2^112 make NaN of their 32 values, and of no others."""
    ctx = make_ctx(dllm, 2, 1, 128, max_pos=64)
    cache, rows = dllm.Cache4(ctx, 0, 1), ctx.rowBatch([5])
    x = np.random.default_rng(0).standard_normal((5, 128)).astype(np.float32)
    for i, v in enumerate([np.nan, np.inf, -np.inf]):
        x[i, 40] = v
    x[3, 3], x[3, 4] = 3e38, -3e38
    x[4] = np.float32(2.0 ** 111) * np.sign(x[4]) * np.float32(0.5)  # a range just inside
    k = f32(ctx, x)
    cache.append(0, rows, k, k)
    got = ctx.readF32(cache.read_rows(0, rows)[0], 640).reshape(5, 4, 32)
    bad = np.zeros((5, 4), bool)
    bad[:3, 1] = bad[3, 0] = True
    assert np.isnan(got[bad]).all()
    assert np.array_equal(got[~bad], codes64(x)[0].reshape(5, 4, 32)[~bad].astype(np.float32))


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("page", [32, 128])
def test_stage_append_rows(dllm, kind, page):
    R = Rows(dllm, 4, 2, 64, kind, [100, 0, 7], [0, 33, 1], page=page, seqs=[2, 0, 1], layers=2)
    for s, want, n in zip(R.seqs, R.values, (100, 33, 8)):
        for which, w in (("k", 0), ("v", 1)):
            got = getattr(R.cache.kv[1], which).read(0, n, s)
            assert np.array_equal(got, want[w].reshape(n, -1).cpu().numpy())
    assert R.cache.t0_of(2) == 100 and R.cache.t0_of(0) == 0
    R.close()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("nq,kvh,hd", HEAD_SHAPES)
@pytest.mark.parametrize("m", [1, 2, 5, 9, 40, 130])
@pytest.mark.parametrize("t0", [0, 1, 63, 333])
def test_window_attention_small(dllm, kind, nq, kvh, hd, m, t0):
    R = Rows(dllm, nq, kvh, hd, kind, [t0], [m])
    for window, sinks in ((0, 0), (1, 0), (1, 3), (37, 0), (100, 4), (64, 64), (200, 130), (10000, 7), (0, 9)):
        check_attention(R, window, sinks)
    R.close()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("t0,m,page,window,sinks", [(4095, 1, 64, 0, 0), (5000, 3, 32, 4096, 4), (3001, 300, 128, 1000, 5),
                                                    (9999, 2, 64, 8192, 1), (2500, 513, 64, 0, 0), (0, 1025, 64, 0, 0),
                                                    (20000, 1, 64, 128, 64)])
def test_window_attention_long(dllm, kind, t0, m, page, window, sinks):
    R = Rows(dllm, 14, 2, 64 if m % 2 else 128, kind, [t0], [m], page=page)
    check_attention(R, window, sinks)
    R.close()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", [32, 64, 256])
def test_window_attention_batch(dllm, kind, page):
    """Decode steps, chunks and a sequence without rows in one batch, in another order than the
    cache's."""
    lens, counts = [700, 0, 33, 2100, 64, 5], [1, 300, 0, 1, 77, 30]
    R = Rows(dllm, 12, 2, 128, kind, lens, counts, page=page, max_pos=2300, seqs=[3, 0, 5, 1, 7, 2])
    for window, sinks in ((0, 0), (256, 4), (50, 70)):
        check_attention(R, window, sinks)
    R.close()


@pytest.mark.parametrize("kind", KINDS)
def test_window_attention_many_sequences(dllm, kind):
    lens = [(37 * i) % 900 for i in range(128)]
    R = Rows(dllm, 4, 1, 64, kind, lens, [1 + (i % 29 == 3) * 70 for i in range(128)])
    check_attention(R)
    check_attention(R, 128, 2)
    R.close()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m", [1, 4, 200])
def test_window_attention_sharp_rows(dllm, kind, m):
    """Scores in the hundreds: one slot takes almost all, and maxima move late."""
    R = Rows(dllm, 8, 2, 128, kind, [1500], [m])
    check_attention(R, scale=40.0)
    check_attention(R, 600, 3, scale=40.0)
    R.close()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m", [1, 6, 150])
@pytest.mark.parametrize("size", [2.0 ** -90, 2.0 ** 60])
def test_window_attention_small_and_large_values(dllm, kind, m, size):
    """V of any size and K of sizes that go with q: nothing is lost to a type's range. (q and K
    together make scores of ordinary size.)"""
    def edit(_, kv):
        kv[0] /= np.float32(size)
        kv[1] *= np.float32(size)
        kv[1][::3] *= np.float32(2.0 ** -20)  # and rows of very unequal sizes
    R = Rows(dllm, 6, 2, 64, kind, [300], [m], edit=edit)
    check_attention(R, 0, 0, scale=1.5 * size)
    check_attention(R, 90, 3, scale=1.5 * size)
    R.close()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m", [1, 8, 90, 300])
@pytest.mark.parametrize("value", [np.nan, np.inf])
def test_hidden_rows_do_not_leak(dllm, kind, m, value):
    """Non-finite K and V rows: those no row sees change nothing; those that some rows see make
    these rows non-finite, in the dims concerned, and no others."""
    t0, window, sinks = 200, 70, 6
    hidden, seen = (6, 9, 64, 129), ((t0 + m - 1,) if m > 1 else ())

    def edit(_, kv):
        for s in hidden:
            kv[0][s] = kv[1][s] = value
        for s in seen:
            kv[1][s, :, 5] = value
    R = Rows(dllm, 8, 2, 64, kind, [t0], [m], edit=edit)
    n = m
    q = np.random.default_rng(3).standard_normal((n, 8, 64)).astype(np.float32)
    out = R.attend(f32(R.ctx, q), window, sinks)
    got = R.ctx.readF32(out, out.n).reshape(n, 8, 64)
    want, vmax, amax = attend64(R, q, window, sinks)
    bad = np.zeros((n, 8, 64), bool)
    if seen:  # 4 bits: the whole group of 32
        bad[-1, :, 0:32 if R.kind == "4" else 6] = True
        if R.kind != "4":
            bad[-1, :, :5] = False
    assert (~np.isfinite(got[bad])).all()
    assert np.isfinite(got[~bad]).all()
    err, bound = np.abs(got - want), np.broadcast_to(attention_bound(R, vmax, amax), got.shape)
    assert (err[~bad] <= bound[~bad]).all()
    R.close()


@pytest.mark.parametrize("kind", KINDS)
def test_rows_one_by_one_and_in_chunks(dllm, kind):
    """A prompt in one chunk, in chunks of 17, and token by token sees the same; and what lies
    behind the rows of a call is not written."""
    t = 90
    R = Rows(dllm, 4, 2, 64, kind, [0], [t])
    q = np.random.default_rng(2).standard_normal((t, 256)).astype(np.float32)
    whole = R.attend(f32(R.ctx, q), 33, 2)
    whole = R.ctx.readF32(whole, whole.n).reshape(t, 256)
    for step in (17, 1):
        for a in range(0, t, step):
            e = min(t, a + step)
            R.cache.set_t0(0, a)
            buf = f32(R.ctx, np.full((e - a + 1) * 256, 9))
            R.attend(f32(R.ctx, q[a:e]), 33, 2, rows=R.ctx.rowBatch([e - a]), out=buf)
            got = R.ctx.readF32(buf, buf.n).reshape(-1, 256)
            assert (got[-1] == 9).all()
            # two results within the bound of the definition; 4e-6 of their size on average
            assert np.linalg.norm(got[:-1] - whole[a:e]) <= 8e-6 * np.linalg.norm(whole[a:e])
    R.close()


@pytest.mark.parametrize("kind", KINDS)
def test_two_runs_give_the_same_bits(dllm, kind):
    R = Rows(dllm, 12, 2, 128, kind, [3000, 40], [1, 200])
    q = f32(R.ctx, np.random.default_rng(0).standard_normal(201 * 12 * 128))
    a, b = R.attend(q), R.attend(q)
    assert np.array_equal(R.ctx.readF32(a, a.n), R.ctx.readF32(b, b.n))
    R.close()


# ---- refusals -----------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["bf16", "4"])
def test_rows_refusals(dllm, kind):
    R = Rows(dllm, 4, 2, 64, kind, [10, 5], [2, 1], max_pos=40)
    ctx, rows = R.ctx, R.rows
    for counts, seqs in (([], None), ([0, 0], None), ([-1], None), ([41], None), ([1, 1], [0, 0]), ([1], [-1]),
                         ([1] * 129, None), ([1, 1], [0])):
        with pytest.raises(dllm.DllmError):
            ctx.rowBatch(counts, seqs)
    q, k = ctx.createF32(3 * 256), ctx.createF32(3 * 128)
    fine = lambda **kw: R.attend(q, **kw)  # noqa: E731
    fine()
    for bad in (lambda: fine(window=-1), lambda: fine(sinks=-1), lambda: fine(window=2 ** 31), lambda: fine(out=q),
                lambda: R.attend(k), lambda: fine(out=k), lambda: fine(rows=ctx.rowBatch([1], [2])),
                lambda: R.append(rows, q, ctx.createF32(3 * 128 - 1)), lambda: R.append(ctx.rowBatch([1], [9]), k, k)):
        with pytest.raises(dllm.DllmError):
            bad()
    with pytest.raises(ValueError):
        R.attend(q, rows=k)
    with pytest.raises(ValueError):
        R.append(rows, k, rows)
    R.cache.set_t0(0, 39)  # no room for two rows
    for bad in (lambda: fine(), lambda: R.append(rows, k, k)):
        with pytest.raises(dllm.KvOverflowError):
            bad()
    R.cache.set_t0(0, 38)
    fine()
    fine(window=2 ** 31 - 1, sinks=2 ** 31 - 1)
    R.layer = 1
    for bad in (lambda: fine(), lambda: R.append(rows, k, k)):
        with pytest.raises(dllm.DllmError):
            bad()
    other = make_ctx(dllm, 4, 2, 64, max_pos=40)
    R.layer = 0
    with pytest.raises(dllm.DllmError):
        fine(rows=other.rowBatch([1, 1]))
    R.close()


def test_cache4_refusals(dllm):
    ctx = make_ctx(dllm, 4, 2, 64, max_pos=100, max_seqs=2)
    for a, b in ((-1, 1), (1, 0), (0, 3)):
        with pytest.raises(dllm.DllmError):
            dllm.Cache4(ctx, a, b)
    cache, rows = dllm.Cache4(ctx, 1, 2), ctx.rowBatch([2])
    k = ctx.createF32(2 * 128)
    for bad in (lambda: cache.append(0, rows, k, k), lambda: cache.read_rows(1, rows, k, k),
                lambda: cache.read_rows(1, rows, ctx.createF32(255)), lambda: cache.set_t0(2, 0), lambda: cache.set_t0(0, 101),
                lambda: cache.set_t0(0, -1), lambda: cache.set_page_table(0, [0]), lambda: cache.set_page_table(0, [0, 0]),
                lambda: cache.set_page_table(0, [0, 4]), lambda: cache.set_page_table(2, [0, 1]),
                lambda: cache.set_page_table(0, [0, 2 ** 32 + 1])):
        with pytest.raises((dllm.DllmError, IndexError)):
            bad()
    assert cache.t0_of(2) == -1 and cache.pages_per_seq() == 2
    cache.set_t0(1, 5)
    cache.reset()
    assert cache.t0_of(1) == 0
    cache.close()
    with pytest.raises(dllm.DllmError):
        cache.append(1, rows, k, k)
    assert cache.t0_of(0) == -1 and cache.size == 0


# ---- streams, graphs, and all of them together --------------------------------------------------------
@pytest.mark.parametrize("kind", KINDS)
def test_rows_on_a_side_stream_and_in_a_captured_graph(dllm, kind):
    """A decode step of a host's own layer (norm + rotation, append, attention) captured once and
    replayed with other inputs gives what the calls give."""
    torch = torch_()
    R = Rows(dllm, 8, 2, 128, kind, [500, 30], [1, 1], max_pos=600)
    ctx = R.ctx
    rng = np.random.default_rng(0)
    make = lambda w: rng.standard_normal(2 * w * 128).astype(np.float32)  # noqa: E731
    steps = [[make(8), make(2), make(2)] for _ in range(3)]
    plan, pos, w = ctx.ropePlan(), i32(ctx, [500, 30]), bf16(ctx, np.ones(128))
    q, k, v, out = ctx.createF32(2 * 1024), ctx.createF32(2 * 256), ctx.createF32(2 * 256), ctx.createF32(2 * 1024)
    qt, kt = ctx.createF32(2 * 1024), ctx.createF32(2 * 256)

    def step():
        ctx.normRopeAt(plan, pos, 2, q, k, w, w, qt, kt)
        R.append(R.rows, kt, v)
        R.attend(qt, 300, 4, out=out)
    want = []
    for s in steps:
        for b, x in zip((q, k, v), s):
            ctx.writeF32(b, x)
        step()
        want.append(ctx.readF32(out, out.n))
    ctx.synchronize()
    stream = torch.cuda.Stream()
    ctx.set_stream(stream.cuda_stream)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        step()
        for refused in (lambda: ctx.rowBatch([1]), lambda: dllm.Cache4(ctx, 0, 1), lambda: R.cache.set_page_table(0, range(R.cache.pages_per_seq()))):
            with pytest.raises(dllm.DllmError):
                refused()
    for s, x in zip(steps, want):
        for b, a in zip((q, k, v), s):
            ctx.writeF32(b, a)
        with torch.cuda.stream(stream):
            g.replay()
        assert np.array_equal(ctx.readF32(out, out.n), x)
    ctx.set_stream(None)
    del g
    R.close()


def test_a_conversation(dllm):
    """A host's own layer through a conversation: a prompt in two chunks beside another sequence's
    decode steps, then decode steps, with windows and sinks, over the cache in 4 bits and over a
    stage's: every step is the definition's on what the caches hold."""
    nq, kvh, hd, window, sinks = 6, 2, 64, 40, 3
    rng = np.random.default_rng(5)
    ctx = make_ctx(dllm, nq, kvh, hd, max_pos=256, max_seqs=2, kv_dtype="f32")
    stage, cache = dllm.Stage(ctx, 0, 1), dllm.Cache4(ctx, 0, 1)
    plan = ctx.ropePlan(rotary_dim=48)
    f, factor = frequencies(48, ctx.cfg.rope_theta, None)
    qn, kn = (cut(1 + 0.2 * rng.standard_normal(hd)) for _ in range(2))
    qw, kw = bf16(ctx, qn), bf16(ctx, kn)
    held = [[np.zeros((0, kvh, hd)) for _ in range(2)] for _ in range(2)]  # fp32 K, V of each sequence
    for counts in ([60, 0], [41, 5], [1, 1], [1, 1], [0, 1]):
        rows, n = ctx.rowBatch(counts), sum(counts)
        assert [stage.t0_of(s) for s in (0, 1)] == [len(h[0]) for h in held] == [cache.t0_of(s) for s in (0, 1)]
        pos = np.concatenate([np.arange(len(held[s][0]), len(held[s][0]) + counts[s]) for s in (0, 1)])
        q, k, v = (rng.standard_normal((n, h, hd)).astype(np.float32) for h in (nq, kvh, kvh))
        qb, kb, vb = f32(ctx, q), f32(ctx, k), f32(ctx, v)
        ctx.normRopeAt(plan, i32(ctx, pos), n, qb, kb, qw, kw)
        qt = ctx.readF32(qb, qb.n).reshape(q.shape)
        kt = ctx.readF32(kb, kb.n).reshape(k.shape)
        for x, w, got in ((q, qn, qt), (k, kn, kt)):
            y, mag = rope64(norm64(x, w, 1e-6), pos, 48, "half", f, factor)
            assert np.abs(got - y).max() <= 24 * EPS * max(mag.max(), np.abs(y).max())
        stage.append_rows(0, rows, kb, vb)
        cache.append(0, rows, kb, vb)
        at = 0
        for s in (0, 1):
            held[s] = [np.concatenate([h, x[at:at + counts[s]]]) for h, x in zip(held[s], (kt, v))]
            at += counts[s]
        for kind, out in (("f32", stage.window_attention(0, rows, qb, window=window, sinks=sinks)),
                          ("4", cache.attention(0, rows, qb, window=window, sinks=sinks))):
            R = object.__new__(Rows)
            R.kind, R.nq, R.kvh, R.hd = kind, nq, kvh, hd
            R.counts, R.lens = counts, [len(h[0]) - c for h, c in zip(held, counts)]
            R.values = [[torch_().from_numpy(Rows.held(R, x.astype(np.float32))).cuda() for x in h] for h in held]
            want, vmax, amax = attend64(R, qt, window, sinks)
            got = ctx.readF32(out, out.n).reshape(want.shape)
            assert (np.abs(got - want) <= attention_bound(R, vmax, amax)).all()
        for s in (0, 1):
            stage.set_t0(s, len(held[s][0]))
            cache.set_t0(s, len(held[s][0]))
    ctx.close()


# ---- where a rule or a limit changes hands ---------------------------------------------------------
@pytest.mark.parametrize("scale", [1.0, 1.5, 2.0 ** -100, 2.0 ** -130, 2.0 ** 100, 1.9921875])
def test_cache4_codes_next_to_a_half(dllm, scale):
    """Values at, just below and just above the middle between two codes: the code is that of the
    quotient in fp32, ties to even, whatever the scale (a product with its inverse would be off, or
    infinite for the smallest)."""
    ctx = make_ctx(dllm, 4, 2, 64, max_pos=64)
    cache, rows = dllm.Cache4(ctx, 0, 1), ctx.rowBatch([6])
    half = np.float32(scale) * (np.arange(15, dtype=np.float32) + np.float32(0.5))
    up, down = np.nextafter(half, np.float32(np.inf)), np.nextafter(half, np.float32(0))
    group = lambda x: np.concatenate([x, [0, 15 * scale], np.float32(scale) * np.arange(15)]).astype(np.float32)  # noqa: E731
    x = np.stack([group(g) for g in (half, up, down, -half + 15 * np.float32(scale))] * 6).reshape(6, 2, 64)
    z = x.reshape(6, 2, 2, 32)
    # the smallest value is 0 in each group, and fifteen scales are 15 * scale exactly
    want = (np.rint(z / np.float32(scale)).clip(0, 15) * np.float64(np.float32(scale))).astype(np.float32).reshape(x.shape)
    k, v = ctx.createF32(x.size), ctx.createF32(x.size)
    cache.append(0, rows, f32(ctx, x), f32(ctx, x[::-1]))
    cache.read_rows(0, rows, k, v)
    assert np.array_equal(ctx.readF32(k, k.n).reshape(x.shape), want)
    assert np.array_equal(ctx.readF32(v, v.n).reshape(x.shape), want[::-1])
    ctx.close()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("m", [7, 8, 9, 16, 17, 32, 33, 64, 65, 128, 129, 256, 257])
def test_window_attention_around_tile_sizes(dllm, kind, hd, m):
    R = Rows(dllm, 2, 2, hd, kind, [210], [m])
    check_attention(R)
    check_attention(R, 100, 3)
    R.close()


@pytest.mark.parametrize("kind", KINDS)
def test_window_attention_mixed_lengths(dllm, kind):
    """Short, middling and long rows in one batch, out of order and with an idle sequence between."""
    R = Rows(dllm, 10, 2, 64, kind, [700, 0, 1500, 31, 40, 64, 2000], [1, 150, 7, 0, 13, 64, 300], seqs=[5, 2, 0, 1, 6, 3, 8])
    check_attention(R)
    check_attention(R, 333, 40)
    R.close()


@pytest.mark.parametrize("kind", KINDS)
def test_long_chunks_in_graphs(dllm, kind):
    """A long chunk captured and replayed with other inputs; a longer one cannot be captured before
    its scratch is there, and the first graph keeps its own when it is."""
    torch = torch_()
    R = Rows(dllm, 6, 2, 128, kind, [100, 20], [90, 1], max_pos=4000)
    ctx, rng = R.ctx, np.random.default_rng(0)
    q, out = ctx.createF32(91 * 768), ctx.createF32(91 * 768)
    inputs = [rng.standard_normal(91 * 768).astype(np.float32) for _ in range(3)]
    want = []
    for x in inputs:
        ctx.writeF32(q, x)
        R.attend(q, 80, 2, out=out)
        want.append(ctx.readF32(out, out.n))
    many = ctx.rowBatch([3000], [0])
    big, far = ctx.createF32(3000 * 768), ctx.createF32(3000 * 768)
    ctx.synchronize()
    stream = torch.cuda.Stream()
    ctx.set_stream(stream.cuda_stream)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        R.attend(q, 80, 2, out=out)
        with pytest.raises(dllm.DllmError):
            R.attend(big, rows=many, out=far)
    replay = lambda x: (ctx.writeF32(q, x), g.replay(), ctx.readF32(out, out.n))[2]  # noqa: E731
    for round_ in range(2):
        for x, w in zip(inputs, want):
            with torch.cuda.stream(stream):
                assert np.array_equal(replay(x), w)
        if round_ == 0:  # the longer chunk, outside: more scratch, and slots behind those of the graph
            R.cache.set_t0(0, 190)
            R.append(ctx.rowBatch([2810], [0]), *(f32(ctx, np.zeros(2810 * 256)) for _ in range(2)))
            R.cache.set_t0(0, 0)
            R.attend(big, rows=many, out=far)
            ctx.synchronize()
    ctx.set_stream(None)
    del g
    R.close()


@pytest.mark.parametrize("kind", ["bf16", "4"])
@pytest.mark.parametrize("m", [1, 9, 70])
def test_rows_of_a_cache_beyond_32_bits(dllm, kind, m):
    """The last slots of the last of 9 sequences of 2^20 slots: their offsets, in elements or bytes, do
    not fit 32 bits."""
    torch = torch_()
    far, kvh, hd, seen = 1 << 20, 8, 128, 300
    ctx = make_ctx(dllm, 8, kvh, hd, max_pos=far, max_seqs=9, kv_dtype="bf16", kv_page_size=256)
    R = object.__new__(Rows)
    R.ctx, R.kind, R.nq, R.kvh, R.hd, R.layer = ctx, kind, 8, kvh, hd, 0
    R.cache = dllm.Cache4(ctx, 0, 1) if kind == "4" else dllm.Stage(ctx, 0, 1)
    rng = np.random.default_rng(m)
    kv = [rng.standard_normal((seen, kvh, hd)).astype(np.float32) for _ in range(2)]
    R.cache.set_t0(8, far - seen)
    R.append(ctx.rowBatch([seen], [8]), *(f32(ctx, x) for x in kv))
    R.cache.set_t0(8, far - m)
    R.rows, R.lens, R.counts = ctx.rowBatch([m], [8]), [seen - m], [m]
    R.values = [[torch.from_numpy(R.held(x)).cuda() for x in kv]]
    check_attention(R, window=200)  # the slots before the last 300 are outside of it
    R.close()


@pytest.mark.parametrize("kind", ["f32", "4"])
def test_scratch_of_a_growing_conversation(dllm, kind):
    """Chunk after chunk the scratch grows by doubling and the one before is given back, so that in the
    end no more than twice the last chunk's share is held."""
    torch = torch_()
    far, chunk = 6000, 200
    ctx = make_ctx(dllm, 8, 8, 128, max_pos=far, max_seqs=1, kv_dtype="f32")
    cache = dllm.Cache4(ctx, 0, 1) if kind == "4" else dllm.Stage(ctx, 0, 1)
    rows, q, out = ctx.rowBatch([chunk]), ctx.createF32(chunk * 1024), ctx.createF32(chunk * 1024)
    k = ctx.createF32(chunk * 1024)
    fn = cache.attention if kind == "4" else cache.window_attention
    append = cache.append if kind == "4" else cache.append_rows
    ctx.synchronize()
    before, held = torch.cuda.mem_get_info()[0], []
    for t in range(0, far, chunk):
        cache.set_t0(0, t)
        append(0, rows, k, k)
        fn(0, rows, q, out)
        held.append(before - torch.cuda.mem_get_info()[0])
    share = 8 * 2 * far * 128 * 4  # 4 bytes per K or V value
    assert share / 2 <= held[-1] <= 2 * share + (64 << 20), (held[-1], share)
    assert len(set(held)) <= 8
    assert (ctx.readF32(out, out.n) == 0).all()
    ctx.close()


def test_captured_scratch_outlives_a_failed_growth(dllm):
    """A chunk captured, a longer one outside, a still longer one that finds no memory, then any chunk:
    the scratch that the graph refers to is still its own."""
    torch = torch_()
    R = Rows(dllm, 8, 8, 128, "f32", [1000], [90], max_pos=70000)
    ctx, rng = R.ctx, np.random.default_rng(0)
    q, out, other = (ctx.createF32(90 * 1024) for _ in range(3))
    inputs = [rng.standard_normal(90 * 1024).astype(np.float32) for _ in range(2)]
    want = []
    for x in inputs:
        ctx.writeF32(q, x)
        R.attend(q, out=out)
        want.append(ctx.readF32(out, out.n))
    ctx.synchronize()
    stream = torch.cuda.Stream()
    ctx.set_stream(stream.cuda_stream)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        R.attend(q, out=out)

    def chunk_at(t0):
        R.cache.set_t0(0, t0)
        R.attend(q, out=other)
        ctx.synchronize()

    def check_replays():
        for x, w in zip(inputs, want):
            ctx.writeF32(q, x)
            with torch.cuda.stream(stream):
                g.replay()
            assert np.array_equal(ctx.readF32(out, out.n), w)
    chunk_at(3000)
    check_replays()
    held = []  # most of the card: less is left than the chunk at 60000 needs (8 x 2 x 60090 x 128 values of 4 bytes, 492 MB)
    for size in (16 << 30, 1 << 30, 64 << 20):
        while torch.cuda.mem_get_info()[0] > size + (200 << 20):
            held.append(torch.empty(size, dtype=torch.uint8, device="cuda"))
    with pytest.raises(dllm.DllmError) as e:
        chunk_at(60000)
    assert e.value.status == dllm._lib.DLLM_ENOMEM
    free = torch.cuda.mem_get_info()[0]
    chunk_at(200)
    assert torch.cuda.mem_get_info()[0] <= free  # nothing was given back
    check_replays()
    held.clear()
    torch.cuda.empty_cache()
    chunk_at(60000)
    check_replays()
    ctx.set_stream(None)
    del g
    R.close()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m", [1, 20, 90, 300])
@pytest.mark.parametrize("size", [2.0 ** 16, 2.0 ** 40, 2.0 ** 100])
def test_window_attention_of_huge_scores(dllm, kind, m, size):
    """Scores far beyond a softmax's range, equal or further apart than that: the largest share the row,
    and nothing overflows."""
    torch = torch_()

    def edit(_, kv):  # 4-bit codes with nothing to round
        kv[0][:] = np.random.default_rng(1).integers(0, 16, kv[0].shape)
        kv[0][..., ::32], kv[0][..., 1::32] = 0, 15
    R = Rows(dllm, 8, 2, 128, kind, [500], [m], edit=edit)
    # elements of one size: a score is a whole multiple of it, so two are equal or size * log2(e) / sqrt(128) >=
    # 2^13 apart, while fp32 takes at most 22 steps of 2^-23 of 128 * 15 * size * 0.13 from them, a hundredth
    # of that: p is 0 but for the slots with the largest score, and the row a mean of these slots' V in some
    # proportion (their scores are equal but for that rounding, which is more than 1)
    q = np.random.default_rng(2).choice([-size, size], (m, 8, 128)).astype(np.float32)
    k, v = R.values[0]
    slot, at = torch.arange(500, 500 + m, device="cuda")[:, None], torch.arange(500 + m, device="cuda")
    for window, sinks in ((0, 0), (70, 6)):
        out = R.attend(f32(R.ctx, q), window, sinks)
        got = torch.from_numpy(R.ctx.readF32(out, out.n).reshape(m, 8, 128)).cuda().double()
        see = (at <= slot) & ((at > slot - window) | (at < sinks) if window else at >= 0)
        for h in range(8):
            z = torch.where(see, torch.from_numpy(q[:, h]).cuda().double() @ k[:, h // 4].T, -math.inf)
            best, vv = (z == z.amax(-1, keepdim=True))[..., None], v[None, :, h // 4]
            low, high = torch.where(best, vv, math.inf).amin(1), torch.where(best, vv, -math.inf).amax(1)
            room = vv.abs().max() * 2.0 ** -18  # V is to 22 bits; a few sums and a quotient
            assert ((got[:, h] >= low - room) & (got[:, h] <= high + room)).all(), (window, h)
    R.close()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m", [1, 5, 20, 90, 300])
@pytest.mark.parametrize("step", [4.0, 8.0, 9.0])
def test_large_scores_that_grow_by_little(dllm, kind, m, step):
    """Scores of 2^22 to 2^29 where each block of slots exceeds the one before by a step or two of fp32, or
    less: whatever the rounding leaves of their differences, a row is a mean of V."""
    torch = torch_()

    def edit(_, kv):
        kv[0][:] = 0
        kv[0][..., 0] = 1
        kv[0][..., 32] = np.arange(len(kv[0]))[:, None] // 64
    R = Rows(dllm, 8, 2, 128, kind, [3000], [m], edit=edit)
    unit = math.sqrt(128) / math.log2(math.e)  # of a score in powers of two
    for base in [2.0 ** (22 + i / 2) for i in range(14)]:
        for sign in (1, -1):
            q = np.zeros((m, 8, 128), np.float32)
            q[..., 0], q[..., 32] = sign * base * unit * (1 + np.arange(8) / 16), step * unit
            out = R.attend(f32(R.ctx, q))
            got = R.ctx.readF32(out, out.n).reshape(m, 8, 128)
            v = R.values[0][1]
            low, high = (torch.repeat_interleave(f(0), 4, 0).cpu().numpy() for f in (v.amin, v.amax))
            assert ((got >= low - 1e-4) & (got <= high + 1e-4)).all(), (base, sign)
    R.close()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m", [90, 300])
def test_scores_where_eight_rounds_away(dllm, kind, m):
    """Maxima between 2^27 and 2^28, where 8 is half a step of fp32."""
    R = Rows(dllm, 8, 2, 128, kind, [300], [m])
    rng = np.random.default_rng(4)
    for size in (2.0 ** 23, 2.0 ** 24, 2.0 ** 25, 2.0 ** 26):
        q = (rng.standard_normal((m, 8, 128)) * size).astype(np.float32)
        out = R.attend(f32(R.ctx, q))
        got, high = R.ctx.readF32(out, out.n), float(R.values[0][1].abs().max())
        assert (np.abs(got) <= high * (1 + 1e-5)).all(), size
    R.close()


def check_unequal(dllm, kind, m, edit, hd=64, t0=200, window=70, sinks=6):
    """Attention where some slots hold far larger numbers than others: each row within the bound of what it
    sees, and where no row sees such a slot, as near as ever on average."""
    R = Rows(dllm, 8, 2, hd, kind, [t0], [m], edit=edit)
    q = np.random.default_rng(3).standard_normal((m, 8, hd)).astype(np.float32)
    out = R.attend(f32(R.ctx, q), window, sinks)
    got = R.ctx.readF32(out, out.n).reshape(m, 8, hd).astype(np.float64)
    want, vmax, amax = attend64(R, q, window, sinks)
    err, bound = np.abs(got - want), attention_bound(R, vmax, amax)
    assert np.isfinite(got).all()
    assert (err <= bound).all(), f"worst {float((err / bound).max())} of the bound"
    small = vmax.max(1) < 100
    assert np.linalg.norm((got - want)[small]) <= 4e-6 * np.linalg.norm(want[small])
    R.close()


def large_slots(value, m, t0=200):
    """Slots that no row sees, one that only the last row sees and one that the later half does."""
    def edit(_, kv):
        for s in {6, 9, 64, 129} | ({t0 + m // 2, t0 + m - 1} if m > 1 else set()):
            kv[0][s] *= np.float32(value)
            kv[1][s] *= np.float32(value)
    return edit


def spread_slots(_, kv):
    """K of each slot by a power of two down to 2^-60, V by one from 2^-60 to 2^60."""
    rng = np.random.default_rng(9)
    n = len(kv[0])
    kv[0] *= np.ldexp(np.float32(1), rng.integers(-60, 1, (n, 1, 1))).astype(np.float32)
    kv[1] *= np.ldexp(np.float32(1), rng.integers(-60, 61, (n, 1, 1))).astype(np.float32)


@pytest.mark.parametrize("kind,m", [("bf16", 1), ("bf16", 8), ("f32", 1), ("f32", 8), ("f32", 20)] +
                         [(k, m) for k in KINDS for m in (90, 300)])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("value", [2.0 ** 12, 2.0 ** 20, 2.0 ** 36, 1e30])
def test_large_hidden_values_do_not_leak(dllm, kind, m, hd, value):
    check_unequal(dllm, kind, m, large_slots(value, m), hd)


@pytest.mark.parametrize("kind,m", [("bf16", 1), ("bf16", 8), ("f32", 1), ("f32", 8), ("f32", 20)] +
                         [(k, m) for k in KINDS for m in (90, 300)])
@pytest.mark.parametrize("window,sinks", [(70, 6), (0, 0), (150, 0), (1, 0)])
def test_slots_of_very_unequal_sizes(dllm, kind, m, window, sinks):
    check_unequal(dllm, kind, m, spread_slots, 64 if m % 4 else 128, 333, window, sinks)


@pytest.mark.parametrize("m", [1, 2, 3, 4, 8, 16])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("value", [2.0 ** 12, 2.0 ** 20, 2.0 ** 40, 1e30, 2.0 ** 106])
def test_large_hidden_codes_do_not_leak(dllm, m, hd, value):
    """The scales of hidden slots of a 4-bit cache, in tiles of 8, 16 and 32 rows."""
    check_unequal(dllm, "4", m, large_slots(value, m), hd)


@pytest.mark.parametrize("m", [1, 2, 3, 4, 8, 16])
@pytest.mark.parametrize("window,sinks", [(70, 6), (0, 0), (150, 0), (1, 0)])
def test_codes_of_very_unequal_scales(dllm, m, window, sinks):
    check_unequal(dllm, "4", m, spread_slots, 64 if m % 4 else 128, 333, window, sinks)


@pytest.mark.parametrize("m", [1, 3, 8])
def test_scales_from_the_smallest_to_the_largest(dllm, m):
    """Rows that see scales of 2^-60 beside slots that they do not see of 2^106, and the other way round."""
    def edit(_, kv):
        kv[1] *= np.float32(2.0 ** -60)
        kv[1][::2] *= np.float32(2.0 ** 60)
        kv[1][64:128] *= np.float32(2.0 ** 106)
        kv[1][200:, :, 32:] *= np.float32(2.0 ** 100)
    check_unequal(dllm, "4", m, edit, 64, 200, 70, 6)


@pytest.mark.parametrize("m", [1, 3, 8, 90])
@pytest.mark.parametrize("value", [-3.4028235e38, 3.4028235e38, -3.397e38, -3.38953139e38, 3.38953139e38])
def test_codes_of_the_largest_numbers(dllm, m, value):
    """32 values beyond the largest bf16 number read NaN, by read_rows and by attention alike, and change
    nothing where they are hidden; the largest number itself is kept."""
    value = np.float32(value)
    fits = abs(float(value)) <= float.fromhex("0x1.fep127")

    def edit(_, kv):
        for x in kv:
            x[40, :, :32] = x[210 + m - 1, :, :32] = value
            x[41, :, 32] = np.float32(-3.4028235e38)  # among ordinary values: a range beyond 2^112 besides
    R = Rows(dllm, 4, 2, 64, "4", [210], [m], edit=edit)
    R.cache.set_t0(0, 0)
    got = R.ctx.readF32(R.cache.read_rows(0, R.ctx.rowBatch([210 + m]))[1], (210 + m) * 128).reshape(-1, 2, 2, 32)
    R.cache.set_t0(0, 210)
    assert np.isnan(got[41, :, 1]).all()
    assert (got[[40, -1], :, 0] == value).all() if fits else np.isnan(got[[40, -1], :, 0]).all()
    got[[40, -1], :, 0] = got[41, :, 1] = 0
    assert np.isfinite(got).all()
    # the last row, which sees its own slot, aside
    R.values = [[torch_().nan_to_num(x, 0.0, 0.0, 0.0) for x in R.values[0]]]
    q = np.random.default_rng(3).standard_normal((m, 4, 64)).astype(np.float32)
    out = R.attend(f32(R.ctx, q), 100, 6)
    got = R.ctx.readF32(out, out.n).reshape(m, 4, 64)
    want, vmax, amax = attend64(R, q, 100, 6)
    assert (np.abs(got - want) <= attention_bound(R, vmax, amax))[:-1].all()
    if not fits:
        assert np.isnan(got[-1, :, :32]).all()
    R.close()


@pytest.mark.parametrize("kind", KINDS)
def test_values_while_the_scratch_grows(dllm, kind):
    """Chunk after chunk of a conversation of ordinary numbers: the outputs are the definition's whenever the
    scratch has just been replaced, and in between."""
    torch = torch_()
    far, chunk, nq, kvh, hd = 3000, 200, 8, 4, 128
    ctx = make_ctx(dllm, nq, kvh, hd, max_pos=far, max_seqs=1, kv_dtype="bf16" if kind == "bf16" else "f32")
    R = object.__new__(Rows)
    R.ctx, R.kind, R.nq, R.kvh, R.hd, R.layer = ctx, kind, nq, kvh, hd, 0
    R.cache = dllm.Cache4(ctx, 0, 1) if kind == "4" else dllm.Stage(ctx, 0, 1)
    rng, rows = np.random.default_rng(8), ctx.rowBatch([chunk])
    R.rows, R.counts, R.values = rows, [chunk], [[torch.empty((0, kvh, hd), dtype=torch.float64, device="cuda")] * 2]
    q, k, v = (ctx.createF32(chunk * h * hd) for h in (nq, kvh, kvh))
    out, held = ctx.createF32(chunk * nq * hd), []
    for t in range(0, far, chunk):
        x = [rng.standard_normal((chunk, h, hd)).astype(np.float32) for h in (nq, kvh, kvh)]
        for b, a in zip((q, k, v), x):
            ctx.writeF32(b, a)
        R.cache.set_t0(0, t)
        R.append(rows, k, v)
        R.lens = [t]
        R.values = [[torch.cat([h, torch.from_numpy(R.held(a)).cuda()]) for h, a in zip(R.values[0], x[1:])]]
        ctx.writeF32(out, np.full(out.n, np.nan))
        free = torch.cuda.mem_get_info()[0]
        R.attend(q, out=out)
        held.append(torch.cuda.mem_get_info()[0] != free)
        got = ctx.readF32(out, out.n).reshape(chunk, nq, hd)
        want, vmax, amax = attend64(R, x[0], 0, 0)
        assert (np.abs(got - want) <= attention_bound(R, vmax, amax)).all(), t
        assert np.linalg.norm(got - want) <= 4e-6 * np.linalg.norm(want)
    assert sum(held) >= 2  # it did grow
    R.close()
