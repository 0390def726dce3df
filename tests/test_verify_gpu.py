"""The operators that verify drafted tokens, each against its definition in 64 bits:
rotary positions per row, attention of a tree over the paged cache, token picks
under penalties, biases and masks, and the cache rows of an accepted path; then all
of them together as speculative decoding runs them.

eps below is half a step of fp32, 2^-24."""
import math

import numpy as np
import pytest

from helpers import assert_close, build_leader, get_weights, oracle_cfg
import synth

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -24


def torch_():
    import torch
    return torch


def f32(ctx, a):
    a = np.ascontiguousarray(a, np.float32)
    b = ctx.createF32(a.size)
    ctx.writeF32(b, a)
    return b


def i32(ctx, a):
    a = np.ascontiguousarray(a).astype(np.int64).astype(np.uint32).view(np.int32)
    b = ctx.createI32(a.size)
    ctx.writeI32(b, a)
    return b


def make_ctx(dllm, nq=4, kvh=2, hd=64, **kw):
    base = dict(vocab_size=4096, hidden_size=256, num_layers=2, num_q_heads=nq, num_kv_heads=kvh, head_dim=hd,
                intermediate_size=512, max_pos=512)
    base.update(kw)
    return dllm.initKernels(0, dllm.ModelConfig(**base))


# ---- rotary positions ------------------------------------------------------------------------
def frequencies(rd, theta, scaling):
    i = np.arange(rd // 2, dtype=np.float64)
    kind = (scaling or {}).get("type")
    if kind == "ntk":
        return (theta * scaling["factor"] ** (rd / (rd - 2))) ** (-2 * i / rd), 1.0
    f = theta ** (-2 * i / rd)
    if kind == "linear":
        return f / scaling["factor"], 1.0
    if kind == "yarn":
        def pair(beta):
            return rd * math.log(scaling["original_max_pos"] / (beta * 2 * math.pi)) / (2 * math.log(theta))
        lo, hi = max(math.floor(pair(32)), 0), min(math.ceil(pair(1)), rd - 1)
        ramp = np.clip((i - lo) / ((hi - lo) or 0.001), 0, 1)
        return f / scaling["factor"] * ramp + f * (1 - ramp), 0.1 * math.log(scaling["factor"]) + 1
    return f, 1.0


def rope64(x, pos, rd, layout, f, factor):
    """x [n, heads, hd] in 64 bits, and |x1| + |x2| of every element's pair (0: passes)."""
    x = x.astype(np.float64)
    a = pos.astype(np.float64)[:, None, None] * f
    c, s = np.cos(a) * factor, np.sin(a) * factor
    i1, i2 = (np.arange(rd // 2), np.arange(rd // 2) + rd // 2) if layout == "half" else (np.arange(0, rd, 2),
                                                                                       np.arange(1, rd, 2))
    y, mag = x.copy(), np.zeros_like(x)
    y[..., i1] = x[..., i1] * c - x[..., i2] * s
    y[..., i2] = x[..., i1] * s + x[..., i2] * c
    mag[..., i1] = mag[..., i2] = np.abs(x[..., i1]) + np.abs(x[..., i2])
    return y, mag


SCALINGS = [None, {"type": "linear", "factor": 8.0}, {"type": "ntk", "factor": 3.0},
            {"type": "yarn", "factor": 4.0, "original_max_pos": 32768}]
ROTARY = [(64, 64), (64, 22), (128, 128), (128, 96), (128, 34), (128, 120)]


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("hd,rd,scaling", [(h, r, s) for h, r in ROTARY for s in SCALINGS] +
                         [(64, 2, s) for s in SCALINGS if not s or s["type"] != "ntk"])  # ntk needs two pairs
def test_rope_at(dllm, layout, hd, rd, scaling):
    nq, kvh = 6, 2
    ctx = make_ctx(dllm, nq, kvh, hd)
    plan = ctx.ropePlan(layout=layout, rotary_dim=rd, theta=1e6, scaling=scaling)
    f, factor = frequencies(rd, 1e6, scaling)
    rng = np.random.default_rng(rd)
    for n in (1, 3, 37):
        pos = rng.integers(0, 1 << 24, n)
        pos[0] = 0
        q, k = rng.standard_normal((n, nq, hd), np.float32), rng.standard_normal((n, kvh, hd), np.float32)
        qb, kb, pb = f32(ctx, q), f32(ctx, k), i32(ctx, pos)
        qo, ko = ctx.createF32(q.size), ctx.createF32(k.size)
        ctx.ropeAt(plan, pb, n, qb, kb, qo, ko)
        outs = [ctx.readF32(b, b.n) for b in (qo, ko)]
        assert np.array_equal(ctx.readF32(qb, qb.n), q.reshape(-1))  # inputs untouched
        ctx.ropeAt(plan, pb, n, qb, kb)  # in place
        inplace = [ctx.readF32(b, b.n) for b in (qb, kb)]
        for x, o, ip in ((q, outs[0], inplace[0]), (k, outs[1], inplace[1])):
            want, mag = rope64(x, pos, rd, layout, f, factor)
            # the turn in 32 bits: pi eps; sincospi: 2 eps; the factor: eps; two rounded products: 2 eps.
            # 9 eps (|x1| + |x2|) factor covers their sum; positions below 2^24 add less than eps / 10.
            err = np.abs(o.reshape(x.shape) - want)
            assert (err <= 9 * EPS * factor * mag).all(), (n, float((err / np.maximum(mag, 1e-30)).max() / EPS))
            assert np.array_equal(o, ip)
    ctx.close()


@pytest.mark.parametrize("theta,original,turns", [(1e6, 4, "few"), (1e4, 1, "few"), (100.0, 2 ** 31 - 1, "many"),
                                                  (1.5, 100000, "many")])
def test_rope_at_yarn_without_a_ramp(dllm, theta, original, turns):
    """Contexts in which every pair makes less than one turn (all of them are slow: divided by
    the factor), or every pair more than 32 (all fast: as they are)."""
    ctx = make_ctx(dllm, 4, 2, 64)
    plan = ctx.ropePlan(theta=theta, scaling={"type": "yarn", "factor": 4.0, "original_max_pos": original})
    f = theta ** (-np.arange(32, dtype=np.float64) / 32)
    of = original * f / (2 * math.pi)
    assert (of < 1).all() if turns == "few" else (of > 32).all()
    rng = np.random.default_rng(1)
    pos = rng.integers(0, 1 << 20, 5)
    q = rng.standard_normal((5, 4, 64), np.float32)
    b = f32(ctx, q)
    ctx.ropeAt(plan, i32(ctx, pos), 5, b)
    factor = 0.1 * math.log(4.0) + 1
    want, mag = rope64(q, pos, 64, "half", f / 4.0 if turns == "few" else f, factor)
    # as in test_rope_at
    assert (np.abs(ctx.readF32(b, b.n).reshape(q.shape) - want) <= 9 * EPS * factor * mag).all()
    ctx.close()


def test_rope_at_one_of_q_and_k_and_far_positions(dllm):
    ctx = make_ctx(dllm, 4, 1, 128)
    plan = ctx.ropePlan(theta=1e4)
    f, _ = frequencies(128, 1e4, None)
    rng = np.random.default_rng(5)
    pos = np.array([2 ** 31 - 1, -5, 123456789, -2 ** 31])
    q, k = rng.standard_normal((4, 4, 128), np.float32), rng.standard_normal((4, 1, 128), np.float32)
    pb = i32(ctx, pos)
    for x, kw in ((q, "qBuf"), (k, "kBuf")):
        b = f32(ctx, x)
        ctx.ropeAt(plan, pb, 4, **{kw: b})
        want, mag = rope64(x, pos, 128, "half", f, 1.0)
        # both sides hold pos * frequency in 64 bits: 2^31 radians to 2^-52 of them each, 16 eps together
        assert (np.abs(ctx.readF32(b, b.n).reshape(x.shape) - want) <= 25 * EPS * mag).all()
    ctx.close()


def test_rope_at_refusals(dllm):
    ctx, other = make_ctx(dllm), make_ctx(dllm)
    E = dllm.DllmError
    for kw in (dict(rotary_dim=0), dict(rotary_dim=7), dict(rotary_dim=66), dict(theta=1.0), dict(theta=float("nan")),
               dict(scaling={"type": "linear", "factor": 0.5}), dict(scaling={"type": "yarn", "factor": 2.0}),
               dict(scaling={"type": "ntk", "factor": 2.0}, rotary_dim=2),
               dict(scaling={"type": "yarn", "factor": 2.0, "original_max_pos": 64, "beta_fast": 1.0}),
               dict(scaling={"attention_factor": -1.0})):
        with pytest.raises(E):
            ctx.ropePlan(**kw)
    plan = ctx.ropePlan()
    q, k, p = ctx.createF32(4 * 256), ctx.createF32(4 * 128), ctx.createI32(4)
    for args in ((plan, p, 0, q, k), (plan, p, 5, q, k), (plan, q, 4, q, k), (plan, p, 4), (plan, p, 4, p, k),
                 (plan, p, 4, None, k, q), (plan, p, 4, q, q), (plan, p, 4, q, k, k, k), (plan, p, 4, q, k, None, q),
                 (other.ropePlan(), p, 4, q, k), (plan, other.createI32(4), 4, q, k)):
        with pytest.raises(E):
            ctx.ropeAt(*args)
    ctx.close()
    other.close()


# ---- attention of a tree ------------------------------------------------------------------------
def chain(m):
    return list(range(-1, m - 1))


def bushy(rng, m, roots=1):
    return [-1 if i < roots else int(rng.integers(0, i)) for i in range(m)]


def ancestors(parents):
    see = np.zeros((len(parents), len(parents)), bool)
    for i, p in enumerate(parents):
        if p >= 0:
            see[i] = see[p]
        see[i, i] = True
    return see


class Paged:
    """A stage with random cache contents under shuffled pages, and the same in numpy."""

    def __init__(self, dllm, nq, kvh, hd, kv, lens, trees, page=64, layers=1, seed=0, max_pos=None, seqs=None):
        torch = torch_()
        self.lens, self.trees = lens, trees
        max_pos = max_pos or max(t + len(p) for t, p in zip(lens, trees))
        self.seqs = seqs or list(range(len(lens)))
        max_seqs = max(self.seqs) + 1
        self.ctx = make_ctx(dllm, nq, kvh, hd, kv_dtype=kv, kv_page_size=page, max_pos=max_pos, max_seqs=max_seqs,
                            num_layers=layers)
        self.stage = dllm.Stage(self.ctx, 0, layers)
        rng = np.random.default_rng(seed)
        per = self.stage.pages_per_seq()
        table = rng.permutation(max_seqs * per).reshape(max_seqs, per)
        g = torch.Generator().manual_seed(seed)
        dt = torch.bfloat16 if kv == "bf16" else torch.float32
        self.pool = []
        for which in ("k", "v"):
            dev = torch.as_tensor(self.stage.kv_pool(which), device="cuda").view(dt)
            host = torch.randn(dev.shape, generator=g).to(dt)
            dev.copy_(host)
            self.pool.append(dev)
        torch.cuda.synchronize()
        self.page = page
        self.table = table
        for s in range(max_seqs):
            self.stage.set_page_table(s, table[s])
        for s, t in zip(self.seqs, lens):
            self.stage.set_t0(s, t)
        self.tree = self.ctx.draftTree([p for t in trees for p in t], [len(t) for t in trees], self.seqs)
        self.nq, self.kvh, self.hd, self.kv = nq, kvh, hd, kv

    def rows(self, which, s, n, layer=0):
        """Slots [0, n) of sequence s as [n, KVH, HD], 64 bits."""
        pool = self.pool[which][layer].float().cpu().numpy().astype(np.float64)
        at = np.arange(n)
        return pool[self.table[s][at // self.page], :, at % self.page]

    def close(self):
        self.stage.close()
        self.ctx.close()


def attend64(P, q):
    """The definition, and per row the largest |v| and the largest sum of |q_i k_i| in
    powers of two (what the error bound is made of)."""
    G = P.nq // P.kvh
    out, vmax, amax, row = [], [], [], 0
    for s, t0, parents in zip(P.seqs, P.lens, P.trees):
        m = len(parents)
        if not m:
            continue
        k, v = P.rows(0, s, t0 + m), P.rows(1, s, t0 + m)
        see = np.concatenate([np.ones((m, t0), bool), ancestors(parents)], 1)
        qq = q[row:row + m].astype(np.float64)
        row += m
        o = np.zeros((m, P.nq, P.hd))
        a = np.zeros((m, P.nq))
        for h in range(P.nq):
            kk, vv = k[:, h // G], v[:, h // G]
            z = np.where(see, qq[:, h] @ kk.T / math.sqrt(P.hd), -np.inf)
            e = np.exp(z - z.max(-1, keepdims=True))
            o[:, h] = (e / e.sum(-1, keepdims=True)) @ vv
            a[:, h] = (np.abs(qq[:, h]) @ np.abs(kk).T).max(-1) * math.log2(math.e) / math.sqrt(P.hd)
        out.append(o)
        amax.append(a)
        vmax.append(np.full((m, P.nq), np.abs(v).max()))
    return np.concatenate(out), np.concatenate(vmax), np.concatenate(amax)


def attention_bound(P, vmax, amax, slots):
    """A score sums hd products in at most hd / 8 + 6 truncated steps of 2^-23 of the sum of
    magnitudes (operands cut to 22 bits or more count as two of the six): e. Every p is
    off by e ln 2 and the exponential's 2^-21 relative, which counts twice (numerator and
    sum); a block's product adds up to 12 truncated steps of 2^-23, the blocks one rounding
    each, the join and the quotient a few more."""
    e = (P.hd / 8 + 6) * 2.0 ** -23 * amax
    return (vmax * (2 * (0.7 * e + 2.0 ** -21) + (20 + slots / 64) * 2.0 ** -23))[:, :, None]


def check_attention(P, seed=1, scale=1.5):
    n = sum(len(t) for t in P.trees)
    q = np.random.default_rng(seed).standard_normal((n, P.nq, P.hd)).astype(np.float32) * np.float32(scale)
    out = P.stage.tree_attention(0, P.tree, f32(P.ctx, q))
    got = P.ctx.readF32(out, out.n).reshape(n, P.nq, P.hd)
    want, vmax, amax = attend64(P, q)
    bound = attention_bound(P, vmax, amax, max(t + len(p) for t, p in zip(P.lens, P.trees)))
    err = np.abs(got - want)
    assert np.isfinite(got).all()
    assert (err <= bound).all(), f"worst {float((err / bound).max())} of the bound, {float(err.max())}"
    # on average the errors are far inside the worst case; fp32 level
    assert np.linalg.norm(got - want) <= 4e-6 * np.linalg.norm(want)


HEAD_SHAPES = [(4, 2, 64), (7, 1, 64), (8, 1, 128), (6, 2, 128), (2, 2, 128)]


@pytest.mark.parametrize("kv", ["bf16", "f32"])
@pytest.mark.parametrize("nq,kvh,hd", HEAD_SHAPES)
@pytest.mark.parametrize("m", [1, 2, 5, 9, 17, 33, 64])
@pytest.mark.parametrize("t0", [0, 1, 63, 200])
def test_tree_attention_small(dllm, kv, nq, kvh, hd, m, t0):
    P = Paged(dllm, nq, kvh, hd, kv, [t0], [bushy(np.random.default_rng(m), m)])
    check_attention(P)
    P.close()


@pytest.mark.parametrize("kv", ["bf16", "f32"])
@pytest.mark.parametrize("t0,m,page", [(4095, 1, 64), (5000, 13, 32), (3001, 64, 128), (9999, 7, 64)])
def test_tree_attention_long(dllm, kv, t0, m, page):
    P = Paged(dllm, 14, 2, 64, kv, [t0], [bushy(np.random.default_rng(m), m)], page=page)
    check_attention(P)
    P.close()


@pytest.mark.parametrize("kv", ["bf16", "f32"])
@pytest.mark.parametrize("page", [32, 64, 256])
def test_tree_attention_batch(dllm, kv, page):
    """Sequences of unequal lengths and trees, one without nodes, in another order than
    the cache's; the slots behind each (other data) are not seen."""
    rng = np.random.default_rng(7)
    lens = [700, 0, 33, 2100, 64, 5]
    trees = [bushy(rng, 9), chain(3), [], bushy(rng, 21, roots=3), [-1], chain(30)]
    P = Paged(dllm, 12, 2, 128, kv, lens, trees, page=page, max_pos=2300, seqs=[3, 0, 5, 1, 7, 2])
    check_attention(P)
    P.close()


@pytest.mark.parametrize("kv", ["bf16", "f32"])
def test_tree_attention_idle_sequences_change_nothing(dllm, kv):
    """A long sequence without nodes has no work, and does not move the others to another kernel."""
    tree = bushy(np.random.default_rng(4), 9)
    P = Paged(dllm, 8, 1, 64, kv, [2000, 9000], [tree, []])
    q = f32(P.ctx, np.random.default_rng(5).standard_normal(9 * 8 * 64))
    out = P.stage.tree_attention(0, P.tree, q)
    alone = P.stage.tree_attention(0, P.ctx.draftTree(tree), q)
    assert np.array_equal(P.ctx.readF32(out, out.n), P.ctx.readF32(alone, alone.n))
    check_attention(P)
    P.close()


@pytest.mark.parametrize("kv", ["bf16", "f32"])
@pytest.mark.parametrize("hd,nq,lens,m", [(128, 12, [8051, 6039], 55), (128, 12, [8051] * 3, 23),
                                          (64, 16, [7990, 8001, 5000, 6666], 40), (128, 16, [2001] * 16, 9)])
def test_tree_attention_many_blocks_per_split(dllm, kv, hd, nq, lens, m):
    """The drafted rows come after many turns of the K/V rings and end inside a block."""
    rng = np.random.default_rng(m)
    P = Paged(dllm, nq, 2, hd, kv, lens, [bushy(rng, m) for _ in lens])
    check_attention(P)
    P.close()


@pytest.mark.parametrize("kv", ["bf16", "f32"])
def test_tree_attention_leftovers_after_many_blocks(dllm, kv):
    """NaN behind the last node, and in a drafted row that only itself sees, far into a split."""
    lens, m = [8051, 6039], 55
    trees = [[-1] + [0] * (m - 1)] * 2
    P = Paged(dllm, 12, 2, 128, kv, lens, trees, max_pos=8192)
    n = 2 * m
    q = f32(P.ctx, np.random.default_rng(3).standard_normal((n, 12 * 128)))
    want = P.ctx.readF32(P.stage.tree_attention(0, P.tree, q), n * 12 * 128).reshape(n, -1)
    assert np.isfinite(want).all()
    for s, t0 in enumerate(lens):
        for slot in [*range(t0 + m, 8192), t0 + 20]:
            for pool in P.pool:
                pool[:, int(P.table[s][slot // 64]), :, slot % 64] = float("nan")
    torch_().cuda.synchronize()
    got = P.ctx.readF32(P.stage.tree_attention(0, P.tree, q), n * 12 * 128).reshape(n, -1)
    seers = [20, m + 20]
    assert np.isnan(got[seers]).all()
    rest = np.delete(np.arange(n), seers)
    assert np.array_equal(got[rest], want[rest])
    P.close()


def test_tree_attention_many_sequences(dllm):
    rng = np.random.default_rng(8)
    lens = [int(x) for x in rng.integers(0, 90, 128)]
    trees = [bushy(rng, int(m)) for m in rng.integers(0, 7, 128)]
    trees[0] = chain(4)
    P = Paged(dllm, 4, 2, 64, "bf16", lens, trees, page=32)
    check_attention(P)
    P.close()


def test_tree_attention_sharp_rows(dllm):
    """Large scores: one slot takes nearly all the weight, the rest underflows."""
    P = Paged(dllm, 4, 2, 128, "f32", [300], [bushy(np.random.default_rng(3), 12)])
    check_attention(P, scale=40.0)
    P.close()


def low_bits(x, bits=13):
    return int(np.float32(x).view(np.uint32)) & ((1 << bits) - 1)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("nq,m", [(2, 1), (16, 3)])  # tiles of 16 and of 32 rows
def test_tree_attention_keeps_the_low_bits_of_q_and_k(dllm, hd, nq, m):
    """An fp32 cache, two slots of equal weight per node: k and, scaled, q hold a leading one
    and ones in their last 13 bits, which the tf32 tiles take as a second term. A node's own k
    is the next number, whose second term is zero.

    With z the score in powers of two (about 2^11), the scores differ by z 2^-23. Of what the
    products lose, everything that is in proportion to k cancels between the slots (the cut of
    q, the rounding of q's scale). What is left: the second term of k, 13 ones, is rounded to
    11 bits, one step of 2^-23; both scores are summed from two accumulators, 2^-24 each. The
    difference is off by d = z 2^-22 at most, the weights 1 / (1 + 2^-difference) by
    d ln2 / 4, and V = 1, -1 counts that twice. p and the sum are off by the exponential's
    2^-21 and roundings below it: 2^-19 covers them. Left out, the product of the two second
    terms would shift one score by z 2^-20, four times d."""
    P = Paged(dllm, nq, 2, hd, "f32", [1], [[-1] * m])
    scale = np.float32(math.log2(math.e) / math.sqrt(hd))
    target = np.float32(64 * (1 + 2.0 ** -10 - 2.0 ** -23))
    near = (np.float32(target / scale).view(np.int32) + np.arange(-4, 5, dtype=np.int32)).view(np.float32)
    q0 = max((c for c in near if c * scale <= target), key=lambda c: c * scale)
    assert low_bits(q0 * scale) >= 0x1ffc and q0 * scale <= target
    k0 = np.float32(32 * (1 + 2.0 ** -10 - 2.0 ** -23))
    k1 = np.float32(32 * (1 + 2.0 ** -10))
    assert low_bits(k0) == 0x1fff and low_bits(k1) == 0
    for pool in P.pool:
        pool.zero_()
    page = int(P.table[0][0])
    P.pool[0][0, page, :, 0, 0], P.pool[0][0, page, :, 1:1 + m, 0] = float(k0), float(k1)
    P.pool[1][0, page, :, 0], P.pool[1][0, page, :, 1:1 + m] = 1.0, -1.0
    torch_().cuda.synchronize()
    q = np.zeros((m, nq, hd), np.float32)
    q[:, :, 0] = q0
    z = [float(q0) * float(k) / math.sqrt(hd) * math.log2(math.e) for k in (k0, k1)]
    want = 2.0 / (1.0 + 2.0 ** (z[1] - z[0])) - 1.0
    out = P.stage.tree_attention(0, P.tree, f32(P.ctx, q))
    err = np.abs(P.ctx.readF32(out, out.n).astype(np.float64) - want).max()
    assert err <= z[0] * 2.0 ** -22 * math.log(2) / 2 + 2.0 ** -19, (err, z[0] * 2.0 ** -20 * math.log(2) / 2)
    P.close()


@pytest.mark.parametrize("kv,operand", [("bf16", "q"), ("f32", "q"), ("f32", "k")])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("nq,m,t0", [(2, 1, 1), (16, 3, 1), (16, 5, 1), (16, 16, 1), (16, 16, 4800)])  # every kernel
def test_tree_attention_operands_keep_their_last_bits(dllm, kv, operand, hd, nq, m, t0):
    """One context slot and a node's own slot of nearly equal scores z of about 2^11 (in powers
    of two); all others have a score of 0 and no weight. One operand of the first score is
    1 + 2^-9 and ones in its last 5 bits, its counterpart 1 + 2^-9: an operand that is held in
    19 bits, or in two bf16 terms, shifts the first score by z 2^-18.

    A score may lose: the rounding of q's scale, z 2^-24; the last bits of q and k, z 2^-22 each
    where two tf32 terms hold them; the sum of its parts in fp32, rounded or cut, z 2^-24 twice:
    10 z 2^-24, and the two scores' difference twice that. V = 1, -1 makes it half that times
    ln2 in the output; 2^-19 covers the exponential and the quotient."""
    trees = [[-1] * m]
    P = Paged(dllm, nq, 2, hd, kv, [t0], trees)
    scale = np.float32(math.log2(math.e) / math.sqrt(hd))

    def unscaled(x):  # the float whose scaled value comes nearest to x
        c = (np.float32(x / scale).view(np.int32) + np.arange(-4, 5, dtype=np.int32)).view(np.float32)
        return min(c, key=lambda y: abs(float(y * scale) - float(x)))

    full, short = (np.float32(1 + 2.0 ** -9 + last) for last in (2.0 ** -18 - 2.0 ** -23, 0.0))
    assert low_bits(full, 14) == 0x1f and low_bits(short, 14) == 0
    if operand == "q":  # q in two dims, each slot has one of them
        q01, k0, k1 = (unscaled(64 * full), unscaled(64 * short)), (32.0, 0.0), (0.0, 32.0)
        assert low_bits(q01[0] * scale, 5) >= 0x1d
    else:
        q01, k0, k1 = (unscaled(np.float32(64)), np.float32(0)), (float(32 * full), 0.0), (float(32 * short), 0.0)
    for pool in P.pool:
        pool.zero_()
    slot = lambda j: (int(P.table[0][j // 64]), j % 64)  # noqa: E731
    for j, k, v in [(0, k0, 1.0)] + [(t0 + i, k1, -1.0) for i in range(m)]:
        page, row = slot(j)
        P.pool[0][0, page, :, row, 0], P.pool[0][0, page, :, row, 1] = k
        P.pool[1][0, page, :, row] = v
    torch_().cuda.synchronize()
    q = np.zeros((m, nq, hd), np.float32)
    q[:, :, 0], q[:, :, 1] = q01
    z = [(float(q01[0]) * k[0] + float(q01[1]) * k[1]) / math.sqrt(hd) * math.log2(math.e) for k in (k0, k1)]
    want = 2.0 / (1.0 + 2.0 ** (z[1] - z[0])) - 1.0
    out = P.stage.tree_attention(0, P.tree, f32(P.ctx, q))
    err = np.abs(P.ctx.readF32(out, out.n).astype(np.float64) - want).max()
    bound = z[0] * 20 * 2.0 ** -24 * math.log(2) / 2 + 2.0 ** -19
    assert bound < 0.5 * z[0] * 2.0 ** -18 * math.log(2) / 2  # a lost term is well outside
    assert err <= bound, (err, bound)
    P.close()


@pytest.mark.parametrize("kv", ["bf16", "f32"])
@pytest.mark.parametrize("nq", [2, 16])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_tree_attention_masked_rows_do_not_leak(dllm, kv, nq, value):
    """A drafted row of non-finite K and V reaches only the nodes that see it."""
    torch = torch_()
    parents = [-1, 0, 0, 1, 2, 4]
    P = Paged(dllm, nq, 2, 64, kv, [130], [parents])
    q = np.random.default_rng(2).standard_normal((6, nq, 64)).astype(np.float32)
    want, vmax, amax = attend64(P, q)
    bound = attention_bound(P, vmax, amax, 136)
    slot = 130 + 2  # node 2: seen by 2, 4, 5
    for pool in P.pool:
        pool[0, int(P.table[0][slot // 64]), :, slot % 64] = value
    # garbage behind the last node is never seen
    for s in range(136, P.stage.pages_per_seq() * 64):
        P.pool[1][0, int(P.table[0][s // 64]), :, s % 64] = float("nan")
    torch.cuda.synchronize()
    out = P.stage.tree_attention(0, P.tree, f32(P.ctx, q))
    got = P.ctx.readF32(out, out.n).reshape(want.shape)
    seen = ancestors(parents)[:, 2]
    assert (np.abs(got - want) <= bound)[~seen].all()
    assert not np.isfinite(got[seen]).any()
    P.close()


def test_tree_attention_infinite_value_seen(dllm):
    """Finite scores, an infinite V element: it comes out where it is seen, its own dim only."""
    torch = torch_()
    parents = [-1, 0, 0]
    P = Paged(dllm, 2, 2, 64, "f32", [10], [parents])
    q = np.random.default_rng(2).standard_normal((3, 2, 64)).astype(np.float32)
    want, vmax, amax = attend64(P, q)
    bound = attention_bound(P, vmax, amax, 13)
    P.pool[1][0, int(P.table[0][0]), 1, 11, 5] = float("inf")  # node 1, head 1, dim 5
    torch.cuda.synchronize()
    out = P.stage.tree_attention(0, P.tree, f32(P.ctx, q))
    got = P.ctx.readF32(out, out.n).reshape(want.shape)
    assert got[1, 1, 5] == float("inf")
    keep = np.ones(got.shape, bool)
    keep[1, 1, 5] = False
    assert (np.abs(got - want) <= bound)[keep].all()
    P.close()


@pytest.mark.parametrize("kv", ["bf16", "f32"])
def test_append_tree(dllm, kv):
    torch = torch_()
    P = Paged(dllm, 4, 2, 64, kv, [70, 0, 31], [chain(5), [], bushy(np.random.default_rng(1), 40)], page=32, layers=2,
              seqs=[2, 1, 0])
    before = [p.clone() for p in P.pool]
    rng = np.random.default_rng(3)
    k, v = (rng.standard_normal((45, 2, 64)).astype(np.float32) for _ in range(2))
    P.stage.append_tree(1, P.tree, f32(P.ctx, k), f32(P.ctx, v))
    P.ctx.synchronize()
    for pool, old, rows in zip(P.pool, before, (k, v)):
        want, row = old.clone(), 0
        for s, t0, tree in zip(P.seqs, P.lens, P.trees):
            for j in range(len(tree)):
                want[1, int(P.table[s][(t0 + j) // 32]), :, (t0 + j) % 32] = torch.from_numpy(rows[row]).to(want.dtype).cuda()
                row += 1
        assert torch.equal(pool, want)
    assert [P.stage.t0_of(s) for s in P.seqs] == P.lens
    P.close()


def test_commit_tree_takes_iterators(dllm):
    P = Paged(dllm, 4, 2, 64, "f32", [5, 9], [[-1, 0, 0], [-1, 0]])
    P.stage.commit_tree(P.tree, (iter(p) for p in ([0, 2], [0])))
    assert [P.stage.t0_of(s) for s in (0, 1)] == [7, 10]
    P.close()


@pytest.mark.parametrize("kv", ["bf16", "f32"])
@pytest.mark.parametrize("hd", [64, 128])
def test_commit_tree(dllm, kv, hd):
    torch = torch_()
    rng = np.random.default_rng(4)
    trees = [chain(64), [-1, 0, 0, 2, 1, 3, 5], [-1], [], [-1, -1, 1], bushy(rng, 30)] + [[-1, 0, 0]] * 40
    deep = [29]
    while trees[5][deep[0]] >= 0:
        deep.insert(0, trees[5][deep[0]])
    paths = [list(range(64)), [0, 2, 3, 5, 6], [0], [], [1, 2], deep] + [[0, 2]] * 40
    lens = [3, 60, 17, 9, 95, 0] + [100] * 40
    P = Paged(dllm, 4, 2, hd, kv, lens, trees, page=32, layers=3)
    want = [p.clone() for p in P.pool]
    for w in want:
        for s, (t0, path) in enumerate(zip(lens, paths)):
            at = lambda j: (int(P.table[s][(t0 + j) // 32]), (t0 + j) % 32)  # noqa: E731
            rows = [w[:, at(j)[0], :, at(j)[1]].clone() for j in path]
            for j, r in enumerate(rows):
                w[:, at(j)[0], :, at(j)[1]] = r
    P.stage.commit_tree(P.tree, paths)
    P.ctx.synchronize()
    for pool, w in zip(P.pool, want):
        assert torch.equal(pool, w)
    assert [P.stage.t0_of(s) for s in range(len(lens))] == [t + len(p) for t, p in zip(lens, paths)]
    P.close()


def test_commit_tree_on_a_stage_without_layers(dllm):
    """Nothing to move, but more sequences whose rows would have to than one launch takes: T0 moves on."""
    n = 128
    ctx = make_ctx(dllm, max_seqs=n, max_pos=64)
    stage = dllm.Stage(ctx, 0, 0)
    tree = ctx.draftTree([-1, 0, 0] * n, [3] * n)
    before = ctx.launch_count
    stage.commit_tree(tree, [[0, 2]] * n)
    ctx.synchronize()
    assert ctx.launch_count == before
    assert [stage.t0_of(s) for s in range(n)] == [2] * n
    stage.close()
    ctx.close()


def test_tree_refusals(dllm):
    ctx, other = make_ctx(dllm, max_seqs=2, max_pos=100), make_ctx(dllm)
    stage = dllm.Stage(ctx, 0, 1)
    E = dllm.DllmError
    for args in (([0], [1]), ([-1, 1], [2]), ([-1, 2, 0], [3]), ([-2], [1]), ([-1] * 65, [65]), ([], [0]), ([], []),
                 ([-1, -1], [1, 1], [4, 4]), ([-1], [1], [-1]), ([-1] * 129, [1] * 129)):
        with pytest.raises(E):
            ctx.draftTree(*args)
    tree, far, foreign = ctx.draftTree([-1, 0, 0]), ctx.draftTree([-1], [1], [2]), other.draftTree([-1])
    q, out, kv = ctx.createF32(3 * 256), ctx.createF32(3 * 256), ctx.createF32(3 * 128)
    for call in (lambda: stage.tree_attention(0, far, q, out), lambda: stage.tree_attention(0, foreign, q, out),
                 lambda: stage.tree_attention(1, tree, q, out), lambda: stage.tree_attention(0, tree, q, q),
                 lambda: stage.tree_attention(0, tree, kv, out), lambda: stage.tree_attention(0, tree, q, kv),
                 lambda: stage.tree_attention(0, tree, ctx.createBf16(3 * 256), out),
                 lambda: stage.append_tree(0, far, kv, kv), lambda: stage.append_tree(0, tree, kv, ctx.createF32(5)),
                 lambda: stage.append_tree(-1, tree, kv, kv),
                 lambda: stage.commit_tree(far, [[0]]), lambda: stage.commit_tree(tree, [[0], [0]]),
                 lambda: stage.commit_tree(tree, [[1]]), lambda: stage.commit_tree(tree, [[0, 0]]),
                 lambda: stage.commit_tree(tree, [[0, 1, 2]]), lambda: stage.commit_tree(tree, [[0, 3]]),
                 lambda: stage.commit_tree(tree, [[0, -1]]), lambda: stage.commit_tree(tree, [[0, 1, 2, 2]]),
                 lambda: stage.forward_tree(tree, q)):
        with pytest.raises(E):
            call()
    assert stage.T0 == 0
    stage.set_t0(0, 98)
    for call in (lambda: stage.tree_attention(0, tree, q, out), lambda: stage.append_tree(0, tree, kv, kv),
                 lambda: stage.commit_tree(tree, [[0]])):
        with pytest.raises(dllm.KvOverflowError):
            call()
    with pytest.raises(ValueError):
        stage.tree_attention(0, None, q, out)
    gone = ctx.draftTree([-1])
    gone.destroy()
    with pytest.raises(ValueError):
        stage.tree_attention(0, gone, q, out)
    stage.close()
    ctx.close()
    other.close()


def test_handles_of_another_kind_are_refused(dllm):
    """The C calls themselves, as a host without the Python checks makes them."""
    ctx = make_ctx(dllm)
    stage = dllm.Stage(ctx, 0, 1)
    lib = ctx.lib
    tree, plan = ctx.draftTree([-1, 0, 0]), ctx.ropePlan()
    b, pos = ctx.createF32(3 * 256), ctx.createI32(3)
    launches = ctx.launch_count
    for wrong in (tree.handle, plan.handle):
        assert lib.dllm_stage_set_weight(stage.handle, b"model.norm.weight", wrong) == 1
        assert lib.dllm_rope_at(ctx.handle, plan.handle, wrong, 3, b.handle, None, None, None) == 1
        assert lib.dllm_rope_at(ctx.handle, plan.handle, pos.handle, 3, wrong, None, None, None) == 1
        assert lib.dllm_stage_tree_attention(stage.handle, 0, tree.handle, wrong, b.handle) == 1
        assert lib.dllm_buf_bytes(wrong) == 0 and not lib.dllm_buf_device_ptr(wrong)
        lib.dllm_buf_free(wrong)
    for wrong in (b.handle, plan.handle):
        assert lib.dllm_stage_append_tree(stage.handle, 0, wrong, b.handle, b.handle) == 1
        assert lib.dllm_stage_tree_attention(stage.handle, 0, wrong, b.handle, b.handle) == 1
        assert lib.dllm_stage_forward_tree(stage.handle, wrong, b.handle, None, None) == 1
        lib.dllm_tree_destroy(wrong)
    for wrong in (b.handle, tree.handle):
        assert lib.dllm_rope_at(ctx.handle, wrong, pos.handle, 3, b.handle, None, None, None) == 1
        lib.dllm_rope_plan_destroy(wrong)
    assert ctx.launch_count == launches
    # all of them are as alive as before
    ctx.writeI32(pos, [0, 1, 1])
    ctx.ropeAt(plan, pos, 3, b)
    out = stage.tree_attention(0, tree, b)
    assert np.array_equal(ctx.readF32(out, out.n), np.zeros(out.n, np.float32))
    stage.close()
    ctx.close()


# ---- token picks -----------------------------------------------------------------------------------
def pick_reference(x, seq_of, hist, prompt, pen, bias, allowed, said):
    """The rules, each step rounded to fp32, and the picks. hist[s], bias[s]: lists; said[row]:
    drafted tokens of the row's path."""
    f = np.float32
    y = x.astype(f).copy()
    n, v = y.shape
    with np.errstate(all="ignore"):
        for r in range(n):
            s = seq_of[r]
            if pen is not None:
                h = [t for t in hist[s] if 0 <= t < v] if hist else []
                new = [t for t in (hist[s][prompt[s]:] if hist else []) if 0 <= t < v] + [t for t in said[r] if 0 <= t < v]
                for t in set(h) | set(new):
                    z = y[r, t] / f(pen[s][0]) if y[r, t] > 0 else y[r, t] * f(pen[s][0])
                    c = new.count(t)
                    if c:
                        z = (z - f(pen[s][1]) * f(c)) - f(pen[s][2])
                    y[r, t] = z
            if bias:
                last = {t: b for t, b in bias[s] if 0 <= t < v}
                for t, b in last.items():
                    y[r, t] = y[r, t] + f(b)
            if allowed is not None:
                y[r, ~allowed[r]] = -np.inf
    picks = []
    for r in range(n):
        ok = np.flatnonzero(allowed[r]) if allowed is not None else np.arange(v)
        z = np.where(np.isnan(y[r, ok]), -np.inf, y[r, ok])
        picks.append(int(ok[np.argmax(z)]) if ok.size else -1)
    return y, np.array(picks, np.int32)


def run_pick(ctx, x, seq_of, hist=None, prompt=None, pen=None, bias=None, allowed=None, tree=None, draft=None, said=None,
             inplace=False):
    n, v = x.shape
    lb = f32(ctx, x)
    kw = {}
    if hist is not None:
        flat = [t for h in hist for t in h]
        kw["history"] = (i32(ctx, flat or [0]), i32(ctx, np.concatenate([[0], np.cumsum([len(h) for h in hist])])),
                         i32(ctx, prompt))
    if pen is not None:
        kw["penalties"] = f32(ctx, pen)
    if bias is not None:
        flat = [e for b in bias for e in b] or [(-1, 0.0)]
        kw["bias"] = (i32(ctx, [t for t, _ in flat]), f32(ctx, [b for _, b in flat]),
                      i32(ctx, np.concatenate([[0], np.cumsum([len(b) for b in bias])])))
    if allowed is not None:
        words = -(-v // 32)
        bits = np.ones((n, words * 32), bool)  # bits behind the vocabulary are set: they allow nothing
        bits[:, :v] = allowed
        kw["mask"] = i32(ctx, np.packbits(bits, axis=1, bitorder="little").view(np.uint32))
    if tree is not None:
        kw["tree"], kw["draft"] = tree, i32(ctx, draft)
    out = lb if inplace else ctx.createF32(x.size)
    toks = ctx.readI32(ctx.pickTokens(lb, n, **kw))  # tokens only
    t2 = ctx.createI32(n)
    ctx.pickTokens(lb, n, out=out, tokens=t2, **kw)
    got = ctx.readF32(out, out.n).reshape(n, v)
    want, picks = pick_reference(x, seq_of, hist, prompt, pen, bias, allowed, said or [[]] * n)
    # every step is one rounded operation on both sides: equal to the bit
    assert np.array_equal(got, want, equal_nan=True)
    assert np.array_equal(toks, picks) and np.array_equal(ctx.readI32(t2), picks)


@pytest.mark.parametrize("v", [1, 31, 33, 127, 1000, 4099, 50257, 151936])
@pytest.mark.parametrize("use", ["plain", "penalties", "bias", "mask", "all"])
def test_pick_rows(dllm, v, use):
    ctx = make_ctx(dllm, vocab_size=v)
    rng = np.random.default_rng(v)
    n = 3
    x = (rng.standard_normal((n, v)) * 3).astype(np.float32)
    kw = {}
    if use in ("penalties", "all"):
        kw["hist"] = [list(rng.integers(-2, v + 2, k)) for k in (0, 40, 700)]
        kw["hist"][1] += [0, 0, v - 1, v - 1, v - 1]
        kw["prompt"] = [0, 20, 700]
        kw["pen"] = [[1.2, 0.3, 0.4], [0.7, -0.1, 0.25], [1.0, 0.5, 0.0]]
    if use in ("bias", "all"):
        kw["bias"] = [[(int(t), float(b)) for t, b in zip(rng.integers(-1, v + 1, k), rng.standard_normal(k) * 5)]
                      for k in (3, 0, 90)]
        kw["bias"][2] += [(0, 1.0), (0, 2.5)]
    if use in ("mask", "all"):
        kw["allowed"] = rng.random((n, v)) < 0.4
        kw["allowed"][1] = False
        kw["allowed"][2] = np.arange(v) == v - 1
    run_pick(ctx, x, range(n), **kw)
    run_pick(ctx, x, range(n), inplace=True, **kw)
    ctx.close()


def test_pick_ties_nan_and_infinities(dllm):
    v = 1003
    ctx = make_ctx(dllm, vocab_size=v)
    x = np.full((8, v), 1.0, np.float32)
    x[1] = np.nan
    x[2] = -np.inf
    x[3, ::7], x[3, 500], x[3, 900] = np.nan, np.inf, np.inf
    x[4] = np.finfo(np.float32).min
    x[5, 11], x[5, 1002] = 2.0, 2.0
    x[6, :200], x[6, 200:] = np.nan, -7.0
    x[7, :-1] = np.nan
    z = np.full((2, v), -1.0, np.float32)  # zeros of both signs tie
    z[0, 700], z[0, 5], z[1, 130], z[1, 131] = 0.0, -0.0, -0.0, 0.0
    run_pick(ctx, z, range(2))
    run_pick(ctx, x, range(8))
    allowed = np.ones((8, v), bool)
    allowed[:, :13] = False
    run_pick(ctx, x, range(8), allowed=allowed)
    hist = [[500, 3, 900, 900, 2 ** 31 - 1, -2 ** 31]] * 8
    run_pick(ctx, x, range(8), hist=hist, prompt=[1] * 8, pen=[[2.0, 0.5, 0.25]] * 8, allowed=allowed,
             bias=[[(900, float("-inf")), (20, float("nan"))]] * 8)
    ctx.close()


@pytest.mark.parametrize("v", [1000, 4099, 50257])
def test_pick_tree(dllm, v):
    """Nodes whose histories end with their own paths; repeated drafted tokens."""
    ctx = make_ctx(dllm, vocab_size=v)
    rng = np.random.default_rng(9)
    trees = [bushy(rng, 19), [], chain(33), [-1, 0, 0]]
    n = sum(map(len, trees))
    seq_of = [s for s, t in enumerate(trees) for _ in t]
    draft = rng.integers(0, 12, n)  # few tokens: a path meets the same one again and again
    draft[-1] = -7  # an id outside the vocabulary
    said, row0 = [], 0
    for t in trees:
        for see in ancestors(t):
            said.append([int(draft[row0 + j]) for j in np.flatnonzero(see)])
        row0 += len(t)
    x = (rng.standard_normal((n, v)) * 3).astype(np.float32)
    hist = [list(map(int, rng.integers(0, 40, k))) for k in (100, 3, 0, 17)]
    tree = ctx.draftTree([p for t in trees for p in t], [len(t) for t in trees])
    run_pick(ctx, x, seq_of, hist=hist, prompt=[50, 3, 0, 9], pen=[[1.3, 0.2, 0.1]] * 4, tree=tree, draft=draft, said=said,
             bias=[[(5, 1.5)], [], [(v - 1, 9.0)], []], allowed=rng.random((n, v)) < 0.7)
    # without a history the path alone counts
    run_pick(ctx, x, seq_of, pen=[[1.3, 0.2, 0.1]] * 4, tree=tree, draft=draft, said=said)
    ctx.close()


@pytest.mark.parametrize("v", [1000, 4099, 50257])
def test_pick_tree_whose_prompt_reaches_into_the_paths(dllm, v):
    """prompt_lens counts over the history and the path: every node equals a row of its own
    that has both as its history."""
    ctx = make_ctx(dllm, vocab_size=v)
    rng = np.random.default_rng(v)
    trees = [bushy(rng, 20), chain(64), [-1, 0, 0], bushy(rng, 11, roots=3), [-1, 0], chain(5)]
    hist = [list(map(int, rng.integers(0, 20, k))) for k in (30, 4, 0, 9, 7, 6)]
    prompt = [31, 40, 2, 11, 2 ** 31 - 1, 6]  # nodes of depth 0; 36 levels; two; two; all; none
    n = sum(map(len, trees))
    seq_of = [s for s, t in enumerate(trees) for _ in t]
    draft = rng.integers(0, 20, n)  # a path meets a token given and generated
    whole, row0 = [], 0
    for s, t in enumerate(trees):
        for see in ancestors(t):
            whole.append(hist[s] + [int(draft[row0 + j]) for j in np.flatnonzero(see)])
        row0 += len(t)
    x = (rng.standard_normal((n, v)) * 3).astype(np.float32)
    pen = np.array([[1.3, 0.2, 0.1], [0.8, 0.5, 0.0], [1.1, 0.0, 0.7], [1.2, -0.3, 0.4], [1.5, 0.6, 0.2], [1.3, 0.2, 0.1]])

    def pick(tokens, prompts, penalties, **kw):
        offsets = np.concatenate([[0], np.cumsum([len(t) for t in tokens])])
        out = ctx.createF32(x.size)
        got = ctx.pickTokens(f32(ctx, x), n, out=out, penalties=f32(ctx, penalties),
                             history=(i32(ctx, sum(tokens, [])), i32(ctx, offsets), i32(ctx, prompts)), **kw)
        return ctx.readI32(got), ctx.readF32(out, out.n)

    tree = ctx.draftTree([p for t in trees for p in t], [len(t) for t in trees])
    got = pick(hist, prompt, pen, tree=tree, draft=i32(ctx, draft))
    want = pick(whole, [prompt[s] for s in seq_of], pen[seq_of])
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
    ctx.close()


def test_pick_many_rows_and_a_vocabulary_beyond_one_chunk(dllm):
    """64 nodes share a history; 400003 tokens need several passes per slice."""
    ctx = make_ctx(dllm, vocab_size=400003, hidden_size=8)
    rng = np.random.default_rng(10)
    parents = bushy(rng, 9)
    draft = rng.integers(0, 400003, 9)
    said = [[int(draft[j]) for j in np.flatnonzero(see)] for see in ancestors(parents)]
    x = rng.standard_normal((9, 400003)).astype(np.float32)
    hist = [list(map(int, rng.integers(0, 400003, 5000)))]
    run_pick(ctx, x, [0] * 9, hist=hist, prompt=[100], pen=[[1.1, 0.2, 0.3]], tree=ctx.draftTree(parents), draft=draft,
             said=said, bias=[[(399999, 3.0)]])
    ctx.close()
    ctx = make_ctx(dllm, vocab_size=5003)
    parents = bushy(rng, 64)
    draft = rng.integers(0, 5003, 64)
    said = [[int(draft[j]) for j in np.flatnonzero(see)] for see in ancestors(parents)]
    x = rng.standard_normal((64, 5003)).astype(np.float32)
    run_pick(ctx, x, [0] * 64, hist=[list(map(int, rng.integers(0, 5003, 5000)))], prompt=[100], pen=[[1.1, 0.2, 0.3]],
             tree=ctx.draftTree(parents), draft=draft, said=said)
    ctx.close()


@pytest.mark.parametrize("v", [152064, 151937])
@pytest.mark.parametrize("use", ["plain", "penalties", "bias"])
def test_pick_slices_of_many_rows(dllm, v, use):
    """Enough rows that a slice is as large as its shared memory allows (or, without rules,
    the whole vocabulary)."""
    ctx = make_ctx(dllm, vocab_size=v)
    rng = np.random.default_rng(v)
    n = 300 if use == "plain" else 40
    x = rng.standard_normal((n, v), np.float32)
    kw = {}
    if use != "plain":
        kw["pen"] = [[1.2, 0.1, 0.3]] * n
        kw["hist"] = [list(map(int, rng.integers(0, v, 200))) + [v - 1, 0] for _ in range(n)]
        kw["prompt"] = [60] * n
    if use == "bias":
        kw["bias"] = [[(int(t), 2.0) for t in rng.integers(0, v, 20)] + [(v - 1, 1.0)] for _ in range(n)]
    run_pick(ctx, x, range(n), **kw)
    ctx.close()


def test_pick_clamps_offsets_outside_the_buffers(dllm):
    """Offsets come from the device: wild ones are clamped, never followed."""
    ctx = make_ctx(dllm, vocab_size=100)
    x = np.random.default_rng(1).standard_normal((2, 100)).astype(np.float32)
    t = ctx.pickTokens(f32(ctx, x), 2, history=(i32(ctx, [1, 2, 3]), i32(ctx, [-50, 2, 2 ** 30]), i32(ctx, [-1, 99])),
                       penalties=f32(ctx, [[1.5, 0.1, 0.1]] * 2),
                       bias=(i32(ctx, [4]), f32(ctx, [0.5]), i32(ctx, [9, -3, 7])))
    # sequence 0 has history [0, 2) and no bias, sequence 1 history [2, 3) and the entry
    _, want = pick_reference(x, [0, 1], [[1, 2], [3]], [0, 1], [[1.5, 0.1, 0.1]] * 2, [[], [(4, 0.5)]], None, [[], []])
    assert np.array_equal(ctx.readI32(t), want)
    ctx.close()


def test_pick_refusals(dllm):
    ctx, other = make_ctx(dllm, vocab_size=100), make_ctx(dllm, vocab_size=100)
    E = dllm.DllmError
    x, h, off2, pl, pen = ctx.createF32(200), ctx.createI32(5), ctx.createI32(3), ctx.createI32(2), ctx.createF32(6)
    vals, tree, dr = ctx.createF32(5), ctx.draftTree([-1, 0]), ctx.createI32(2)
    small = ctx.createI32(1)
    for args, kw in (((x, 0), {}), ((x, 3), {}), ((h, 2), {}), ((x, 2), dict(tokens=small)), ((x, 2), dict(out=pen)),
                     ((x, 2), dict(history=(h, off2, pl))), ((x, 2), dict(history=(h, pl, pl), penalties=pen)),
                     ((x, 2), dict(history=(h, off2, small), penalties=pen)), ((x, 2), dict(history=(None, off2, None))),
                     ((x, 2), dict(penalties=vals)), ((x, 2), dict(bias=(h, pen, off2), mask=x)),
                     ((x, 2), dict(bias=(h, ctx.createF32(4), off2))), ((x, 2), dict(bias=(h, vals, pl))),
                     ((x, 2), dict(bias=(None, vals, off2))), ((x, 2), dict(mask=off2)), ((x, 2), dict(tree=tree)),
                     ((x, 2), dict(draft=dr)), ((x, 1), dict(tree=tree, draft=dr)), ((x, 2), dict(tree=tree, draft=small)),
                     ((x, 2), dict(tree=other.draftTree([-1, 0]), draft=dr)), ((other.createF32(200), 2), {})):
        with pytest.raises(E):
            ctx.pickTokens(*args, **kw)
    with pytest.raises(E):
        ctx.createI32(0)
    # an output that other rows still read as their input
    mask, wide = ctx.createI32(2 * 4), ctx.createF32(200)
    offs = i32(ctx, [0, 0, 0, 0, 0])
    for kw in (dict(history=(h, offs, pl), penalties=pen, tokens=h), dict(history=(h, offs, pl), penalties=pen, tokens=offs),
               dict(history=(h, offs, pl), penalties=pen, tokens=pl), dict(bias=(h, vals, offs), tokens=h),
               dict(bias=(h, vals, offs), tokens=offs), dict(mask=mask, tokens=mask), dict(penalties=wide, out=wide),
               dict(bias=(h, wide, offs), out=wide)):
        with pytest.raises(E):
            ctx.pickTokens(x, 2, **kw)
    ctx.close()
    other.close()


def test_pick_over_its_inputs(dllm):
    """The tokens may replace the drafted ones, and the processed logits the logits."""
    ctx = make_ctx(dllm, vocab_size=10007)
    rng = np.random.default_rng(8)
    n, V = 21, 10007
    parents = [bushy(rng, 13), chain(7), [-1]]
    tree = ctx.draftTree([p for t in parents for p in t], [13, 7, 1])
    x, said = rng.standard_normal((n, V)).astype(np.float32), rng.integers(0, V, n)
    pen = f32(ctx, [[1.3, 0.2, 0.1]] * 3)
    out = ctx.createF32(n * V)
    want = ctx.readI32(ctx.pickTokens(f32(ctx, x), n, penalties=pen, tree=tree, draft=i32(ctx, said), out=out))
    processed = ctx.readF32(out, out.n)
    for _ in range(3):
        both, over = i32(ctx, said), f32(ctx, x)
        ctx.pickTokens(over, n, penalties=pen, tree=tree, draft=both, tokens=both, out=over)
        assert np.array_equal(ctx.readI32(both), want)
        assert np.array_equal(ctx.readF32(over, over.n), processed)
    ctx.close()


# ---- streams and graphs ---------------------------------------------------------------------------------
def test_on_a_side_stream_and_in_a_captured_graph(dllm):
    """The step's calls on a caller's stream, captured once and replayed on new inputs."""
    torch = torch_()
    P = Paged(dllm, 8, 2, 128, "bf16", [900, 40], [bushy(np.random.default_rng(1), 12), chain(3)])
    ctx, stage, tree = P.ctx, P.stage, P.tree
    s = torch.cuda.Stream()
    ctx.synchronize()
    ctx.set_stream(s.cuda_stream)
    rng = np.random.default_rng(2)
    n, V = 15, ctx.cfg.vocab_size
    plan = ctx.ropePlan(rotary_dim=64, scaling={"type": "yarn", "factor": 2.0, "original_max_pos": 512})
    q, k, v = (ctx.createF32(n * h * 128) for h in (8, 2, 2))
    qo, ko, out = ctx.createF32(q.n), ctx.createF32(k.n), ctx.createF32(q.n)
    pos, logits, lo = i32(ctx, np.arange(n) + 900), ctx.createF32(n * V), ctx.createF32(n * V)
    toks, draft, pen = ctx.createI32(n), i32(ctx, rng.integers(0, V, n)), f32(ctx, [[1.2, 0.1, 0.2]] * 2)

    def step():
        ctx.ropeAt(plan, pos, n, q, k, qo, ko)
        stage.append_tree(0, tree, ko, v)
        stage.tree_attention(0, tree, qo, out)
        ctx.pickTokens(logits, n, penalties=pen, tree=tree, draft=draft, out=lo, tokens=toks)

    def fill(seed):
        r = np.random.default_rng(seed)
        for b in (q, k, v, logits):
            ctx.writeF32(b, r.standard_normal(b.n).astype(np.float32))

    def result():
        ctx.synchronize()
        return [ctx.readF32(out, out.n), ctx.readF32(lo, lo.n), ctx.readI32(toks)]

    wants = []
    for seed in (5, 6):
        fill(seed)
        step()
        wants.append(result())
    assert not np.array_equal(wants[0][0], wants[1][0])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        step()
        for call in (lambda: ctx.draftTree([-1]), lambda: ctx.ropePlan(), lambda: stage.commit_tree(tree, [[0], []])):
            with pytest.raises(dllm.DllmError):
                call()
    assert [stage.t0_of(0), stage.t0_of(1)] == [900, 40]
    for seed, want in zip((5, 6, 5), wants + wants[:1]):
        fill(seed)
        with torch.cuda.stream(s):
            g.replay()
        for a, b in zip(result(), want):
            assert np.array_equal(a, b)
    del g
    P.close()


def test_host_copies_are_refused_in_a_capture(dllm):
    """A graph would keep the host's address: replays would read and write memory that the host
    has long given to something else. The capture itself stays good."""
    torch = torch_()
    ctx = make_ctx(dllm)
    s = torch.cuda.Stream()
    ctx.synchronize()
    ctx.set_stream(s.cuda_stream)
    ints, logits, toks = i32(ctx, [1, 2, 3]), f32(ctx, np.zeros(4096)), ctx.createI32(1)
    x = np.zeros(4096, np.float32)
    x[77] = 1.0
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        ctx.pickTokens(logits, 1, tokens=toks)
        for call in (lambda: ctx.writeI32(ints, [4, 5, 6]), lambda: ctx.readI32(ints), lambda: ctx.readF32(logits, 4)):
            with pytest.raises(dllm.DllmError, match="captured"):
                call()
    ctx.writeF32(logits, x)
    with torch.cuda.stream(s):
        g.replay()
    assert list(ctx.readI32(toks)) == [77]
    assert list(ctx.readI32(ints)) == [1, 2, 3]
    del g
    ctx.close()


def test_two_runs_give_the_same_bits(dllm):
    P = Paged(dllm, 14, 2, 64, "f32", [3000], [bushy(np.random.default_rng(1), 40)])
    q = f32(P.ctx, np.random.default_rng(2).standard_normal(40 * 14 * 64))
    first = P.ctx.readF32(P.stage.tree_attention(0, P.tree, q), q.n)
    for _ in range(5):
        assert np.array_equal(P.ctx.readF32(P.stage.tree_attention(0, P.tree, q), q.n), first)
    P.close()


# ---- all together ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("kv", ["f32", "bf16"])
def test_verify_tree_decodes_what_generate_decodes(dllm, weights_cache, kv):
    """Drafts that hold the true continuation among wrong branches, and drafts that are
    wrong: the tokens equal plain greedy decode, in fewer passes, and the cache holds the
    same rows."""
    cfg = oracle_cfg("tiny")
    W = get_weights(weights_cache, "tiny", cfg)
    prompt = synth.prompt_tokens(cfg, 7, seed=3)
    ctx, ld = build_leader(dllm, cfg, W, kv)
    want = []
    ld.onToken = want.append
    ld.generate(prompt, 30)
    assert len(want) == 30
    ref_kv = [ld.stage.kv[1].k.read(0, len(prompt) + 20), ld.stage.kv[0].v.read(0, len(prompt) + 20)]
    ctx2, ld2 = build_leader(dllm, cfg, W, kv)
    got = [ld2.generate(prompt, 1)]
    rng = np.random.default_rng(0)
    passes = 0
    while len(got) < 21:
        true = want[len(got):len(got) + 4]
        wrong = [int(t) for t in rng.integers(0, cfg.vocab_size, 6)]
        if passes % 3 == 2:  # a draft with nothing in it
            tree, draft = ctx2.draftTree([-1, 0, 0]), [got[-1], wrong[0], wrong[1]]
        else:  # 0 -> wrong, true0; true0 -> wrong, true1 -> wrong ...
            parents, draft, last = [-1], [got[-1]], 0
            for i, t in enumerate(true):
                parents += [last, last]
                draft += [wrong[i], t]
                last = len(parents) - 1
            tree = ctx2.draftTree(parents)
        new = ld2.verify_tree(tree, draft)[0]
        assert 1 <= len(new) <= 5
        got += new
        passes += 1
        assert ld2.stage.T0 == len(prompt) + len(got) - 1
    assert got == want[:len(got)]
    assert passes < 12
    n = len(prompt) + 20
    for a, b in zip(ref_kv, (ld2.stage.kv[1].k.read(0, n), ld2.stage.kv[0].v.read(0, n))):
        # hi + lo activations keep 16 bits, a bf16 cache rounds to 8: a row may land one step beside
        assert_close(b, a, rtol=2.0 ** -7 if kv == "bf16" else 1e-3, atol=2e-3, what="cache rows")
    # a plain decode continues from the committed cache
    assert ld2.decode(got[-1], 4) == want[len(got):len(got) + 4]
    for x in (ld, ld2):
        x.close()
    ctx.close()
    ctx2.close()


def test_verify_tree_under_rules_and_batches(dllm, weights_cache):
    """Two sequences in one pass; a mask that allows one token per node; penalties."""
    cfg = oracle_cfg("tiny")
    W = get_weights(weights_cache, "tiny", cfg)
    ctx, ld = build_leader(dllm, cfg, W, "f32", max_seqs=2)
    V = cfg.vocab_size
    tree = ctx.draftTree([-1, 0, 1, -1, 0], [3, 2])
    words = np.zeros((5, V // 32), np.uint32)
    for row, t in enumerate((11, 12, 13, 21, 22)):
        words[row, t // 32] |= np.uint32(1) << np.uint32(t % 32)
    new = ld.verify_tree(tree, [5, 11, 12, 6, 99], mask=i32(ctx, words), penalties=f32(ctx, [[1.1, 0.1, 0.1]] * 2))
    assert new == [[11, 12, 13], [21]]
    assert [ld.stage.t0_of(0), ld.stage.t0_of(1)] == [3, 1]
    words[:] = 0
    assert ld.verify_tree(tree, [13, 1, 2, 21, 3], mask=i32(ctx, words)) == [[-1], [-1]]
    with pytest.raises(dllm.DllmError):
        ld.verify_tree(tree, [1, 2, 3, 4, V])
    with pytest.raises(dllm.DllmError):
        ld.verify_tree(tree, [1, 2, 3, 4])
    ctx.set_tensor_core_rows(0)
    with pytest.raises(dllm.DllmError):
        ld.verify_tree(tree, [1, 2, 3, 4, 5])
    ld.close()
    ctx.close()


def test_verify_tree_under_penalties_picks_what_single_steps_pick(dllm, weights_cache):
    """A prompt, then drafted steps with a history: the tokens are those of one pick per token
    over the whole text. The first step's root is the prompt's last token, which was given: a
    bias makes it the pick unless it counted as generated."""
    cfg = oracle_cfg("tiny")
    W = get_weights(weights_cache, "tiny", cfg)
    prompt = [int(t) for t in synth.prompt_tokens(cfg, 9, seed=5)]
    rep, freq, pres = 1.25, 0.4, 0.3
    ctx, ld = build_leader(dllm, cfg, W, "f32")
    pen = f32(ctx, [[rep, freq, pres]])
    text, bias = list(prompt), None
    row = ld.forward(ld.embedTokens(prompt), len(prompt), 0)
    while len(text) < len(prompt) + 12:
        x = ld.sampleLast(row, return_logits=True)[1]
        if bias is None:
            y = x.astype(np.float64)
            seen = sorted(set(prompt))
            y[seen] = np.where(y[seen] > 0, y[seen] / rep, y[seen] * rep)
            lead = np.delete(y, prompt[-1]).max() - y[prompt[-1]]
            bias = (i32(ctx, [prompt[-1]]), f32(ctx, [lead + (freq + pres) / 2]), i32(ctx, [0, 1]))
        text.append(int(ctx.readI32(ctx.pickTokens(
            f32(ctx, x), 1, history=(i32(ctx, text), i32(ctx, [0, len(text)]), i32(ctx, [len(prompt)])), penalties=pen,
            bias=bias))[0]))
        row = ld.forward(ld.embedTokens(text[-1:]), 1, len(text) - 1)
    assert text[len(prompt)] == prompt[-1]
    ctx2, ld2 = build_leader(dllm, cfg, W, "f32")
    pen2, bias2 = f32(ctx2, [[rep, freq, pres]]), (i32(ctx2, [prompt[-1]]), f32(ctx2, ctx.readF32(bias[1], 1)), i32(ctx2, [0, 1]))
    ld2.forward(ld2.embedTokens(prompt[:-1]), len(prompt) - 1, 0)
    got = list(prompt)
    while len(got) < len(text):
        true = (text[len(got):len(got) + 3] + [1, 2, 3])[:3]
        tree = ctx2.draftTree([-1, 0, 0, 2, 3])
        new = ld2.verify_tree(tree, [got[-1], (true[0] + 1) % cfg.vocab_size] + true, penalties=pen2, bias=bias2,
                              history=(i32(ctx2, got[:-1]), i32(ctx2, [0, len(got) - 1]), i32(ctx2, [len(prompt)])))
        assert len(new) == 1 and len(new[0]) >= min(4, len(text) - len(got))
        got += new[0]
    assert got[:len(text)] == text
    for x in (ld, ld2):
        x.close()
    ctx.close()
    ctx2.close()


def test_verify_tree_into_buffers_of_the_caller(dllm, weights_cache):
    """`tokens` and `out` of pickTokens may be larger than the tree."""
    cfg = oracle_cfg("tiny")
    ctx, ld = build_leader(dllm, cfg, get_weights(weights_cache, "tiny", cfg), "f32")
    tree, draft = ctx.draftTree([-1, 0, 1]), [3, 4, 5]
    want = ld.verify_tree(tree, draft)
    ld.stage.reset()
    toks, out = ctx.createI32(7), ctx.createF32(5 * cfg.vocab_size)
    assert ld.verify_tree(tree, draft, tokens=toks, out=out) == want
    assert ld.stage.T0 == len(want[0])
    assert list(ctx.readI32(toks)[3:]) == [0] * 4
    ld.close()
    ctx.close()
