"""The operators of long conversations, as cases to measure.

A host with layers of its own normalises and rotates its queries and keys head by head
("norm"), keeps their K/V rows in a cache of 4-bit codes ("quant"), and attends over that
cache ("code") or over a stage's own one ("window"): one new token per sequence, whole
chunks of a prompt, or both in one batch, with a sliding window and the first few tokens
kept visible where the model was trained so.

`run` computes them in plain torch (own = False) or through the framework (own = True).
"""
import functools
import importlib
import math

import numpy as np
import torch

own = False

HEADS = {  # query heads, KV heads, head size of the framework's model presets
    "0.5b": (14, 2, 64),
    "1.5b": (12, 2, 128),
    "7b": (28, 4, 128),
    "32b": (40, 8, 128),
}
PAGE = 64
GROUP = 32  # dims that share a scale and a minimum
THETA = 1e6
EPS = 1e-6


# ---- cases -----------------------------------------------------------------------------
def listed():
    return [
        # one decode row of the smallest preset: what a token costs when nothing hides the latency
        {"name": "norm one row", "op": "norm", "dims": "0.5b", "rows": 1, "layout": "half", "rotary": 64, "far": 2048},
        # a long chunk of a prompt
        {"name": "norm prefill 6007", "op": "norm", "dims": "7b", "rows": 6007, "layout": "half", "rotary": 128, "far": 32768},
        # the K/V rows of one new token for each of a few sequences
        {"name": "quant 5 tokens", "op": "quant", "dims": "1.5b", "seqs": 5, "rows": 1, "mixed": False, "t0": 1900},
        # the K/V rows of a long chunk of a prompt
        {"name": "quant prefill 8185", "op": "quant", "dims": "7b", "seqs": 1, "rows": 8185, "mixed": False, "t0": 100},
        # a decode step far into a conversation whose model sees 4096 tokens and the first four
        {"name": "window one row", "op": "window", "dims": "7b", "seqs": 1, "rows": 1, "mixed": False, "t0": 31999,
         "kv": "bf16", "window": 4096, "sinks": 4},
        # decode steps of a batch on the default fp32 cache, everything visible
        {"name": "window batch fp32", "op": "window", "dims": "1.5b", "seqs": 24, "rows": 1, "mixed": False, "t0": 4001,
         "kv": "f32", "window": 0, "sinks": 0},
        # a chunk of a long prompt under the same window
        {"name": "window chunk 2048", "op": "window", "dims": "7b", "seqs": 1, "rows": 2048, "mixed": False, "t0": 6100,
         "kv": "bf16", "window": 4096, "sinks": 4},
        # a short prompt from its first token on an fp32 cache
        {"name": "window prompt fp32", "op": "window", "dims": "0.5b", "seqs": 1, "rows": 1501, "mixed": False, "t0": 0,
         "kv": "f32", "window": 0, "sinks": 0},
        # one decode row over a long context in codes
        {"name": "code one row", "op": "code", "dims": "7b", "seqs": 1, "rows": 1, "mixed": False, "t0": 32000, "window": 0,
         "sinks": 0},
        # decode steps of a large batch
        {"name": "code batch 64", "op": "code", "dims": "1.5b", "seqs": 64, "rows": 1, "mixed": False, "t0": 8000, "window": 0,
         "sinks": 0},
        # a chunk of one prompt in a batch with decode steps of other sequences
        {"name": "code mixed", "op": "code", "dims": "1.5b", "seqs": 16, "rows": 700, "mixed": True, "t0": 5003, "window": 2000,
         "sinks": 16},
        # a chunk of a long prompt, everything visible
        {"name": "code chunk 2048", "op": "code", "dims": "7b", "seqs": 1, "rows": 2048, "mixed": False, "t0": 6100, "window": 0,
         "sinks": 0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("norm", "quant", "window", "window", "code", "code"))
    dims = rng.choice(tuple(HEADS))
    if op == "norm":
        return {"op": op, "dims": rng.choice(("0.5b", "1.5b", "7b")), "rows": _log(rng, 1, 6000),
                "layout": rng.choice(("half", "interleaved")), "rotary": 2 * rng.randint(2, 32), "far": _log(rng, 10, 1000000)}
    if op == "quant":
        seqs = _log(rng, 1, 64)
        return {"op": op, "dims": rng.choice(("0.5b", "1.5b", "7b")), "seqs": seqs, "rows": _log(rng, 1, 8000 // seqs),
                "mixed": rng.random() < 0.3, "t0": rng.randint(0, 300)}
    t0 = _log(rng, 1, 30000)
    seqs = _log(rng, 1, max(1, min(64, 200000 // t0)))
    # decode steps, or a chunk of a prompt: what its rows could see, times the heads, is bounded
    most = 4.5e8 / (HEADS[dims][0] * seqs)
    rows = 1 if rng.random() < 0.4 else _log(rng, 1, max(1, min(2000, int(((t0 * t0 + 4 * most) ** 0.5 - t0) / 2))))
    case = {"op": op, "dims": dims, "seqs": seqs, "rows": rows, "mixed": rows > 1 and rng.random() < 0.4, "t0": t0 - 1,
            "window": 0 if rng.random() < 0.4 else _log(rng, 1, 8000), "sinks": rng.choice((0, 1, 4, rng.randint(0, 200)))}
    if op == "window":
        case["kv"] = rng.choice(("bf16", "f32"))
    return case


# ---- shapes that follow from a case ------------------------------------------------------
def _counts(case):
    """Rows of each sequence: the same for all, or a chunk of the first and one row of the others."""
    b, m = case["seqs"], case["rows"]
    return [m] + [1 if case["mixed"] else m] * (b - 1)


def _lens(case):
    """Cached slots of each sequence before its rows: the first has t0, the last about half as many."""
    b = case["seqs"]
    return [case["t0"] - (case["t0"] * i) // (2 * b) for i in range(b)]


def _max_pos(case):
    return case["t0"] + case["rows"]


@functools.lru_cache(maxsize=4)
def _ctx(preset, overrides):
    dllm = importlib.import_module("distributed-llm1_b200")
    ctx = dllm.initKernels(0, dllm.PRESETS["qwen2.5-" + preset].with_(**dict(overrides)))
    ctx.set_stream(1)  # CUDA's handle of the legacy default stream, the one torch uses unless told otherwise
    return dllm, ctx


def _buf(ctx, t):
    """A device buffer of the framework with a tensor's values, and the tensor that shares its memory."""
    b = {torch.int32: ctx.createI32, torch.bfloat16: ctx.createBf16}.get(t.dtype, ctx.createF32)(t.numel())
    v = torch.as_tensor(b, device="cuda")
    v = (v.view(torch.bfloat16) if t.dtype == torch.bfloat16 else v).view(t.shape)
    v.copy_(t)
    return b, v


# ---- inputs --------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    h = np.random.default_rng(seed)
    s = {"case": case, "op": case["op"]}
    if own:
        over = {"num_layers": 1}
        if case["op"] != "norm":
            over.update(max_pos=_max_pos(case), max_seqs=case["seqs"], kv_dtype=case.get("kv", "bf16"), kv_page_size=PAGE)
        s["dllm"], s["ctx"] = _ctx(case["dims"], tuple(sorted(over.items())))
    {"norm": _prepare_norm, "quant": _prepare_quant, "window": _prepare_window, "code": _prepare_code}[case["op"]](s, case, g, h)
    return s


def _prepare_norm(s, case, g, h):
    nq, kvh, hd = HEADS[case["dims"]]
    n, r = case["rows"], case["rotary"]
    s["q"] = torch.randn(n, nq, hd, device="cuda", generator=g) * 3.0
    s["k"] = torch.randn(n, kvh, hd, device="cuda", generator=g) * 5.0
    s["q_norm"] = (1.0 + 0.3 * torch.randn(hd, device="cuda", generator=g)).bfloat16()
    s["k_norm"] = (1.0 + 0.3 * torch.randn(hd, device="cuda", generator=g)).bfloat16()
    s["pos"] = torch.randint(0, case["far"], (n,), device="cuda", generator=g, dtype=torch.int32)
    s["inv_freq"] = torch.from_numpy(THETA ** (-2 * np.arange(r // 2, dtype=np.float64) / r)).cuda()
    if own:
        ctx = s["ctx"]
        s["plan"] = ctx.ropePlan(layout=case["layout"], rotary_dim=r, theta=THETA)
        for k in ("q", "k", "q_norm", "k_norm", "pos"):
            s[k + "_buf"], s[k] = _buf(ctx, s[k])
        for k in ("q", "k"):
            s[k + "_out"], s[k + "_res"] = _buf(ctx, torch.zeros_like(s[k]))


def _batch(s, case, h):
    """Where each row of the batch lies, and a shuffled page table."""
    b = case["seqs"]
    counts, lens = _counts(case), _lens(case)
    s["counts"], s["lens"] = counts, lens
    s["n"] = sum(counts)
    per = -(-_max_pos(case) // PAGE)
    s["pages"] = h.permutation(b * per).astype(np.int32).reshape(b, per)
    s["table"] = torch.from_numpy(s["pages"]).cuda().long()
    s["seq"] = torch.from_numpy(np.repeat(np.arange(b), counts)).cuda()
    s["row"] = torch.from_numpy(np.concatenate([np.arange(c) for c in counts])).cuda()
    s["t0"] = torch.tensor(lens, device="cuda")
    s["slot"] = s["t0"][s["seq"]] + s["row"]


def _channels(g, kvh, hd):
    """What K's channels are offset by: keys sit around a bias, and a few channels far from zero."""
    off = torch.randn(kvh, hd, device="cuda", generator=g)
    return torch.where(torch.rand(kvh, hd, device="cuda", generator=g) < 0.05, off * 8.0, off * 0.5)


def _prepare_quant(s, case, g, h):
    nq, kvh, hd = HEADS[case["dims"]]
    _batch(s, case, h)
    s["k"] = torch.randn(s["n"], kvh, hd, device="cuda", generator=g) + _channels(g, kvh, hd)
    s["v"] = torch.randn(s["n"], kvh, hd, device="cuda", generator=g)
    per = s["pages"].size
    if own:
        ctx = s["ctx"]
        cache = s["cache"] = s["dllm"].Cache4(ctx, 0, 1)
        for i, t0 in enumerate(s["lens"]):
            cache.set_page_table(i, s["pages"][i])
            cache.set_t0(i, t0)
        s["rows"] = ctx.rowBatch(s["counts"])
        for k in ("k", "v"):
            s[k + "_buf"], s[k] = _buf(ctx, s[k])
            s[k + "_out"], s[k + "_res"] = _buf(ctx, torch.zeros_like(s[k]))
    else:
        for k in ("k", "v"):
            s[k + "_codes"] = torch.zeros(per, kvh, PAGE, hd // 2, dtype=torch.uint8, device="cuda")
            s[k + "_scales"] = torch.zeros(per, kvh, PAGE, hd // GROUP, 2, dtype=torch.bfloat16, device="cuda")


def _context(s, case, g):
    """K and V [pages, KV heads, page, head size] fp32 of all slots, in their pages."""
    nq, kvh, hd = HEADS[case["dims"]]
    shape = (s["pages"].size, kvh, PAGE, hd)
    k = torch.randn(shape, device="cuda", generator=g)
    k += _channels(g, kvh, hd)[:, None, :]
    return k, torch.randn(shape, device="cuda", generator=g)


def _prepare_window(s, case, g, h):
    nq, kvh, hd = HEADS[case["dims"]]
    _batch(s, case, h)
    s["q"] = torch.randn(s["n"], nq, hd, device="cuda", generator=g) * 1.5
    dt = torch.bfloat16 if case["kv"] == "bf16" else torch.float32
    s["k"], s["v"] = (x.to(dt) for x in _context(s, case, g))
    if own:
        ctx = s["ctx"]
        stage = s["stage"] = s["dllm"].Stage(ctx, 0, 1)
        for which in ("k", "v"):
            pool = torch.as_tensor(stage.kv_pool(which), device="cuda")
            pool = pool.view(dt).view(s[which].shape)
            pool.copy_(s[which])
            s[which] = pool
        for i, t0 in enumerate(s["lens"]):
            stage.set_page_table(i, s["pages"][i])
            stage.set_t0(i, t0)
        s["rows"] = ctx.rowBatch(s["counts"])
        s["q_buf"], s["q"] = _buf(ctx, s["q"])
        s["out_buf"], s["out"] = _buf(ctx, torch.zeros_like(s["q"]))


def _prepare_code(s, case, g, h):
    nq, kvh, hd = HEADS[case["dims"]]
    _batch(s, case, h)
    s["q"] = torch.randn(s["n"], nq, hd, device="cuda", generator=g) * 1.5
    k, v = _context(s, case, g)
    if own:
        ctx = s["ctx"]
        cache = s["cache"] = s["dllm"].Cache4(ctx, 0, 1)
        for i, (t0, c) in enumerate(zip(s["lens"], s["counts"])):
            cache.set_page_table(i, s["pages"][i])
            at = torch.arange(t0 + c, device="cuda")
            page = s["table"][i][at // PAGE]
            bufs = [_buf(ctx, x[page, :, at % PAGE].contiguous())[0] for x in (k, v)]
            cache.append(0, ctx.rowBatch([t0 + c], [i]), *bufs)
            cache.set_t0(i, t0)
        s["rows"] = ctx.rowBatch(s["counts"])
        s["q_buf"], s["q"] = _buf(ctx, s["q"])
        s["out_buf"], s["out"] = _buf(ctx, torch.zeros_like(s["q"]))
    else:
        for name, x in (("k", k), ("v", v)):
            s[name + "_codes"], s[name + "_scales"] = _quantise(x)


# ---- the operators ---------------------------------------------------------------------------
def run(state):
    if own:
        return {"norm": _own_norm, "quant": _own_quant, "window": _own_window, "code": _own_code}[state["op"]](state)
    return {"norm": _norm, "quant": _quant, "window": _window, "code": _code}[state["op"]](state)


def _own_norm(s):
    s["ctx"].normRopeAt(s["plan"], s["pos_buf"], s["case"]["rows"], s["q_buf"], s["k_buf"], s["q_norm_buf"], s["k_norm_buf"],
                        s["q_out"], s["k_out"])
    return s["q_res"], s["k_res"]


def _own_quant(s):
    s["cache"].append(0, s["rows"], s["k_buf"], s["v_buf"])
    s["cache"].read_rows(0, s["rows"], s["k_out"], s["v_out"])
    return s["k_res"], s["v_res"]


def _own_window(s):
    s["stage"].window_attention(0, s["rows"], s["q_buf"], s["out_buf"], window=s["case"]["window"], sinks=s["case"]["sinks"])
    return s["out"]


def _own_code(s):
    s["cache"].attention(0, s["rows"], s["q_buf"], s["out_buf"], window=s["case"]["window"], sinks=s["case"]["sinks"])
    return s["out"]


def _norm(s):
    """Each head divided by its root mean square, scaled by the norm's weights, then the
    pairs (x1, x2) of its first `rotary` dims turned by position * inv_freq."""
    r, half = s["case"]["rotary"], s["case"]["layout"] == "half"
    angle = s["pos"].double()[:, None] * s["inv_freq"]
    cos, sin = torch.cos(angle).float()[:, None, :], torch.sin(angle).float()[:, None, :]
    return tuple(_turned(x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float(), cos, sin, r, half)
                 for x, w in ((s["q"], s["q_norm"]), (s["k"], s["k_norm"])))


def _turned(x, cos, sin, r, half):
    a, b = (x[..., : r // 2], x[..., r // 2 : r]) if half else (x[..., 0:r:2], x[..., 1:r:2])
    a, b = a * cos - b * sin, a * sin + b * cos
    turned = torch.cat([a, b], -1) if half else torch.stack([a, b], -1).flatten(-2)
    return torch.cat([turned, x[..., r:]], -1)


def _to_bf16_down(x):
    """fp32 -> the largest bf16 that is not above it (as fp32)."""
    bits = x.view(torch.int32)
    bits = torch.where(x < 0, bits + 0xFFFF, bits) & -0x10000
    return bits.view(torch.float32)


def _quantise(x):
    """Codes (two per byte, the even dim in the low half) and (scale, minimum) of groups of 32
    dims: the minimum rounded down to bf16, scale = (largest - minimum) / 15 rounded up to
    bf16, code = (x - minimum) / scale to the nearest whole number, ties to even."""
    z = x.view(*x.shape[:-1], -1, GROUP)
    low = _to_bf16_down(z.amin(-1, keepdim=True))
    scale = -_to_bf16_down(-((z.amax(-1, keepdim=True) - low).double() / 15.0).float())
    step = torch.where(scale > 0, scale, torch.ones_like(scale)).double()
    code = torch.round((z - low).double() / step).clamp_(0, 15).to(torch.uint8).view(x.shape)
    scales = torch.cat([scale, low], -1).bfloat16()
    return code[..., 0::2] | (code[..., 1::2] << 4), scales


def _values(codes, scales):
    """The fp32 values that codes stand for: minimum + code * scale."""
    c = torch.stack([codes & 15, codes >> 4], -1).float().view(*codes.shape[:-1], -1, GROUP)
    scales = scales.float()
    return (c * scales[..., 0:1] + scales[..., 1:2]).flatten(-2)


def _quant(s):
    page, off = s["table"][s["seq"], s["slot"] // PAGE], s["slot"] % PAGE
    out = []
    for k in ("k", "v"):
        codes, scales = _quantise(s[k])
        s[k + "_codes"][page, :, off] = codes
        s[k + "_scales"][page, :, off] = scales
        out.append(_values(s[k + "_codes"][page, :, off], s[k + "_scales"][page, :, off]))
    return tuple(out)


def _slots(s, x):
    """A paged tensor [pages, KV heads, page, ...] as [sequences, KV heads, slots, ...]."""
    y = x[s["table"]].transpose(1, 2)
    return y.reshape(y.shape[0], y.shape[1], -1, *y.shape[4:])


def _attend(s, k, v):
    """Every row over the slots up to its own that the window or the sinks show it."""
    case = s["case"]
    nq, kvh, hd = HEADS[case["dims"]]
    b, m = case["seqs"], max(s["counts"])
    q = torch.zeros(b, m, nq, hd, device="cuda")
    q[s["seq"], s["row"]] = s["q"]
    q = q.view(b, m, kvh, nq // kvh, hd).permute(0, 2, 1, 3, 4).reshape(b, kvh, -1, hd)
    score = (q @ k.transpose(-1, -2)).view(b, kvh, m, nq // kvh, -1) * (1.0 / math.sqrt(hd))
    at = torch.arange(k.shape[2], device="cuda")
    slot = s["t0"][:, None] + torch.arange(m, device="cuda")
    see = at <= slot[..., None]
    if case["window"]:
        see &= (at > slot[..., None] - case["window"]) | (at < case["sinks"])
    score = torch.where(see[:, None, :, None], score, float("-inf"))
    p = torch.exp(score - score.amax(-1, keepdim=True))
    out = (p.view(b, kvh, -1, p.shape[-1]) @ v).view(b, kvh, m, -1, hd) / p.sum(-1, keepdim=True)
    return out.permute(0, 2, 1, 3, 4).reshape(b, m, nq, hd)[s["seq"], s["row"]]


def _window(s):
    return _attend(s, _slots(s, s["k"]).float(), _slots(s, s["v"]).float())


def _code(s):
    return _attend(s, *(_values(_slots(s, s[k + "_codes"]), _slots(s, s[k + "_scales"])) for k in ("k", "v")))


# ---- what a pass cannot do without ---------------------------------------------------------------
def _seen(case):
    """(row, slot) pairs that are visible, and cached slots that some row of their sequence sees."""
    pairs = slots = 0
    for t0, c in zip(_lens(case), _counts(case)):
        at = np.arange(t0, t0 + c)
        if not case["window"]:
            pairs, slots = pairs + int((at + 1).sum()), slots + t0 + c
            continue
        first = np.maximum(0, at + 1 - case["window"])
        pairs += int((at + 1 - first + np.minimum(first, case["sinks"])).sum())
        slots += t0 + c - int(first[0]) + min(int(first[0]), case["sinks"])
    return pairs, slots


def work(case):
    nq, kvh, hd = HEADS[case["dims"]]
    if case["op"] == "norm":
        n = case["rows"]
        return {"bytes": 2 * 4 * n * (nq + kvh) * hd + 4 * n + 4 * hd, "flops": n * (nq + kvh) * (4 * hd + 3 * case["rotary"])}
    rows = sum(_counts(case))
    row = {"f32": 4 * hd, "bf16": 2 * hd}.get(case.get("kv"), hd // 2 + 4 * hd // GROUP)  # bytes of one head's K or V row
    if case["op"] == "quant":
        return {"bytes": 2 * rows * kvh * (8 * hd + row), "flops": 2 * 6 * rows * kvh * hd}
    pairs, slots = _seen(case)
    return {"bytes": 2 * slots * kvh * row + 2 * 4 * rows * nq * hd, "flops": 4 * pairs * nq * hd}


# ---- the definitions in 64 bits ------------------------------------------------------------------
def exact(case, seed):
    global own
    mine, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = mine
    return {"norm": _exact_norm, "quant": _exact_quant, "window": _exact_window, "code": _exact_code}[case["op"]](s, case)


def _exact_norm(s, case):
    r = case["rotary"]
    turn = torch.exp(1j * (s["pos"].double()[:, None] * s["inv_freq"]))[:, None, :]
    out = []
    for x, w in ((s["q"], s["q_norm"]), (s["k"], s["k_norm"])):
        x = x.double()
        y = x * w.double() / ((x ** 2).sum(-1, keepdim=True) / x.shape[-1] + EPS) ** 0.5
        if case["layout"] == "half":
            z = torch.complex(y[..., : r // 2], y[..., r // 2 : r]) * turn
            y[..., : r // 2], y[..., r // 2 : r] = z.real, z.imag
        else:
            z = torch.complex(y[..., 0:r:2], y[..., 1:r:2]) * turn
            y[..., 0:r:2], y[..., 1:r:2] = z.real, z.imag
        out.append(y)
    return tuple(out)


def _floor8(x):
    """The largest number of 8 significant bits that is not above x (64 bits)."""
    mantissa = torch.frexp(x.abs()).mantissa  # in [1/2, 1)
    step = torch.where(x == 0, 1.0, x.abs() / mantissa / 256)
    return torch.floor(x / step) * step


def _exact_quant(s, case):
    out = []
    for x in (s["k"], s["v"]):
        z = x.unflatten(-1, (-1, GROUP))
        low = _floor8(z.min(-1, keepdim=True).values.double()).float()  # differences are taken in 32 bits
        scale = -_floor8(-((z.max(-1, keepdim=True).values - low).double() / 15.0).float().double())
        code = ((z - low).double() / scale).round().clamp(0, 15)
        out.append((low.double() + code * scale).flatten(-2))
    return tuple(out)


def _exact_attend(s, case, head_of):
    """head_of(x, sequence, KV head) -> [slots, head size] in 64 bits."""
    nq, kvh, hd = HEADS[case["dims"]]
    group = nq // kvh
    if 4.0 * nq * hd * _seen(case)[0] > 5e12 or 4.0 * nq * hd * sum(c * t for c, t in zip(_counts(case), _lens(case))) > 1e13:
        return None
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    row0 = 0
    for i, (t0, c) in enumerate(zip(s["lens"], s["counts"])):
        for head in range(kvh):
            k, v = (head_of(x, i, head)[: t0 + c] for x in ("k", "v"))
            for j in range(0, c, 256):
                e = min(c, j + 256)
                rows = s["q"][row0 + j : row0 + e, head * group : (head + 1) * group].double()
                last = torch.arange(t0 + j, t0 + e, device="cuda")[:, None]
                at = torch.arange(t0 + e, device="cuda")[None]
                hidden = at > last
                if case["window"]:
                    hidden = hidden | ((last - at >= case["window"]) & (at >= case["sinks"]))
                z = torch.einsum("rgd,td->rgt", rows, k[: t0 + e]) / hd ** 0.5
                p = torch.softmax(z.masked_fill(hidden[:, None], -math.inf), -1)
                out[row0 + j : row0 + e, head * group : (head + 1) * group] = torch.einsum("rgt,td->rgd", p, v[: t0 + e])
        row0 += c
    return out


def _exact_window(s, case):
    return _exact_attend(s, case, lambda x, i, head: s[x][s["table"][i], head].flatten(0, 1).double())


def _exact_code(s, case):
    def head_of(x, i, head):
        codes = s[x + "_codes"][s["table"][i], head].flatten(0, 1)
        scales = s[x + "_scales"][s["table"][i], head].flatten(0, 1).double().repeat_interleave(GROUP, 1)
        both = torch.empty(codes.shape[0], codes.shape[1] * 2, dtype=torch.float64, device="cuda")
        both[:, 0::2], both[:, 1::2] = codes % 16, codes // 16
        return scales[..., 1] + both * scales[..., 0]
    return _exact_attend(s, case, head_of)
