"""The operators of one verification step of drafted tokens, as cases to measure.

A draft proposes a tree of tokens for each sequence; the model scores all of them in
one pass. That pass rotates q and k at the nodes' positions ("rope"), attends from
every node to the cached context and to the node's own ancestors ("tree"), picks one
token per node from its logits under penalties, biases and a grammar mask ("pick"),
and moves the K/V rows of the accepted path to the front of the drafted slots
("commit").

`run` computes them in plain torch (own = False) or through the framework (own = True).
"""
import functools
import importlib
import math

import numpy as np
import torch

own = False

HEADS = {  # query heads, KV heads, head size, vocabulary, layers of the framework's model presets
    "0.5b": (14, 2, 64, 151936, 24),
    "1.5b": (12, 2, 128, 151936, 28),
    "7b": (28, 4, 128, 152064, 28),
    "32b": (40, 8, 128, 152064, 64),
}
PAGE = 64
THETA = 1e6
YARN = {"type": "yarn", "factor": 4.0, "original_max_pos": 32768}


# ---- cases -----------------------------------------------------------------------------
def listed():
    return [
        # one decode row of the smallest preset: what a token costs when nothing hides the latency
        {"name": "rope one row", "op": "rope", "dims": "0.5b", "rows": 1, "layout": "half", "rotary": 64, "scaling": "none",
         "far": 2048},
        # a 64-node tree far into a context that was stretched by YaRN
        {"name": "rope tree 64 yarn", "op": "rope", "dims": "7b", "rows": 64, "layout": "half", "rotary": 128,
         "scaling": "yarn", "far": 131072},
        # a long prefill of a partly rotated, interleaved layout
        {"name": "rope prefill 8191", "op": "rope", "dims": "7b", "rows": 8191, "layout": "interleaved", "rotary": 96,
         "scaling": "linear", "far": 32768},
        # one node: an ordinary decode step over the benchmark's 2048-slot cache
        {"name": "tree 1 at 2k", "op": "tree", "dims": "7b", "seqs": 1, "nodes": 1, "t0": 2047, "kv": "bf16"},
        # a small draft, as a lookup of the prompt's own n-grams gives
        {"name": "tree 13 at 8k", "op": "tree", "dims": "1.5b", "seqs": 1, "nodes": 13, "t0": 8191, "kv": "bf16"},
        # the widest tree over a long context
        {"name": "tree 64 at 32k", "op": "tree", "dims": "7b", "seqs": 1, "nodes": 64, "t0": 32000, "kv": "bf16"},
        # a batch of sequences of unequal lengths on the default fp32 cache
        {"name": "tree 8x7 fp32", "op": "tree", "dims": "1.5b", "seqs": 8, "nodes": 7, "t0": 4001, "kv": "f32"},
        # greedy decode of one sequence: only the token is wanted
        {"name": "pick one row", "op": "pick", "vocab": 151936, "seqs": 1, "nodes": 0, "history": 1500, "bias": 0,
         "mask": False, "keep": False},
        # sixteen sequences under a grammar, odd vocabulary, logits kept for a sampler
        {"name": "pick 16 masked", "op": "pick", "vocab": 50257, "seqs": 16, "nodes": 0, "history": 700, "bias": 40,
         "mask": True, "keep": True},
        # every node of a 64-node tree, each with a history and a grammar state of its own
        {"name": "pick tree 64", "op": "pick", "vocab": 152064, "seqs": 1, "nodes": 64, "history": 32000, "bias": 300,
         "mask": True, "keep": True},
        # one sequence after a small draft
        {"name": "commit 1x4", "op": "commit", "dims": "7b", "seqs": 1, "nodes": 16, "t0": 1000, "take": 4, "kv": "bf16"},
        # a batch, every layer of the largest preset
        {"name": "commit 16x9", "op": "commit", "dims": "32b", "seqs": 16, "nodes": 48, "t0": 150, "take": 9, "kv": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("rope", "tree", "tree", "pick", "pick", "commit"))
    dims = rng.choice(tuple(HEADS))
    if op == "rope":
        return {"op": op, "dims": rng.choice(("0.5b", "1.5b", "7b")), "rows": _log(rng, 1, 8000),
                "layout": rng.choice(("half", "interleaved")), "rotary": 2 * rng.randint(2, 32),
                "scaling": rng.choice(("none", "linear", "ntk", "yarn")), "far": _log(rng, 10, 1000000)}
    if op == "tree":
        t0 = _log(rng, 1, 30000)
        seqs = _log(rng, 1, max(1, min(24, 60000 // t0)))
        return {"op": op, "dims": dims if t0 * seqs < 16000 else "1.5b", "seqs": seqs, "nodes": _log(rng, 1, 64), "t0": t0,
                "kv": rng.choice(("bf16", "f32"))}
    if op == "pick":
        tree = rng.random() < 0.5
        return {"op": op, "vocab": _log(rng, 1000, 152064), "seqs": _log(rng, 1, 4 if tree else 60),
                "nodes": _log(rng, 1, 16) if tree else 0, "history": _log(rng, 1, 20000), "bias": rng.choice((0, 1, 77, 300)),
                "mask": rng.random() < 0.6, "keep": rng.random() < 0.6}
    nodes = rng.randint(2, 64)
    return {"op": op, "dims": rng.choice(("0.5b", "1.5b", "7b")), "seqs": rng.randint(1, 16), "nodes": nodes,
            "t0": rng.randint(0, 190), "take": rng.randint(1, nodes), "kv": rng.choice(("bf16", "f32"))}


# ---- shapes that follow from a case ------------------------------------------------------
def _lens(case):
    """Cached slots of each sequence: the first has t0, the last about half as many."""
    b = case["seqs"]
    return [max(0, case["t0"] - (case["t0"] * i) // (2 * b)) for i in range(b)]


def _max_pos(case):
    return case["t0"] + max(1, case["nodes"])


def _model(case):
    """(presets name, overrides) of the framework's configuration of a case."""
    if case["op"] == "pick":
        return "1.5b", {"vocab_size": case["vocab"], "num_layers": 1}
    if case["op"] == "rope":
        return case["dims"], {"num_layers": 1}
    layers = HEADS[case["dims"]][4] if case["op"] == "commit" else 1
    return case["dims"], {"num_layers": layers, "max_pos": _max_pos(case), "max_seqs": case["seqs"], "kv_dtype": case["kv"],
                          "kv_page_size": PAGE}


def _parents(g, nodes, take=1):
    """Parents of one drafted tree: a root, an accepted path through `take` nodes, the rest anywhere."""
    path = np.zeros(0, np.int64)
    if take > 1:
        path = np.sort(g.choice(np.arange(1, nodes), take - 1, replace=False))
    path = np.concatenate([[0], path])
    parents = np.array([-1] + [int(g.integers(max(0, i - 6), i)) for i in range(1, nodes)], np.int64)
    parents[path[1:]] = path[:-1]
    return parents, path


@functools.lru_cache(maxsize=4)
def _ctx(preset, overrides):
    dllm = importlib.import_module("distributed-llm1_b200")
    ctx = dllm.initKernels(0, dllm.PRESETS["qwen2.5-" + preset].with_(**dict(overrides)))
    ctx.set_stream(1)  # CUDA's handle of the legacy default stream, the one torch uses unless told otherwise
    return dllm, ctx


def _buf(ctx, t):
    """A device buffer of the framework with a tensor's values, and the tensor that shares its memory."""
    b = ctx.createI32(t.numel()) if t.dtype == torch.int32 else ctx.createF32(t.numel())
    v = torch.as_tensor(b, device="cuda").view(t.shape)
    v.copy_(t)
    return b, v


# ---- inputs --------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    h = np.random.default_rng(seed)
    s = {"case": case, "op": case["op"]}
    if own:
        preset, over = _model(case)
        s["dllm"], s["ctx"] = _ctx(preset, tuple(sorted(over.items())))
    {"rope": _prepare_rope, "tree": _prepare_tree, "pick": _prepare_pick, "commit": _prepare_commit}[case["op"]](s, case, g, h)
    return s


def _prepare_rope(s, case, g, h):
    nq, kvh, hd, _, _ = HEADS[case["dims"]]
    n = case["rows"]
    s["q"] = torch.randn(n, nq, hd, device="cuda", generator=g)
    s["k"] = torch.randn(n, kvh, hd, device="cuda", generator=g)
    s["pos"] = torch.randint(0, case["far"], (n,), device="cuda", generator=g, dtype=torch.int32)
    inv_freq, s["factor"] = _frequencies(case["rotary"], case["scaling"])
    s["inv_freq"] = torch.from_numpy(inv_freq).cuda()
    if own:
        ctx = s["ctx"]
        scaling = {"none": None, "linear": {"type": "linear", "factor": 4.0}, "ntk": {"type": "ntk", "factor": 4.0},
                   "yarn": YARN}[case["scaling"]]
        s["plan"] = ctx.ropePlan(layout=case["layout"], rotary_dim=case["rotary"], theta=THETA, scaling=scaling)
        for k in ("q", "k", "pos"):
            s[k + "_buf"], s[k] = _buf(ctx, s[k])
        for k in ("q", "k"):
            s[k + "_out"], s[k + "_res"] = _buf(ctx, torch.zeros_like(s[k]))


def _frequencies(rotary, scaling):
    """Inverse frequencies (64 bits) and the factor on cos and sin."""
    i = np.arange(rotary // 2, dtype=np.float64)
    if scaling == "ntk":
        return (THETA * 4.0 ** (rotary / (rotary - 2))) ** (-2 * i / rotary), 1.0
    f = THETA ** (-2 * i / rotary)
    if scaling == "linear":
        return f / 4.0, 1.0
    if scaling == "yarn":
        turn = lambda r: rotary * math.log(YARN["original_max_pos"] / (r * 2 * math.pi)) / (2 * math.log(THETA))  # noqa: E731
        low, high = max(math.floor(turn(32.0)), 0), min(math.ceil(turn(1.0)), rotary - 1)
        ramp = np.clip((i - low) / ((high - low) or 0.001), 0, 1)
        return f / 4.0 * ramp + f * (1 - ramp), 0.1 * math.log(4.0) + 1.0
    return f, 1.0


def _paged(s, case, g, h, layers):
    """A paged cache of random K/V with shuffled pages, and the drafted trees over it."""
    nq, kvh, hd, _, _ = HEADS[case["dims"]]
    b, dt = case["seqs"], torch.bfloat16 if case["kv"] == "bf16" else torch.float32
    per = -(-_max_pos(case) // PAGE)
    table = h.permutation(b * per).astype(np.int32).reshape(b, per)
    made = [_parents(h, case["nodes"], case.get("take", 1)) for _ in range(b)]
    s["parents"] = np.concatenate([p for p, _ in made]).astype(np.int32)
    s["paths"] = [p.tolist() for _, p in made]
    s["lens"] = _lens(case)
    s["k"], s["v"] = (torch.randn(layers, b * per, kvh, PAGE, hd, device="cuda", generator=g, dtype=dt) for _ in range(2))
    s["table"] = torch.from_numpy(table).cuda().long()
    s["t0"] = torch.tensor(s["lens"], device="cuda")
    s["tree_parents"] = torch.from_numpy(s["parents"]).cuda().long()
    if own:
        stage = s["stage"] = s["dllm"].Stage(s["ctx"], 0, layers)
        for which in ("k", "v"):
            pool = torch.as_tensor(stage.kv_pool(which), device="cuda")
            pool = pool.view(dt).view(s[which].shape)
            pool.copy_(s[which])
            s[which] = pool
        for i in range(b):
            stage.set_page_table(i, table[i])
            stage.set_t0(i, s["lens"][i])
        s["tree"] = s["ctx"].draftTree(s["parents"], [case["nodes"]] * b)


def _prepare_tree(s, case, g, h):
    nq, kvh, hd, _, _ = HEADS[case["dims"]]
    _paged(s, case, g, h, 1)
    s["q"] = torch.randn(case["seqs"] * case["nodes"], nq, hd, device="cuda", generator=g) * 2.0
    if own:
        s["q_buf"], s["q"] = _buf(s["ctx"], s["q"])
        s["out_buf"], s["out"] = _buf(s["ctx"], torch.zeros_like(s["q"]))


def _prepare_pick(s, case, g, h):
    v, b, m = case["vocab"], case["seqs"], case["nodes"]
    n = b * max(1, m)
    s["logits"] = torch.randn(n, v, device="cuda", generator=g) * 3.0
    lens = [max(1, case["history"] - (case["history"] * i) // (2 * b)) for i in range(b)]
    total = sum(lens)
    # text repeats itself: tokens near the start of the vocabulary come often
    tokens = (torch.rand(total, device="cuda", generator=g) ** 4 * v).to(torch.int32).clamp_(max=v - 1)
    s["history"] = tokens
    s["offsets"] = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")
    s["prompt"] = torch.tensor([ln // 2 for ln in lens], dtype=torch.int32, device="cuda")
    s["penalties"] = torch.tensor([[1.0 + 0.05 * (1 + i % 5), 0.1 * (i % 4), 0.2 * (i % 3)] for i in range(b)], device="cuda")
    if case["bias"]:
        k = min(case["bias"], v)
        s["bias_tokens"] = torch.cat([torch.randperm(v, device="cuda", generator=g)[:k] for _ in range(b)]).to(torch.int32)
        s["bias_values"] = torch.randn(b * k, device="cuda", generator=g) * 4.0
        s["bias_offsets"] = torch.arange(b + 1, device="cuda", dtype=torch.int32) * k
    if case["mask"]:
        words = torch.randint(-(1 << 31), 1 << 31, (n, -(-v // 32)), device="cuda", generator=g)
        s["mask"] = (words & torch.randint(-(1 << 31), 1 << 31, words.shape, device="cuda", generator=g)).to(torch.int32)
    if m:
        made = [_parents(h, m)[0] for _ in range(b)]
        s["parents"] = np.concatenate(made).astype(np.int32)
        s["tree_parents"] = torch.from_numpy(s["parents"]).cuda().long()
        s["draft"] = (torch.rand(n, device="cuda", generator=g) ** 4 * v).to(torch.int32).clamp_(max=v - 1)
    if own:
        ctx = s["ctx"]
        for k in ("logits", "history", "offsets", "prompt", "penalties", "bias_tokens", "bias_values", "bias_offsets", "mask",
                  "draft"):
            if k in s:
                s[k + "_buf"], s[k] = _buf(ctx, s[k])
        s["tokens_buf"], s["tokens"] = _buf(ctx, torch.zeros(n, dtype=torch.int32, device="cuda"))
        if case["keep"]:
            s["out_buf"], s["out"] = _buf(ctx, torch.zeros_like(s["logits"]))
        if m:
            s["tree"] = ctx.draftTree(s["parents"], [m] * b)


def _prepare_commit(s, case, g, h):
    _paged(s, case, g, h, HEADS[case["dims"]][4])


# ---- the operators ---------------------------------------------------------------------------
def run(state):
    if own:
        return {"rope": _own_rope, "tree": _own_tree, "pick": _own_pick, "commit": _own_commit}[state["op"]](state)
    return {"rope": _rope, "tree": _tree, "pick": _pick, "commit": _commit}[state["op"]](state)


def _own_rope(s):
    s["ctx"].ropeAt(s["plan"], s["pos_buf"], s["case"]["rows"], s["q_buf"], s["k_buf"], s["q_out"], s["k_out"])
    return s["q_res"], s["k_res"]


def _own_tree(s):
    s["stage"].tree_attention(0, s["tree"], s["q_buf"], s["out_buf"])
    return s["out"]


def _own_pick(s):
    bias = (s["bias_tokens_buf"], s["bias_values_buf"], s["bias_offsets_buf"]) if "bias_tokens" in s else None
    s["ctx"].pickTokens(s["logits_buf"], s["logits"].shape[0],
                        history=(s["history_buf"], s["offsets_buf"], s["prompt_buf"]), penalties=s["penalties_buf"],
                        bias=bias, mask=s.get("mask_buf"), tree=s.get("tree"), draft=s.get("draft_buf"),
                        out=s.get("out_buf"), tokens=s["tokens_buf"])
    return (s["tokens"], s["out"]) if s["case"]["keep"] else (s["tokens"],)


def _own_commit(s):
    stage = s["stage"]
    for i, t0 in enumerate(s["lens"]):  # back to the state before the draft, as after a step that was thrown away
        stage.set_t0(i, t0)
    stage.commit_tree(s["tree"], s["paths"])
    return s["k"], s["v"], [stage.t0_of(i) for i in range(len(s["lens"]))]


def _rope(s):
    """Pairs (x1, x2) of the first `rotary` dims turn by position * inv_freq; the rest pass."""
    r, half = s["case"]["rotary"], s["case"]["layout"] == "half"
    angle = s["pos"].double()[:, None] * s["inv_freq"]
    cos, sin = ((f(angle) * s["factor"]).float()[:, None, :] for f in (torch.cos, torch.sin))
    out = []
    for x in (s["q"], s["k"]):
        a, b = (x[..., : r // 2], x[..., r // 2 : r]) if half else (x[..., 0:r:2], x[..., 1:r:2])
        a, b = a * cos - b * sin, a * sin + b * cos
        turned = torch.cat([a, b], -1) if half else torch.stack([a, b], -1).flatten(-2)
        out.append(torch.cat([turned, x[..., r:]], -1))
    return tuple(out)


def _ancestors(parents, b, m):
    """[b, m, m] truth values: node j is node i or one of its ancestors."""
    p = parents.view(b, m)
    at = torch.arange(m, device=p.device)
    step = (p[:, :, None] == at) & (p[:, :, None] >= 0)
    see = step.float() + torch.eye(m, device=p.device)
    for _ in range(max(1, m - 1).bit_length()):  # paths of twice the length with each product
        see = ((see @ see) > 0).float()
    return see > 0


def _slots(s, case):
    """Each sequence's cache gathered into [b, slots, KV heads, head size], fp32."""
    b, hd = case["seqs"], s["k"].shape[-1]
    longest = max(s["lens"]) + case["nodes"]
    at = torch.arange(longest, device="cuda")
    page = s["table"][:, at // PAGE]
    return [x[0][page, :, (at % PAGE)[None, :].expand(b, -1)].float() for x in (s["k"], s["v"])]


def _tree(s):
    case = s["case"]
    nq, kvh, hd, _, _ = HEADS[case["dims"]]
    b, m = case["seqs"], case["nodes"]
    k, v = _slots(s, case)
    q = s["q"].view(b, m, kvh, nq // kvh, hd)
    score = torch.einsum("bmhgd,bthd->bhmgt", q, k) * (1.0 / math.sqrt(hd))
    at = torch.arange(k.shape[1], device="cuda")
    node = at[None, :] - s["t0"][:, None]  # the node of a slot, negative in the context
    see = torch.gather(_ancestors(s["tree_parents"], b, m), 2, node.clamp(0, m - 1)[:, None, :].expand(b, m, -1))
    see = torch.where((node < 0)[:, None], True, see & (node < m)[:, None])[:, None, :, None, :]
    score = torch.where(see, score, float("-inf"))
    p = torch.exp(score - score.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    return torch.einsum("bhmgt,bthd->bmhgd", p, v).reshape(b * m, nq, hd)


def _pick(s):
    case = s["case"]
    v, b, m = case["vocab"], case["seqs"], case["nodes"]
    x = s["logits"]
    n = x.shape[0]
    off = s["offsets"].long()
    at = torch.arange(s["history"].numel(), device="cuda")
    seq = torch.searchsorted(off, at, right=True) - 1
    made = (at - off[seq] >= s["prompt"].long()[seq]).float()
    cell = seq * v + s["history"].long()
    count = torch.zeros(b * v, device="cuda").scatter_add_(0, cell, made).view(b, v)
    seen = torch.zeros(b * v, device="cuda").scatter_(0, cell, 1.0).view(b, v)
    row = torch.arange(n, device="cuda") // max(1, m)
    count, seen = count[row], seen[row]
    if m:
        see = _ancestors(s["tree_parents"], b, m).float().view(n, m)
        token = s["draft"].long().view(b, m)[row]
        count = count.scatter_add(1, token, see)
        seen = seen.scatter_add(1, token, see)
    rep, freq, pres = (s["penalties"][row, j, None] for j in range(3))
    y = torch.where(seen > 0, torch.where(x > 0, x / rep, x * rep), x)
    y = torch.where(count > 0, y - freq * count - pres, y)
    if "bias_tokens" in s:
        boff = s["bias_offsets"].long()
        of = torch.searchsorted(boff, torch.arange(s["bias_tokens"].numel(), device="cuda"), right=True) - 1
        bias = torch.zeros(b * v, device="cuda").scatter_(0, of * v + s["bias_tokens"].long(), s["bias_values"]).view(b, v)
        y = y + bias[row]
    if "mask" in s:
        at = torch.arange(v, device="cuda")
        allowed = (s["mask"][:, at // 32] >> (at % 32).int()) & 1
        y = torch.where(allowed > 0, y, float("-inf"))
    best = y.amax(-1, keepdim=True)
    token = torch.where(y == best, torch.arange(v, device="cuda"), v).amin(-1).to(torch.int32)
    return (token, y) if case["keep"] else (token,)


def _commit(s):
    lens = s["lens"]
    src = torch.tensor([[i, t + j] for i, (t, p) in enumerate(zip(lens, s["paths"])) for j in p], device="cuda")
    dst = torch.tensor([[i, t + j] for i, (t, p) in enumerate(zip(lens, s["paths"])) for j in range(len(p))], device="cuda")
    page = lambda c: s["table"][c[:, 0], c[:, 1] // PAGE]  # noqa: E731
    for x in (s["k"], s["v"]):
        x[:, page(dst), :, dst[:, 1] % PAGE] = x[:, page(src), :, src[:, 1] % PAGE]
    return s["k"], s["v"], [t + len(p) for t, p in zip(lens, s["paths"])]


# ---- what a pass cannot do without ---------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "pick":
        n = case["seqs"] * max(1, case["nodes"])
        read = n * case["vocab"] * 4 + 4 * sum(max(1, case["history"] - (case["history"] * i) // (2 * case["seqs"]))
                                               for i in range(case["seqs"]))
        read += n * -(-case["vocab"] // 32) * 4 if case["mask"] else 0
        return {"bytes": read + (n * case["vocab"] * 4 if case["keep"] else 0) + 4 * n, "flops": 4 * n * case["vocab"]}
    nq, kvh, hd, _, layers = HEADS[case["dims"]]
    if op == "rope":
        n = case["rows"]
        return {"bytes": 2 * 4 * n * (nq + kvh) * hd + 4 * n, "flops": 6 * n * (nq + kvh) * (case["rotary"] // 2)}
    size = 2 if case["kv"] == "bf16" else 4
    rows = case["seqs"] * case["nodes"]
    if op == "tree":
        slots = sum(_lens(case)) + rows
        pairs = sum(t + 1 for t in _lens(case)) * case["nodes"]
        return {"bytes": 2 * slots * kvh * hd * size + 2 * 4 * rows * nq * hd, "flops": 4 * pairs * nq * hd}
    return {"bytes": 2 * 2 * layers * case["seqs"] * case["take"] * kvh * hd * size, "flops": 0}


# ---- the definitions in 64 bits ------------------------------------------------------------------
def exact(case, seed):
    global own
    mine, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = mine
    return {"rope": _exact_rope, "tree": _exact_tree, "pick": _exact_pick, "commit": _exact_commit}[case["op"]](s, case)


def _exact_rope(s, case):
    r = case["rotary"]
    turn = torch.polar(torch.full((1,), s["factor"], dtype=torch.float64, device="cuda"),
                       s["pos"].double()[:, None] * s["inv_freq"])[:, None, :]
    out = []
    for x in (s["q"].double(), s["k"].double()):
        y = x.clone()
        if case["layout"] == "half":
            z = torch.complex(x[..., : r // 2], x[..., r // 2 : r]) * turn
            y[..., : r // 2], y[..., r // 2 : r] = z.real, z.imag
        else:
            z = torch.complex(x[..., 0:r:2], x[..., 1:r:2]) * turn
            y[..., 0:r:2], y[..., 1:r:2] = z.real, z.imag
        out.append(y)
    return tuple(out)


def _lineage(parents, i):
    line = [i]
    while parents[line[-1]] >= 0:
        line.append(int(parents[line[-1]]))
    return line


def _exact_tree(s, case):
    nq, kvh, hd, _, _ = HEADS[case["dims"]]
    m, group = case["nodes"], nq // kvh
    if 4.0 * nq * hd * m * sum(_lens(case)) > 4e11:
        return None
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for i, t0 in enumerate(s["lens"]):
        at = torch.arange(t0 + m, device="cuda")
        page, off = s["table"][i][at // PAGE], at % PAGE
        see = torch.zeros(m, t0 + m, dtype=torch.bool)
        see[:, :t0] = True
        for j in range(m):
            see[j, [t0 + a for a in _lineage(s["parents"][i * m : (i + 1) * m], j)]] = True
        see = see.cuda().repeat_interleave(group, 0)
        for head in range(kvh):
            k, v = (x[0][page, head, off].double() for x in (s["k"], s["v"]))
            rows = s["q"][i * m : (i + 1) * m, head * group : (head + 1) * group].double().reshape(m * group, hd)
            z = (rows @ k.T / math.sqrt(hd)).masked_fill(~see, -math.inf)
            out[i * m : (i + 1) * m, head * group : (head + 1) * group] = (torch.softmax(z, -1) @ v).view(m, group, hd)
    return out


def _exact_pick(s, case):
    if not case["keep"]:
        return None
    v, m = case["vocab"], case["nodes"]
    y = s["logits"].double()
    history, off, prompt = s["history"].cpu().numpy(), s["offsets"].tolist(), s["prompt"].tolist()
    pen = s["penalties"].double()
    for row in range(y.shape[0]):
        i = row // max(1, m)
        told = history[off[i] : off[i + 1]]
        said = told[prompt[i] :]
        if m:
            tree = s["parents"][i * m : (i + 1) * m]
            said = np.concatenate([said, s["draft"].cpu().numpy()[[i * m + a for a in _lineage(tree, row - i * m)]]])
        any_ = torch.from_numpy(np.union1d(told, said).astype(np.int64)).cuda()
        new, times = np.unique(said, return_counts=True)
        z = y[row, any_]
        y[row, any_] = torch.where(z > 0, z / pen[i, 0], z * pen[i, 0])
        y[row, torch.from_numpy(new.astype(np.int64)).cuda()] -= torch.from_numpy(times).cuda() * pen[i, 1] + pen[i, 2]
        if "bias_tokens" in s:
            a, e = s["bias_offsets"][i], s["bias_offsets"][i + 1]
            y[row, s["bias_tokens"][a:e].long()] += s["bias_values"][a:e].double()
        if "mask" in s:
            bits = np.unpackbits(s["mask"][row].cpu().numpy().view(np.uint8), bitorder="little")[:v]
            y[row, torch.from_numpy(bits == 0).cuda()] = -math.inf
    return None, y


def _exact_commit(s, case):
    for i, (t0, path) in enumerate(zip(s["lens"], s["paths"])):
        for x in (s["k"], s["v"]):
            rows = [x[:, int(s["table"][i, (t0 + j) // PAGE]), :, (t0 + j) % PAGE].clone() for j in path]
            for j, r in enumerate(rows):
                x[:, int(s["table"][i, (t0 + j) // PAGE]), :, (t0 + j) % PAGE] = r
    return s["k"], s["v"], None
