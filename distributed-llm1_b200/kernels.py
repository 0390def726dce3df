"""Kernel context: the `ctx` object of kernels.js on the B200 path.

`initKernels(device)` (kernels.js:5) returns a context whose methods keep the
reference's names, argument order and error behaviour (kernels.js:179-301):
buffer helpers `loadWeightBits / createF32 / writeF32 / readF32` and one op
launcher per shader `matmul / rmsnorm / ropeQ / ropeK / attention / siluMul /
add / addBias`. Each op allocates and returns a new device buffer, as the
reference does; every op runs a hand-written sm_100a kernel from libdllm.so.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import _lib
from .constants import CFG, ModelConfig


class GpuBuffer:
    """A device buffer (the GPUBuffer of the reference). Freed with the object."""

    __slots__ = ("ctx", "handle", "n", "dtype", "label", "__weakref__")

    def __init__(self, ctx: "KernelContext", handle: int, n: int, dtype: str, label: str = ""):
        self.ctx, self.handle, self.n, self.dtype, self.label = ctx, handle, n, dtype, label

    @property
    def size(self) -> int:
        """Bytes on the device (GPUBuffer.size)."""
        return int(self.ctx.lib.dllm_buf_bytes(self.handle))

    @property
    def device_ptr(self) -> int:
        return int(self.ctx.lib.dllm_buf_device_ptr(self.handle) or 0)

    @property
    def __cuda_array_interface__(self) -> dict:
        """The buffer's memory as a flat array (bf16 as int16 bits), e.g. for
        torch.as_tensor(buf, device="cuda"). No stream is synchronised: order the
        other library's work with the ctx stream (set_stream)."""
        if not self.handle:
            raise ValueError(f"buffer {self.label!r} has been destroyed")
        return {"shape": (self.n,), "typestr": {"f32": "<f4", "i32": "<i4", "bf16": "<i2"}[self.dtype],
                "data": (self.device_ptr, False), "version": 3, "strides": None}

    def destroy(self):
        if self.handle:
            self.ctx.lib.dllm_buf_free(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.destroy()
        except Exception:
            pass


class RopePlan:
    """Rotary frequencies of ropeAt on the device. Freed with the object."""

    LAYOUTS = {"half": 0, "interleaved": 1}
    SCALINGS = {"none": 0, "linear": 1, "ntk": 2, "yarn": 3}

    def __init__(self, ctx: "KernelContext", layout: str, rotary_dim: int, theta: float, scaling: dict | None):
        s = dict(scaling or {})
        kind = s.pop("type", "none")
        if layout not in self.LAYOUTS or kind not in self.SCALINGS:
            raise _lib.DllmError(_lib.DLLM_EINVAL, f"ropePlan: unknown layout {layout!r} or scaling {kind!r}")
        c = _lib.dllm_rope_config(self.LAYOUTS[layout], int(rotary_dim), float(theta), self.SCALINGS[kind],
                                  float(s.pop("factor", 1.0)), int(s.pop("original_max_pos", 0)),
                                  float(s.pop("beta_fast", 32.0)), float(s.pop("beta_slow", 1.0)),
                                  float(s.pop("attention_factor", 0.0)))
        if s:
            raise _lib.DllmError(_lib.DLLM_EINVAL, f"ropePlan: unknown scaling keys {sorted(s)}")
        self.ctx, self.handle = ctx, None
        h = C.c_void_p()
        ctx._check(ctx.lib.dllm_rope_plan_create(ctx.handle, C.byref(c), C.byref(h)), "ropePlan")
        self.handle = h.value

    def destroy(self):
        if self.handle:
            self.ctx.lib.dllm_rope_plan_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.destroy()
        except Exception:
            pass


def int32s(values, what: str) -> np.ndarray:
    """Integers as a flat int32 array; numbers that do not fit, or are no integers, are refused."""
    a = np.asarray(values).reshape(-1)
    b = a.astype(np.int32) if a.dtype.kind in "iu" or not a.size else None
    if b is None or (a != b).any():
        raise _lib.DllmError(_lib.DLLM_EINVAL, f"{what}: need 32-bit integers")
    return b


class DraftTree:
    """Drafted trees of one or more sequences (dllm_tree_create). Freed with the object."""

    def __init__(self, ctx: "KernelContext", parents, counts=None, seqs=None):
        self.ctx, self.handle = ctx, None
        self.parents = int32s(parents, "draftTree parents")
        n = self.parents.size
        self.counts = np.array([n], np.int32) if counts is None else int32s(counts, "draftTree counts")
        self.seqs = np.arange(self.counts.size, dtype=np.int32) if seqs is None else int32s(seqs, "draftTree seqs")
        if self.seqs.size != self.counts.size or (self.counts < 0).any() or int(self.counts.sum()) != self.parents.size:
            raise _lib.DllmError(_lib.DLLM_EINVAL, f"draftTree: {self.parents.size} parents for counts "
                                                   f"{self.counts.tolist()} of sequences {self.seqs.tolist()}")
        self.n = int(self.parents.size)
        h = C.c_void_p()
        ctx._check(ctx.lib.dllm_tree_create(ctx.handle, _lib.ptr(self.parents, C.c_int32),
                                            _lib.ptr(self.counts, C.c_int32), _lib.ptr(self.seqs, C.c_int32),
                                            self.counts.size, C.byref(h)), "draftTree")
        self.handle = h.value

    def accept(self, draft, picked) -> tuple[list, list]:
        """Greedy verification: per sequence, the path of nodes whose tokens the picks
        agree with and the new tokens. Node 0 is the sequence's last token; from it on,
        the lowest child whose drafted token is the current node's pick continues the
        path, and the last node's pick ends the new tokens."""
        draft, picked = np.asarray(draft).reshape(-1), np.asarray(picked).reshape(-1)
        if draft.size != self.n or picked.size != self.n:
            raise _lib.DllmError(_lib.DLLM_EINVAL, f"accept: {draft.size} drafted, {picked.size} picked, {self.n} nodes")
        paths, tokens, row0 = [], [], 0
        for m in self.counts.tolist():
            path, new = ([0], [int(picked[row0])]) if m else ([], [])
            for j in range(1, m):
                if self.parents[row0 + j] == path[-1] and draft[row0 + j] == new[-1]:
                    path.append(j)
                    new.append(int(picked[row0 + j]))
            paths.append(path)
            tokens.append(new)
            row0 += m
        return paths, tokens

    def destroy(self):
        if self.handle:
            self.ctx.lib.dllm_tree_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.destroy()
        except Exception:
            pass


class KernelContext:
    def __init__(self, device: int = 0, cfg: ModelConfig | None = None):
        self.lib = _lib.load()
        self.cfg = cfg or CFG
        self.device = device
        h = C.c_void_p()
        c = self.cfg.to_c()
        st = self.lib.dllm_init_kernels(device, C.byref(c), C.byref(h))
        if st != _lib.DLLM_OK:
            raise _lib.DllmError(st, f"initKernels(device={device}) failed: "
                                     f"{self.lib.dllm_status_string(st).decode()} (is this an sm_100 GPU?)")
        self.handle = h.value
        # kernels.js:173 dims, exposed on ctx like the reference
        self.D = self.cfg.hidden_size
        self.KVH = self.cfg.num_kv_heads
        self.NQ = self.cfg.num_q_heads
        self.HD = self.cfg.head_dim

    # ---- plumbing
    def _check(self, st: int, what: str = ""):
        if st:
            _lib.check(st, self.handle, what)

    def _out(self, fn, *args, n: int, label: str) -> GpuBuffer:
        out = C.c_void_p()
        self._check(fn(self.handle, *args, C.byref(out)), label)
        return GpuBuffer(self, out.value, n, "f32", label)

    @staticmethod
    def _h(obj, kind=GpuBuffer):
        """The handle of a live object of one kind: the library takes plain pointers."""
        if not isinstance(obj, kind) or not obj.handle:
            raise ValueError(f"expected a live {kind.__name__}")
        return obj.handle

    @classmethod
    def _opt(cls, obj, kind=GpuBuffer):
        return None if obj is None else cls._h(obj, kind)

    def close(self):
        if getattr(self, "handle", None):
            self.lib.dllm_ctx_destroy(self.handle)
            self.handle = None

    def set_stream(self, cuda_stream: int | None):
        """Enqueue on a caller-owned cudaStream_t (e.g. torch.cuda.Stream().cuda_stream); 0 / None
        (the legacy default stream's handle) selects the ctx's own stream."""
        self._check(self.lib.dllm_ctx_set_stream(self.handle, cuda_stream or None), "set_stream")

    def set_tensor_core_rows(self, min_rows: int):
        """Passes of >= min_rows rows use the tcgen05 GEMM (0: never); default 8."""
        self._check(self.lib.dllm_ctx_set_tensor_core_rows(self.handle, int(min_rows)), "set_tensor_core_rows")

    def synchronize(self, timeout_ms: int = 15000):
        self._check(self.lib.dllm_ctx_synchronize(self.handle, timeout_ms), "synchronize")

    @property
    def launch_count(self) -> int:
        return int(self.lib.dllm_ctx_launch_count(self.handle))

    # ---- buffers (kernels.js:181-211)
    def loadWeightBits(self, u32arr, label: str | None = None) -> GpuBuffer:
        a = np.ascontiguousarray(u32arr, dtype=np.uint32) if u32arr is not None else None
        if a is None or a.size == 0:
            raise _lib.DllmError(_lib.DLLM_EINVAL, "loadWeightBits: empty weights")  # kernels.js:182
        out = C.c_void_p()
        self._check(self.lib.dllm_load_weight_bits(self.handle, _lib.ptr(a, C.c_uint32), a.size,
                                                   (label or "weights").encode(), C.byref(out)), "loadWeightBits")
        return GpuBuffer(self, out.value, a.size, "bf16", label or "weights")

    def loadWeightBf16(self, u16arr, label: str | None = None) -> GpuBuffer:
        a = np.ascontiguousarray(u16arr, dtype=np.uint16) if u16arr is not None else None
        if a is None or a.size == 0:
            raise _lib.DllmError(_lib.DLLM_EINVAL, "loadWeightBits: empty weights")
        out = C.c_void_p()
        self._check(self.lib.dllm_load_weight_bf16(self.handle, _lib.ptr(a, C.c_uint16), a.size,
                                                   (label or "weights").encode(), C.byref(out)), "loadWeightBf16")
        return GpuBuffer(self, out.value, a.size, "bf16", label or "weights")

    def createBf16(self, n: int, label: str = "") -> GpuBuffer:
        out = C.c_void_p()
        self._check(self.lib.dllm_create_bf16(self.handle, int(n), label.encode(), C.byref(out)), "createBf16")
        return GpuBuffer(self, out.value, int(n), "bf16", label)

    def fillNormalBf16(self, buf: GpuBuffer, seed: int, std: float):
        self._check(self.lib.dllm_fill_normal_bf16(self.handle, self._h(buf), seed, std), "fillNormalBf16")

    def fillConstBf16(self, buf: GpuBuffer, value: float):
        self._check(self.lib.dllm_fill_const_bf16(self.handle, self._h(buf), value), "fillConstBf16")

    def readBf16(self, buf: GpuBuffer, n: int | None = None) -> np.ndarray:
        n = buf.n if n is None else n
        out = np.empty(n, np.uint16)
        self._check(self.lib.dllm_read_bf16(self.handle, self._h(buf), _lib.ptr(out, C.c_uint16), n), "readBf16")
        return out

    def createF32(self, numFloats: int, label: str = "") -> GpuBuffer:
        if not numFloats or numFloats <= 0:
            raise _lib.DllmError(_lib.DLLM_EINVAL, f"createF32: invalid size {numFloats}")  # kernels.js:189
        out = C.c_void_p()
        self._check(self.lib.dllm_create_f32(self.handle, int(numFloats), label.encode(), C.byref(out)), "createF32")
        return GpuBuffer(self, out.value, int(numFloats), "f32", label)

    def writeF32(self, buf: GpuBuffer, f32):
        a = np.ascontiguousarray(f32, dtype=np.float32).reshape(-1)
        self._check(self.lib.dllm_write_f32(self.handle, self._h(buf), _lib.ptr(a, C.c_float), a.size), "writeF32")

    def readF32(self, buf: GpuBuffer, numFloats: int, label: str = "") -> np.ndarray:
        if not numFloats or numFloats <= 0:
            raise _lib.DllmError(_lib.DLLM_EINVAL, f"readF32: invalid size {numFloats}")  # kernels.js:196
        out = np.empty(int(numFloats), np.float32)
        self._check(self.lib.dllm_read_f32(self.handle, self._h(buf), _lib.ptr(out, C.c_float), out.size,
                                           label.encode()), "readF32")
        return out

    def createI32(self, n: int, label: str = "") -> GpuBuffer:
        out = C.c_void_p()
        self._check(self.lib.dllm_create_i32(self.handle, max(0, int(n)), label.encode(), C.byref(out)), "createI32")
        return GpuBuffer(self, out.value, int(n), "i32", label)

    def writeI32(self, buf: GpuBuffer, values):
        a = np.ascontiguousarray(values, dtype=np.int32).reshape(-1)
        self._check(self.lib.dllm_write_i32(self.handle, self._h(buf), _lib.ptr(a, C.c_int32), a.size), "writeI32")

    def readI32(self, buf: GpuBuffer, n: int | None = None) -> np.ndarray:
        out = np.empty(buf.n if n is None else int(n), np.int32)
        self._check(self.lib.dllm_read_i32(self.handle, self._h(buf), _lib.ptr(out, C.c_int32), out.size), "readI32")
        return out

    # ---- ops (kernels.js:222-301)
    def matmul(self, xBuf, wBuf, n, din, dout) -> GpuBuffer:
        return self._out(self.lib.dllm_matmul, self._h(xBuf), self._h(wBuf), n, din, dout, n=n * dout,
                         label=f"mm_out_{n}x{dout}")

    def rmsnorm(self, xBuf, gBuf, n) -> GpuBuffer:
        return self._out(self.lib.dllm_rmsnorm, self._h(xBuf), self._h(gBuf), n, n=n * self.D, label=f"rms_out_{n}")

    def ropeQ(self, xBuf, posStart, n) -> GpuBuffer:
        self._check(self.lib.dllm_rope_q(self.handle, self._h(xBuf), posStart, n), "ropeQ")
        return xBuf

    def ropeK(self, xBuf, posStart, n) -> GpuBuffer:
        self._check(self.lib.dllm_rope_k(self.handle, self._h(xBuf), posStart, n), "ropeK")
        return xBuf

    def attention(self, qBuf, kCacheBuf, vCacheBuf, T0, n) -> GpuBuffer:
        return self._out(self.lib.dllm_attention, self._h(qBuf), self._h(kCacheBuf), self._h(vCacheBuf), T0, n,
                         n=n * self.NQ * self.HD, label=f"attn_out_{n}")

    def siluMul(self, aBuf, bBuf, total) -> GpuBuffer:
        return self._out(self.lib.dllm_silu_mul, self._h(aBuf), self._h(bBuf), total, n=total,
                         label=f"silu_out_{total}")

    def add(self, aBuf, bBuf, numFloats) -> GpuBuffer:
        return self._out(self.lib.dllm_add, self._h(aBuf), self._h(bBuf), numFloats, n=numFloats,
                         label=f"add_out_{numFloats}")

    def addBias(self, aBuf, biasBuf, n, dout) -> GpuBuffer:
        return self._out(self.lib.dllm_add_bias, self._h(aBuf), self._h(biasBuf), n, dout, n=n * dout,
                         label=f"bias_out_{n * dout}")

    def argmax(self, logitsBuf, n) -> int:
        """Greedy pick over device logits: the strict '>' scan of pipeline.js:159-162."""
        idx = C.c_int32()
        self._check(self.lib.dllm_argmax(self.handle, self._h(logitsBuf), n, C.byref(idx)), "argmax")
        return int(idx.value)

    # ---- verification of drafted tokens (include/dllm.h; no counterpart in the reference)
    def ropePlan(self, layout: str = "half", rotary_dim: int | None = None, theta: float | None = None,
                 scaling: dict | None = None) -> RopePlan:
        """Rotary frequencies for ropeAt. layout "half" (pairs i, i + rotary_dim / 2) or
        "interleaved" (2i, 2i + 1); rotary_dim defaults to the head size, theta to the
        config's. scaling: None, {"type": "linear" | "ntk", "factor": f} or {"type":
        "yarn", "factor": f, "original_max_pos": n[, "beta_fast": 32, "beta_slow": 1]};
        "attention_factor" overrides the factor on cos and sin."""
        return RopePlan(self, layout, self.HD if rotary_dim is None else rotary_dim,
                        self.cfg.rope_theta if theta is None else theta, scaling)

    def ropeAt(self, plan: RopePlan, positions: GpuBuffer, n: int, qBuf: GpuBuffer | None = None,
               kBuf: GpuBuffer | None = None, qOut: GpuBuffer | None = None, kOut: GpuBuffer | None = None):
        """Row t of q [n, NQ*HD] and k [n, KVH*HD] at positions[t]; in place without outputs."""
        h, o = self._h, self._opt
        self._check(self.lib.dllm_rope_at(self.handle, h(plan, RopePlan), h(positions), n, o(qBuf), o(kBuf), o(qOut),
                                          o(kOut)), "ropeAt")
        return qOut or qBuf, kOut or kBuf

    def draftTree(self, parents, counts=None, seqs=None) -> DraftTree:
        """Drafted trees of one or more cache sequences: counts[i] nodes for sequence
        seqs[i] (default i), each node with the index of its parent in the sequence
        (below its own), -1 for a root. counts defaults to one sequence."""
        return DraftTree(self, parents, counts, seqs)

    def pickTokens(self, logits: GpuBuffer, n: int, history=None, penalties: GpuBuffer | None = None, bias=None,
                   mask: GpuBuffer | None = None, tree: DraftTree | None = None, draft: GpuBuffer | None = None,
                   out: GpuBuffer | None = None, tokens: GpuBuffer | None = None) -> GpuBuffer:
        """One token per row of logits [n, vocab] under penalties for repeated tokens,
        biases and a grammar mask (dllm_pick_tokens); i32 [n], -1 where the mask allows
        nothing. history: (tokens, offsets, prompt_lens or None), with a tree the tokens
        before each root, and prompt_lens may reach into the nodes' paths; bias: (tokens,
        values, offsets); `out` also receives the processed logits."""
        if tokens is None:
            tokens = self.createI32(n, "picked")
        h, o = self._h, self._opt
        ht, ho, hp = history if history is not None else (None, None, None)
        bt, bv, bo = bias if bias is not None else (None, None, None)
        a = _lib.dllm_pick(n, h(logits), o(ht), o(ho), o(hp), o(penalties), o(bt), o(bv), o(bo), o(mask),
                           o(tree, DraftTree), o(draft), o(out), h(tokens))
        self._check(self.lib.dllm_pick_tokens(self.handle, C.byref(a)), "pickTokens")
        return tokens

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def initKernels(device: int = 0, cfg: ModelConfig | None = None) -> KernelContext:
    """kernels.js:5. `device` is a CUDA ordinal (the reference takes a GPUDevice)."""
    return KernelContext(device, cfg)


init_kernels = initKernels
