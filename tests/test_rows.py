"""Host side of batches of rows and of the 4-bit cache: what is refused before anything
reaches a GPU."""
import importlib

import numpy as np
import pytest

from test_verify import NoLibrary, bare_tree

kernels = importlib.import_module("distributed-llm1_b200.kernels")


def bare(dllm):
    """A context, a stage and a cache that no library stands behind."""
    ctx = object.__new__(kernels.KernelContext)
    ctx.lib, ctx.handle, ctx.cfg = NoLibrary(), None, dllm.CFG
    ctx.NQ, ctx.KVH, ctx.HD, ctx.D = 2, 2, 64, 8
    stage, cache = object.__new__(dllm.Stage), object.__new__(dllm.Cache4)
    for x in (stage, cache):
        x.k, x.lib, x.handle = ctx, ctx.lib, None
    stage._owned = False
    return ctx, stage, cache


@pytest.mark.parametrize("counts,seqs", [([1, -1], None), ([1, 2], [0]), ([1], [0, 1]), ([1.5], None), ([1], [0.5]),
                                         (np.array([2 ** 32]), None), (np.array([1]), np.array([2 ** 32]))])
def test_counts_are_checked(dllm, counts, seqs):
    with pytest.raises(dllm.DllmError):
        kernels.RowBatch(None, counts, seqs)


def test_objects_of_another_kind_are_refused(dllm):
    """The library takes plain pointers: buffers, batches, trees and plans must not pass for one another."""
    ctx, stage, cache = bare(dllm)
    buf, tree = kernels.GpuBuffer(ctx, 16, 2, "f32"), bare_tree([-1], [1])
    plan, rows = object.__new__(kernels.RopePlan), object.__new__(kernels.RowBatch)
    plan.ctx = rows.ctx = ctx
    rows.n = 1
    tree.handle, plan.handle, rows.handle = 32, 48, 64
    try:
        for wrong in (buf, tree, plan, None):
            for call in (lambda: stage.append_rows(0, wrong, buf, buf), lambda: stage.window_attention(0, wrong, buf, buf),
                         lambda: cache.append(0, wrong, buf, buf), lambda: cache.attention(0, wrong, buf),
                         lambda: cache.read_rows(0, wrong, buf)):
                with pytest.raises(ValueError):
                    call()
        for wrong in (rows, tree, plan, "buffer"):
            for call in (lambda: stage.append_rows(0, rows, wrong, buf), lambda: stage.append_rows(0, rows, buf, wrong),
                         lambda: stage.window_attention(0, rows, wrong, buf), lambda: stage.window_attention(0, rows, buf, wrong),
                         lambda: cache.append(0, rows, buf, wrong), lambda: cache.attention(0, rows, wrong),
                         lambda: cache.read_rows(0, rows, wrong, buf), lambda: ctx.normRopeAt(plan, wrong, 1, buf, None, buf),
                         lambda: ctx.normRopeAt(plan, buf, 1, wrong, None, buf), lambda: ctx.normRopeAt(plan, buf, 1, buf, None, wrong),
                         lambda: ctx.normRopeAt(plan, buf, 1, buf, None, buf, qOut=wrong)):
                with pytest.raises(ValueError):
                    call()
        for wrong in (rows, tree, buf):
            with pytest.raises(ValueError):
                ctx.normRopeAt(wrong, buf, 1, buf, None, buf)
        # windows and sinks are 32-bit integers
        for kw in ({"window": 2 ** 31}, {"window": 1.5}, {"sinks": -2 ** 32 + 4}):
            with pytest.raises(dllm.DllmError):
                stage.window_attention(0, rows, buf, buf, **kw)
        with pytest.raises(dllm.DllmError):
            cache.set_page_table(0, [2 ** 32])
    finally:  # the handles are made up
        for x in (buf, tree, plan, rows):
            x.handle = None


def test_null_arguments_are_refused(dllm):
    lib = dllm.load_library()
    bad = dllm._lib.DLLM_EINVAL
    assert lib.dllm_norm_rope_at(None, None, None, 1, None, None, None, None, None, None) == bad
    assert lib.dllm_rows_create(None, None, None, 1, None) == bad
    assert lib.dllm_stage_append_rows(None, 0, None, None, None) == bad
    assert lib.dllm_stage_window_attention(None, 0, None, None, None, 0, 0) == bad
    assert lib.dllm_kv4_create(None, 0, 1, None) == bad
    assert lib.dllm_kv4_reset(None) == bad and lib.dllm_kv4_set_t0(None, 0, 0) == bad
    assert lib.dllm_kv4_get_t0(None, 0) == -1 and lib.dllm_kv4_pages_per_seq(None) == -1 and lib.dllm_kv4_bytes(None) == 0
    assert lib.dllm_kv4_set_page_table(None, 0, None, 0) == bad
    assert lib.dllm_kv4_append(None, 0, None, None, None) == bad
    assert lib.dllm_kv4_read_rows(None, 0, None, None, None) == bad
    assert lib.dllm_kv4_attention(None, 0, None, None, None, 0, 0) == bad
    lib.dllm_rows_destroy(None)
    lib.dllm_kv4_destroy(None)


@pytest.mark.parametrize("wrong", [2 ** 32, 2 ** 32 + 1, -2 ** 32, 2 ** 31, np.int64(2 ** 32), 0.5, "0", None])
def test_layers_sequences_and_slots_are_32_bit_integers(dllm, wrong):
    """ctypes cuts larger numbers to some other layer, sequence or slot."""
    ctx, stage, cache = bare(dllm)
    buf = kernels.GpuBuffer(ctx, 16, 2, "f32")
    plan, rows = object.__new__(kernels.RopePlan), object.__new__(kernels.RowBatch)
    plan.ctx = rows.ctx = ctx
    rows.n = 1
    plan.handle, rows.handle = 48, 64
    try:
        for call in (lambda: stage.append_rows(wrong, rows, buf, buf), lambda: stage.window_attention(wrong, rows, buf, buf),
                     lambda: stage.window_attention(wrong, rows, buf), lambda: stage.t0_of(wrong), lambda: stage.set_t0(wrong, 0),
                     lambda: stage.set_page_table(wrong, [0]), lambda: cache.append(wrong, rows, buf, buf),
                     lambda: cache.attention(wrong, rows, buf), lambda: cache.read_rows(wrong, rows, buf),
                     lambda: cache.read_rows(wrong, rows), lambda: cache.t0_of(wrong), lambda: cache.set_t0(wrong, 0),
                     lambda: cache.set_page_table(wrong, [0]), lambda: dllm.Cache4(ctx, wrong, 1), lambda: dllm.Cache4(ctx, 0, wrong),
                     lambda: ctx.normRopeAt(plan, buf, wrong, buf, None, buf), lambda: ctx.ropeAt(plan, buf, wrong, buf)):
            with pytest.raises(dllm.DllmError):
                call()
        if isinstance(wrong, (int, np.integer)):  # T0 takes what int() takes, as it did
            for cached in (stage, cache):
                with pytest.raises(dllm.DllmError):
                    cached.set_t0(0, wrong)
                with pytest.raises(dllm.DllmError):
                    cached.T0 = wrong
    finally:  # the handles are made up
        for x in (buf, plan, rows):
            x.handle = None
