"""Host side of verifying drafted tokens: the greedy acceptance of a tree, and the
calls that are refused before anything reaches a GPU."""
import ctypes as C
import gc
import importlib
import os
import re

import numpy as np
import pytest

kernels = importlib.import_module("distributed-llm1_b200.kernels")


def bare_tree(parents, counts):
    t = object.__new__(kernels.DraftTree)
    t.ctx, t.handle = None, None
    t.parents, t.counts = np.array(parents, np.int32), np.array(counts, np.int32)
    t.n = len(parents)
    return t


def test_accept_walks_the_picks():
    #        0 -> 1, 2;  1 -> 3;  2 -> 4, 5;  5 -> 6
    t = bare_tree([-1, 0, 0, 1, 2, 2, 5], [7])
    draft = [10, 11, 12, 13, 14, 15, 16]
    assert t.accept(draft, [12, 0, 15, 0, 0, 16, 99]) == ([[0, 2, 5, 6]], [[12, 15, 16, 99]])
    assert t.accept(draft, [77, 0, 0, 0, 0, 0, 0]) == ([[0]], [[77]])
    assert t.accept(draft, [11, 13, 0, 55, 0, 0, 0]) == ([[0, 1, 3]], [[11, 13, 55]])


def test_accept_takes_the_lowest_of_equal_children_and_ignores_other_roots():
    t = bare_tree([-1, 0, 0, 2, -1], [5])
    assert t.accept([1, 5, 5, 6, 5], [5, 8, 6, 0, 0]) == ([[0, 1]], [[5, 8]])


def test_accept_several_sequences_and_empty_ones():
    t = bare_tree([-1, 0, -1], [2, 0, 1])
    assert t.accept([4, 5, 9], [5, 6, 7]) == ([[0, 1], [], [0]], [[5, 6], [], [7]])
    # nothing allowed (-1) ends a path
    assert t.accept([4, 5, 9], [-1, 6, -1]) == ([[0], [], [0]], [[-1], [], [-1]])


def test_accept_refuses_other_sizes(dllm):
    t = bare_tree([-1, 0], [2])
    with pytest.raises(dllm.DllmError):
        t.accept([1], [1, 2])
    with pytest.raises(dllm.DllmError):
        t.accept([1, 2], [1, 2, 3])


@pytest.mark.parametrize("parents,counts,seqs", [([-1, 0], [1], None), ([-1], [2], None), ([-1, 0], [3, -1], None),
                                                 ([-1, -1], [1, 1], [0])])
def test_tree_counts_are_checked(dllm, parents, counts, seqs):
    with pytest.raises(dllm.DllmError):
        kernels.DraftTree(None, parents, counts, seqs)


@pytest.mark.parametrize("bad", [2 ** 32, -2 ** 32 - 1, 2 ** 31])
def test_numbers_beyond_32_bits_are_refused(dllm, bad):
    """An int64 array must not turn into other parents, counts, sequences or tokens."""
    for args in (([-1, bad], None, None), ([-1], [bad + 1], None), ([-1], [1], [bad])):
        with pytest.raises(dllm.DllmError):
            kernels.DraftTree(None, *(a if a is None else np.array(a, np.int64) for a in args))
    ctx = object.__new__(kernels.KernelContext)
    ctx.lib, ctx.handle, ctx.cfg = NoLibrary(), None, dllm.CFG
    leader = object.__new__(dllm.LeaderPipeline)
    leader.k, leader.lib, leader.singleNode, leader.handle = ctx, ctx.lib, True, None
    tree = bare_tree([-1, 0], [2])
    tree.handle = 8
    try:
        for draft in (np.array([1, bad], np.int64), np.array([1.0, 2.5])):
            with pytest.raises(dllm.DllmError):
                leader.verify_tree(tree, draft)
    finally:  # the handle is made up
        tree.handle = None


def test_rope_plan_names_are_checked(dllm):
    for kw in ({"layout": "spiral", "scaling": None}, {"layout": "half", "scaling": {"type": "cubic"}},
               {"layout": "half", "scaling": {"type": "linear", "factor": 2.0, "speed": 3}}):
        with pytest.raises(dllm.DllmError):
            kernels.RopePlan(None, kw["layout"], 64, 1e4, kw["scaling"])


def test_null_handles_are_refused(dllm):
    lib = dllm.load_library()
    out = C.c_void_p()
    one = (C.c_int32 * 1)(0)
    assert lib.dllm_tree_create(None, one, one, None, 1, C.byref(out)) == 1
    assert lib.dllm_rope_plan_create(None, None, C.byref(out)) == 1
    assert lib.dllm_rope_at(None, None, None, 1, None, None, None, None) == 1
    assert lib.dllm_pick_tokens(None, None) == 1
    assert lib.dllm_create_i32(None, 4, b"", C.byref(out)) == 1
    for fn in (lib.dllm_stage_append_tree, lib.dllm_stage_tree_attention):
        assert fn(None, 0, None, None, None) == 1
    assert lib.dllm_stage_commit_tree(None, None, None, None) == 1
    assert lib.dllm_stage_forward_tree(None, None, None, None, None) == 1
    assert not lib.dllm_stage_kv_device_ptr(None, 0)
    lib.dllm_tree_destroy(None)
    lib.dllm_rope_plan_destroy(None)


def test_a_wait_that_ran_out_is_told_where_it_ran_out(dllm):
    """Every kind of device error has a text of its own: the matmul's and the attention's waits too."""
    lib = dllm.load_library()
    csrc = os.path.join(os.path.dirname(dllm.LIB_PATH), "csrc")
    codes = {}
    for name in os.listdir(csrc):
        for const, value in re.findall(r"constexpr int (kErr\w+) = (\d+);", open(os.path.join(csrc, name)).read()):
            codes[const] = int(value)
    assert len(codes) >= 6 and len(set(codes.values())) == len(codes), codes
    texts = {const: lib.dllm_device_error_string(value).decode() for const, value in codes.items()}
    assert len(set(texts.values())) == len(codes) and lib.dllm_device_error_string(99).decode() not in texts.values()
    assert "matmul" in texts["kErrTcWait"]
    assert "attention" in texts["kErrTreeWait"]


def test_memory_of_freed_buffers_is_refused():
    b = kernels.GpuBuffer(None, None, 4, "f32", "gone")
    with pytest.raises(ValueError):
        b.__cuda_array_interface__


class NoLibrary:
    """Stands in for the library where no call may reach it."""

    def __getattr__(self, name):
        def call(*args):
            raise AssertionError(f"{name} was called")
        return call


def test_objects_of_another_kind_are_refused(dllm):
    """The library takes plain pointers: a buffer, a tree and a plan must not pass for one another."""
    ctx = object.__new__(kernels.KernelContext)
    ctx.lib, ctx.handle, ctx.cfg = NoLibrary(), None, dllm.CFG
    ctx.NQ, ctx.KVH, ctx.HD, ctx.D = 2, 2, 64, 8
    stage = object.__new__(dllm.Stage)
    stage.k, stage.lib, stage.handle, stage._owned = ctx, ctx.lib, 8, False
    stage.W = importlib.import_module("distributed-llm1_b200.pipeline")._StageWeights(stage)
    leader = object.__new__(dllm.LeaderPipeline)
    leader.k, leader.lib, leader.stage, leader.singleNode, leader.handle = ctx, ctx.lib, stage, True, None
    buf = kernels.GpuBuffer(ctx, 16, 2, "f32")
    tree = bare_tree([-1, 0], [2])
    plan = object.__new__(kernels.RopePlan)
    tree.handle, plan.handle, plan.ctx = 32, 48, ctx
    try:
        for wrong in (tree, plan, None, "buffer"):
            for call in (lambda: ctx.add(wrong, buf, 2), lambda: ctx.readF32(wrong, 2), lambda: ctx.readI32(wrong, 2),
                         lambda: ctx.ropeAt(plan, wrong, 2, buf), lambda: ctx.pickTokens(wrong, 2, tokens=buf),
                         lambda: stage.append_tree(0, tree, wrong, buf), lambda: stage.append_tree(0, tree, buf, wrong),
                         lambda: stage.tree_attention(0, tree, wrong, buf), lambda: stage.forward_tree(tree, wrong),
                         lambda: stage.W.__setitem__("model.norm.weight", wrong), lambda: leader.setLeaderWeights(tree)):
                with pytest.raises(ValueError):
                    call()
        for wrong in (tree, plan):
            for call in (lambda: ctx.ropeAt(plan, buf, 2, wrong), lambda: ctx.ropeAt(plan, buf, 2, buf, qOut=wrong),
                         lambda: stage.tree_attention(0, tree, buf, wrong), lambda: stage.forward_tree(tree, buf, wrong),
                         lambda: ctx.pickTokens(buf, 2, tokens=wrong), lambda: ctx.pickTokens(buf, 2, mask=wrong, tokens=buf)):
                with pytest.raises(ValueError):
                    call()
        for wrong in (buf, plan):
            for call in (lambda: stage.append_tree(0, wrong, buf, buf), lambda: stage.tree_attention(0, wrong, buf, buf),
                         lambda: stage.tree_attention(0, wrong, buf), lambda: stage.commit_tree(wrong, [[0]]),
                         lambda: stage.forward_tree(wrong, buf), lambda: leader.verify_tree(wrong, [1, 2]),
                         lambda: ctx.pickTokens(buf, 2, tree=wrong, draft=buf, tokens=buf)):
                with pytest.raises(ValueError):
                    call()
        for wrong in (buf, tree):
            with pytest.raises(ValueError):
                ctx.ropeAt(wrong, buf, 2, buf)
    finally:  # the handles are made up
        buf.handle = tree.handle = plan.handle = stage.handle = None


class LeaderLibrary:
    """A library whose leader lives at made-up addresses."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append(name)
            if name.endswith("_create"):
                args[-1]._obj.value = 16
            return {"dllm_leader_stage": 32, "dllm_stage_kv_device_ptr": 4096, "dllm_stage_pages_per_seq": 2}.get(name, 0)
        return call


def test_a_pool_keeps_the_leader_of_its_stage(dllm):
    """A leader frees its stage's cache when it goes; a pool in use must not lose it."""
    ctx = object.__new__(kernels.KernelContext)
    ctx.lib, ctx.handle, ctx.cfg = LeaderLibrary(), None, dllm.CFG
    leader = dllm.LeaderPipeline(ctx, (0, 1))
    pool = leader.stage.kv_pool("k")
    assert pool.__cuda_array_interface__["data"][0] == 4096
    del leader
    gc.collect()
    assert "dllm_leader_destroy" not in ctx.lib.calls
    del pool
    gc.collect()
    assert ctx.lib.calls.count("dllm_leader_destroy") == 1
    # without a pool nothing holds a leader
    leader = dllm.LeaderPipeline(ctx, (0, 1))
    stage = leader.stage
    del leader
    assert ctx.lib.calls.count("dllm_leader_destroy") == 2 and stage.handle is None
    with pytest.raises(ValueError):
        stage.kv_pool("v")
