"""Sizes of calls on drafted tokens: workspaces that serve smaller calls, calls past one dispatch, buffers of a cache that grow."""

import ctypes

import pytest
import torch

from falcon_perception_amd import ops
from falcon_perception_amd.paged_attention import PagedKVCache

P = ctypes.c_void_p(4096)  # a pointer that is never followed


@pytest.mark.parametrize("V", [1, 500, 4096, 32000, 65536, 150001, 1 << 24])
def test_a_verification_workspace_serves_every_smaller_call(native_lib, V):
    """Fewer requests, fewer rows, a smaller vocabulary: of what a program asks for its largest call it can run all others."""
    largest = 0
    for B in range(1, 65):
        n = ops.verify_workspace_bytes(B, 16, V)
        assert n >= largest, (B, n, largest)
        largest = n
    for S in (1, 2, 7, 16, 33, 64):
        sizes = [ops.verify_workspace_bytes(B, S, V) for B in (1, 2, 3, 5, 6, 9, 24, 25, 64, 130)]
        assert sizes == sorted(sizes), (S, sizes)
    for B in (1, 6, 24, 64):
        sizes = [ops.verify_workspace_bytes(B, S, V) for S in range(1, 65)]
        assert sizes == sorted(sizes), (B, sizes)
    sizes = [ops.verify_workspace_bytes(6, 16, v) for v in sorted({1, 7, 1000, 4096, 4097, 32000, 32769, 65536, V})]
    assert sizes == sorted(sizes)


def test_a_workspace_is_not_much_larger_than_its_call(native_lib):
    assert ops.verify_workspace_bytes(1, 1, 1) < 1 << 17
    # 512 requests of 33 rows of 65536: 4 chunks of 16384 a row, 256 pieces of 256 a request
    assert ops.verify_workspace_bytes(512, 33, 65536) < 512 * (33 * 4 * 16 + 256 * 32) + (1 << 18)


@pytest.mark.parametrize("B,S,V,fits", [(1 << 18, 64, 1000, False), ((1 << 18) - 1, 64, 1000, True), (1 << 24, 1, 5, False), ((1 << 24) - 1, 1, 5, True),
                                        (1 << 19, 1, 1 << 18, False), (1 << 20, 64, 1, False), (1 << 30, 1, 1, False)])
def test_verifications_past_one_dispatch(native_lib, B, S, V, fits):
    """A dispatch has fewer than 2^32 lanes: 2^24 workgroups, of a row's chunk or of a request's share of the row that is drawn from."""
    n = native_lib.fp_verify_drafts_workspace_bytes(B, S, V)
    if fits:
        assert n > 0
        return
    assert n == -2 and "too many" in native_lib.fp_last_error().decode()
    for dtype in (0, 1, 2):
        rc = native_lib.fp_verify_drafts(P, S * V, V, dtype, P, P, P, None, None, 0, 0, 0, P, P, P, P, P, 1 << 50, B, S, V, None)
        assert rc == -2 and "too many" in native_lib.fp_last_error().decode()


def test_elements_of_32_bits_reach_the_end_of_a_dispatch_first(native_lib):
    """16 bits: 2^18 requests of 32 rows of 32768 are 2^23 workgroups; of 32 bits they are 2^24, and too many."""
    B, S, V = 1 << 18, 32, 32768
    assert native_lib.fp_verify_drafts_workspace_bytes(B, S, V) > 0
    rc = native_lib.fp_verify_drafts(P, S * V, V, 0, P, P, P, None, None, 0, 0, 0, P, P, P, P, P, 1 << 50, B, S, V, None)
    assert rc == -2 and "too many" in native_lib.fp_last_error().decode()


def test_trees_past_one_dispatch(native_lib):
    for B in (1 << 26, (1 << 26) - 3, 2 ** 31 - 1):
        assert native_lib.fp_draft_tree(P, P, 0, B, 64, P, P, P, None) == -2 and "too many" in native_lib.fp_last_error().decode()


def test_attention_past_one_dispatch(native_lib):
    """Rows of the join, D / 4 lanes each, and a workgroup a cached head of the products."""
    for size in (native_lib.fp_shared_decode_plan_bytes, native_lib.fp_shared_decode_workspace_bytes):
        assert size(1024, 64, 8 * 256, 256, 128) == -2 and "too many" in native_lib.fp_last_error().decode()
        assert size(1024, 64, 8 * 255, 255, 128) > 0
        assert size(1, 1, 1 << 24, 1 << 24, 64) == -2 and "too many" in native_lib.fp_last_error().decode()


def retained(cache):
    held = {t.data_ptr(): t.numel() for t in cache._retired_workspaces}
    held.update({t.data_ptr(): t.numel() for hit in cache._tree_buffers.values() for t in hit[:2]})
    return sum(held.values())


@pytest.mark.parametrize("order", ["batch", "tokens", "down"])
def test_buffers_of_trees_are_bounded(native_lib, order):
    """Batches that grow one request at a time, steps of every number of tokens: what a cache holds on to is within four times what its
    largest step needs."""
    cache = PagedKVCache(8, 16, 80, 8, 128, 1, torch.bfloat16, device="cpu")
    Hq, Hc, D = 32, 8, 128
    shape = dict(q_heads=Hq, cached_heads=Hc, head_dim=D)
    steps = {"batch": [(B, S) for B in range(1, 65) for S in (3, 24)], "tokens": [(B, S) for S in range(1, 65) for B in (2, 17, 64)],
             "down": [(B, S) for B in range(64, 0, -9) for S in range(64, 0, -1)]}[order]
    largest = 0
    for B, S in steps:
        plan, workspace = cache.tree_decode_buffers(B, S, Hq, Hc, D)
        need = ops.shared_decode_plan_bytes(B, S, **shape), ops.shared_decode_workspace_bytes(B, S, **shape)
        assert plan.numel() >= need[0] and workspace.numel() >= need[1] and plan.dtype == workspace.dtype == torch.uint8
        again = cache.tree_decode_buffers(B, S, Hq, Hc, D)
        assert again[0] is plan and again[1] is workspace
        largest = max(largest, sum(need))
    assert retained(cache) <= 4 * largest


def test_a_plan_that_moved_is_made_again(native_lib):
    """Of larger buffers the plan of the step in flight is not in the new one; where they stay, it stands."""
    cache = PagedKVCache(8, 16, 80, 2, 64, 1, torch.bfloat16, device="cpu")
    first = cache.tree_decode_buffers(8, 8, 4, 2, 64)
    cache._tree_plan_owner = owner = object()
    assert cache.tree_decode_buffers(3, 5, 4, 2, 64)[0] is first[0] and cache._tree_plan_owner is owner
    more = cache.tree_decode_buffers(40, 64, 4, 2, 64)
    assert more[0] is not first[0] and cache._tree_plan_owner is None
    assert any(t is first[0] for t in cache._retired_workspaces)  # a graph captured with it still writes to it
    assert cache.tree_decode_buffers(40, 64, 8, 2, 64)[0] is not more[0]
