"""What the entry points for shared prefixes refuse, and the sizes they ask for: no GPU is touched."""

import ctypes

import pytest
import torch

from falcon_perception_amd import ops
from falcon_perception_amd.paged_attention import PagedKVCache

P = ctypes.c_void_p(4096)  # a pointer that is never followed


def error(lib):
    return lib.fp_last_error().decode()


def tables(lib, **kw):
    a = dict(slots=P, old=P, new=P, idx=0, parents=None, free=P, count=ctypes.c_void_p(8192), n_free=4, table=P, stride=8, inverse=None, inv_stride=0,
             inv_cols=0, bidx=P, pos=P, smap=P, starts=P, left=P, src=P, dst=P, rows=P, status=P, B=2, max_rows=4, multiple=1, page=16, cols=8,
             batch=4, stream=None)
    a.update(kw)
    return lib.fp_step_tables(*a.values())


@pytest.mark.parametrize("change,code,text", [
    (dict(page=0), -1, "page_size=0"), (dict(multiple=0), -1, "row_multiple=0"), (dict(B=-1), -1, "B=-1"), (dict(max_rows=-1), -1, "max_rows=-1"),
    (dict(batch=0), -1, "max_batch=0"), (dict(n_free=-1), -1, "n_free=-1"), (dict(idx=2), -1, "len_index_type 2"),
    (dict(B=5000), -2, "at most 4096 requests"), (dict(batch=1 << 18), -2, "131072 slots"), (dict(slots=None), -1, "null pointer"),
    (dict(status=None), -1, "null pointer"), (dict(bidx=None), -1, "null pointer"), (dict(left=ctypes.c_void_p(8192)), -1, "may not be free_count"),
])
def test_step_tables_refuses(native_lib, change, code, text):
    assert tables(native_lib, **change) == code and text in error(native_lib)


@pytest.mark.parametrize("change,code,text", [
    (dict(dtype=7), -2, "dtype code 7"), (dict(D=7), -1, "bad sizes"), (dict(n=-1), -1, "bad sizes"), (dict(n=70000), -2, "65535 pages"),
    (dict(src=None), -1, "null pointer"), (dict(pool=ctypes.c_void_p(4104)), -1, "16-byte aligned"), (dict(page=0), -1, "bad sizes"),
])
def test_copy_pages_refuses(native_lib, change, code, text):
    a = dict(pool=P, src=P, dst=P, rows=P, n=2, planes=4, slots=64, D=64, page=16, dtype=1, stream=None)
    a.update(change)
    assert native_lib.fp_copy_pages(*a.values()) == code and text in error(native_lib)


def test_nothing_to_copy(native_lib):
    assert native_lib.fp_copy_pages(None, None, None, None, 0, 4, 64, 64, 16, 1, None) == 0
    assert native_lib.fp_copy_pages(None, None, None, None, 3, 0, 64, 64, 16, 1, None) == 0


def attend(lib, **kw):
    a = dict(q=P, qb=256, qh=64, qs=64, pk=P, pv=P, table=P, stride=8, bidx=P, pos=P, idx=0, out=P, ob=256, oh=64, os=64, lse=P, sinks=None, ws=P,
             ws_bytes=1 << 40, plan=P, plan_bytes=1 << 40, B=2, S=1, Hq=4, Hc=2, D=64, page=16, cols=8, batch=4, slots=640, room=128, scale=0.1,
             dtype=1, stream=None)
    a.update(kw)
    return lib.fp_paged_decode_shared(*a.values())


@pytest.mark.parametrize("change,code,text", [
    (dict(D=96), -2, "head_dim 96"), (dict(Hq=6), -2, "3 query heads"), (dict(Hq=5), -1, "bad sizes"), (dict(S=0), -1, "bad sizes"),
    (dict(B=4000), -2, "at most 1536 sequences"), (dict(B=1500, S=1024), -2, "rows a cached head"), (dict(dtype=5), -2, "dtype code 5"),
    (dict(page=0), -1, "page_size=0"), (dict(room=0), -1, "max_context=0"), (dict(room=1 << 22), -2, "at most 2097152"), (dict(slots=8), -1, "n_slots=8"),
    (dict(idx=3), -1, "pos_index_type 3"), (dict(q=None), -1, "null pointer"), (dict(plan=None), -1, "null pointer"),
    (dict(qh=63), -1, "16-byte aligned"), (dict(out=ctypes.c_void_p(4104)), -1, "16-byte aligned"), (dict(plan_bytes=64), -4, "too small"),
    (dict(ws=None), -4, "is needed"), (dict(ws_bytes=100), -4, "is needed"), (dict(ws=ctypes.c_void_p(4104)), -4, "is needed"),
])
def test_attention_refuses(native_lib, change, code, text):
    assert attend(native_lib, **change) == code and text in error(native_lib)


@pytest.mark.parametrize("change,code,text", [
    (dict(batch=0), -1, "max_batch 0"), (dict(room=0), -1, "max_context 0"), (dict(room=1 << 22), -2, "at most 2097152"), (dict(ids=None), -1, "null pointer"),
    (dict(plan_bytes=100), -4, "the plan needs"), (dict(plan=ctypes.c_void_p(4104)), -4, "16-byte aligned"), (dict(Hc=3), -1, "bad sizes"),
    (dict(idx=9), -1, "pos_index_type 9"),
])
def test_plan_refuses(native_lib, change, code, text):
    a = dict(bidx=P, pos=P, idx=0, ids=P, lens=P, B=2, S=1, Hq=4, Hc=2, D=64, batch=4, room=128, plan=P, plan_bytes=1 << 40, stream=None)
    a.update(change)
    assert native_lib.fp_shared_decode_plan(*a.values()) == code and text in error(native_lib)


def test_sizes_grow_with_the_batch(native_lib):
    for Hq, Hc, D in ((4, 2, 64), (32, 8, 128), (8, 8, 128), (16, 2, 64)):
        shape = dict(q_heads=Hq, cached_heads=Hc, head_dim=D)
        for size in (ops.shared_decode_plan_bytes, ops.shared_decode_workspace_bytes):
            got = [size(B, 1, **shape) for B in (1, 2, 7, 64, 257, 1536)]
            assert got == sorted(got) and got[0] > 0
            assert size(64, 3, **shape) > size(64, 1, **shape)
    with pytest.raises(RuntimeError, match="head_dim 80"):
        ops.shared_decode_plan_bytes(1, 1, q_heads=4, cached_heads=2, head_dim=80)


def test_an_empty_batch_is_no_launch(native_lib):
    assert attend(native_lib, B=0) == 0


def test_operators_refuse_the_cpu():
    cpu = torch.zeros(4, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.step_tables(cpu, cpu, cpu, cpu, cpu.int(), cpu.view(2, 2), 16, 4)
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.copy_pages(torch.zeros(2, 32, 64), cpu, cpu, cpu.int(), 16)
    cache = PagedKVCache(16, 16, 4, 2, 64, 1, torch.float32, device="cpu")
    slot = cache.allocate()
    cache.reserve(slot, None, 40)
    before = (list(cache.free_pages), list(cache.free_batch_idx))
    for call in (lambda: cache.fork(slot, 20), lambda: cache.step_tables([slot], [40], [50])):
        with pytest.raises(RuntimeError, match="GPU only"):
            call()
    assert before == (cache.free_pages, cache.free_batch_idx)


def test_shapes_of_more_than_32_bits_are_refused(native_lib):
    shape = dict(q_heads=8, cached_heads=8, head_dim=64)
    for size in (ops.shared_decode_plan_bytes, ops.shared_decode_workspace_bytes):
        for B, S, change in ((1 << 32) + 2, 1, {}), (2, (1 << 32) + 1, {}), (2, 1, dict(q_heads=(1 << 32) + 8)), (2, 1, dict(head_dim=(1 << 32) + 64)):
            with pytest.raises(RuntimeError, match="does not fit 32 bits"):
                size(B, S, **(shape | change))


def test_the_limits_have_one_name_each(native_lib):
    """What the decode path of a sharing cache takes as the limits of one call are those of the library."""
    for B, room, code in ((ops.SHARED_SEQUENCES, ops.SHARED_CONTEXT, -1), (ops.SHARED_SEQUENCES + 1, ops.SHARED_CONTEXT, -2),
                          (ops.SHARED_SEQUENCES, ops.SHARED_CONTEXT + 1, -2)):
        assert attend(native_lib, B=B, room=room, q=None) == code
