"""What the entry points for drafted tokens refuse, and the sizes they ask for: no GPU is touched."""

import ctypes

import pytest
import torch

from falcon_perception_amd import ops

P = ctypes.c_void_p(4096)  # a pointer that is never followed
ODD = ctypes.c_void_p(4104)


def error(lib):
    return lib.fp_last_error().decode()


@pytest.mark.parametrize("change,code,text", [
    (dict(B=-1), -1, "B=-1"), (dict(S=0), -1, "S=0"), (dict(S=65), -2, "at most 64 tokens"), (dict(idx=2), -1, "cached_index_type 2"),
    (dict(parents=None), -1, "null pointer"), (dict(cached=None), -1, "null pointer"), (dict(masks=None), -1, "null pointer"),
    (dict(pos=None), -1, "null pointer"), (dict(rope=None), -1, "null pointer"),
])
def test_draft_tree_refuses(native_lib, change, code, text):
    a = dict(parents=P, cached=P, idx=0, B=2, S=4, masks=P, pos=P, rope=P, stream=None)
    a.update(change)
    assert native_lib.fp_draft_tree(*a.values()) == code and text in error(native_lib)


def attend(lib, **kw):
    a = dict(masks=P, q=P, qb=256, qh=64, qs=64, pk=P, pv=P, table=P, stride=8, bidx=P, pos=P, idx=0, out=P, ob=256, oh=64, os=64, lse=P,
             sinks=None, ws=P, ws_bytes=1 << 40, plan=P, plan_bytes=1 << 40, B=2, S=1, Hq=4, Hc=2, D=64, page=16, cols=8, batch=4, slots=640,
             room=128, scale=0.1, dtype=1, stream=None)
    a.update(kw)
    return lib.fp_paged_decode_tree(*a.values())


@pytest.mark.parametrize("change,code,text", [
    (dict(masks=None), -1, "null pointer"), (dict(S=65), -2, "at most 64 tokens"), (dict(D=96), -2, "head_dim 96"), (dict(Hq=6), -2, "3 query heads"),
    (dict(S=0), -1, "bad sizes"), (dict(B=4000), -2, "at most 1536 sequences"), (dict(dtype=5), -2, "dtype code 5"), (dict(page=0), -1, "page_size=0"),
    (dict(room=1 << 22), -2, "at most 2097152"), (dict(idx=3), -1, "pos_index_type 3"), (dict(q=None), -1, "null pointer"),
    (dict(qh=63), -1, "16-byte aligned"), (dict(plan_bytes=64), -4, "too small"), (dict(ws=None), -4, "is needed"), (dict(ws=ODD), -4, "is needed"),
])
def test_attention_refuses(native_lib, change, code, text):
    assert attend(native_lib, **change) == code and text in error(native_lib) and "fp_paged_decode_tree" in error(native_lib)


@pytest.mark.parametrize("change,code,text", [
    (dict(S=65), -2, "at most 64 tokens"), (dict(batch=0), -1, "max_batch 0"), (dict(room=0), -1, "max_context 0"), (dict(ids=P), -1, "null pointer"),
    (dict(lens=P), -1, "null pointer"), (dict(plan_bytes=100), -4, "the plan needs"), (dict(plan=ODD), -4, "16-byte aligned"),
])
def test_plan_refuses(native_lib, change, code, text):
    a = dict(bidx=P, pos=P, idx=0, ids=None, lens=None, B=2, S=5, Hq=4, Hc=2, D=64, batch=4, room=128, plan=P, plan_bytes=1 << 40, stream=None)
    a.update(change)
    assert native_lib.fp_tree_decode_plan(*a.values()) == code and text in error(native_lib)


@pytest.mark.parametrize("change,code,text", [
    (dict(B=-1), -1, "B=-1"), (dict(S=0), -1, "S=0"), (dict(V=0), -1, "V=0"), (dict(S=65), -2, "at most 64 tokens"),
    (dict(V=(1 << 24) + 1), -2, "16777216"), (dict(B=1 << 21, S=64, V=1 << 16), -2, "too many"), (dict(dtype=3), -2, "dtype code 3"),
    (dict(probs=P, pdtype=9), -2, "dtype code 9"), (dict(logits=None), -1, "null pointer"), (dict(tokens=None), -1, "null pointer"),
    (dict(parents=None), -1, "null pointer"), (dict(uniforms=None), -1, "null pointer"), (dict(accepted=None), -1, "null pointer"),
    (dict(path=None), -1, "null pointer"), (dict(answer=None), -1, "null pointer"), (dict(logprobs=None), -1, "null pointer"),
    (dict(logits=ctypes.c_void_p(4097)), -1, "aligned to their elements"), (dict(probs=ctypes.c_void_p(4098)), -1, "aligned to their elements"),
    (dict(ws=None), -4, "is needed"), (dict(ws=ODD), -4, "is needed"), (dict(ws_bytes=100), -4, "is needed"),
])
def test_verify_drafts_refuses(native_lib, change, code, text):
    a = dict(logits=P, lb=4000, ls=1000, dtype=1, tokens=P, parents=P, uniforms=P, temperatures=None, probs=None, pb=4000, ps=1000, pdtype=0,
             accepted=P, path=P, answer=P, logprobs=P, ws=P, ws_bytes=1 << 40, B=2, S=4, V=1000, stream=None)
    a.update(change)
    assert native_lib.fp_verify_drafts(*a.values()) == code and text in error(native_lib)


@pytest.mark.parametrize("change,code,text", [
    (dict(dtype=7), -2, "dtype code 7"), (dict(D=7), -1, "bad sizes"), (dict(B=-1), -1, "bad sizes"), (dict(S=0), -1, "bad sizes"),
    (dict(S=65), -2, "64 rows"), (dict(B=65536), -2, "65535 sequences"), (dict(D=4096), -2, "4096 bytes"), (dict(page=0), -1, "bad sizes"),
    (dict(cols=0), -1, "bad sizes"), (dict(batch=0), -1, "bad sizes"), (dict(idx=4), -1, "cached_index_type 4"), (dict(path=None), -1, "null pointer"),
    (dict(table=None), -1, "null pointer"), (dict(pool=ODD), -1, "16-byte aligned"),
])
def test_keep_rows_refuses(native_lib, change, code, text):
    a = dict(pool=P, table=P, stride=8, bidx=P, cached=P, idx=0, path=P, B=2, S=4, planes=4, slots=64, D=64, page=16, cols=4, batch=4, dtype=1,
             stream=None)
    a.update(change)
    assert native_lib.fp_keep_rows(*a.values()) == code and text in error(native_lib)


def test_nothing_to_do(native_lib):
    assert native_lib.fp_draft_tree(None, None, 0, 0, 5, None, None, None, None) == 0
    assert native_lib.fp_keep_rows(None, None, 8, None, None, 0, None, 0, 4, 4, 64, 64, 16, 4, 4, 1, None) == 0
    assert native_lib.fp_keep_rows(None, None, 8, None, None, 0, None, 3, 4, 0, 64, 64, 16, 4, 4, 1, None) == 0
    assert native_lib.fp_verify_drafts(None, 0, 0, 1, None, None, None, None, None, 0, 0, 0, None, None, None, None, None, 0, 0, 4, 100, None) == 0
    assert attend(native_lib, B=0, q=None) == 0


def test_workspace_grows_with_the_call(native_lib):
    assert ops.verify_workspace_bytes(0, 4, 1000) == 0
    one = ops.verify_workspace_bytes(1, 1, 1)
    assert 0 < one < ops.verify_workspace_bytes(64, 8, 65536) < 1 << 24
    with pytest.raises(RuntimeError, match="at most 64 tokens"):
        ops.verify_workspace_bytes(1, 65, 100)
    with pytest.raises(RuntimeError, match="does not fit 32 bits"):
        ops.verify_workspace_bytes(1, 1, 1 << 32)


def test_operators_run_on_the_gpu_only():
    parents, cached = torch.full((2, 3), -1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.draft_tree(parents, cached)
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.verify_drafts(torch.zeros(2, 3, 10), torch.zeros(2, 3, dtype=torch.int64), parents, torch.zeros(2, 3))
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.keep_rows(torch.zeros(2, 2, 32, 64), torch.zeros(3, 2, dtype=torch.int64), torch.ones(2, dtype=torch.int64), cached, parents, 16)
