"""Which decode calls of a cache with prefix_sharing go over shared prefixes, and what the others do instead."""

import pytest
import torch
from torch.nn.attention.flex_attention import AuxRequest, BlockMask

from falcon_perception_amd import attention as A
from falcon_perception_amd import ops
from falcon_perception_amd.paged_attention import PagedKVCache
from tests.test_gpu_prefix_sharing import DEV, Server

pytestmark = pytest.mark.gpu


def decode_alike(monkeypatch, B, room, n_pages, slots, P, *, shared):
    """Two layers of a decode step of B forks of 40 tokens, on a cache with prefix_sharing and on one without it: bit for bit alike
    where the step does not go over shared prefixes."""
    calls = []
    real = ops.paged_decode_shared
    monkeypatch.setattr(ops, "paged_decode_shared", lambda *a, **kw: calls.append(1) or real(*a, **kw))
    got = []
    for sharing in (True, False):
        s = Server(prefix_sharing=sharing, n_pages=n_pages, P=P, slots=slots, Hc=1, Hq=2, layers=2, max_blocks_per_seq=-(-room // P), seed=3)
        idx = [s.picture(40)]
        idx += s.fork(idx[0], 40, B - 1)
        s.cache.step_tables(idx, [40] * B, [41] * B)
        pos = torch.full((B,), 40, dtype=torch.int32, device=DEV)
        n = torch.full((B, 1, 1), 40 // P + 1, dtype=torch.int32, device=DEV)
        logical = BlockMask.from_kv_blocks(n, torch.zeros(B, 1, 1, 2, dtype=torch.int32, device=DEV), None, None,
                                           BLOCK_SIZE=(P, P), mask_mod=lambda b, h, q, kv: q + pos[b] >= kv, seq_lengths=(1, room))
        mask = s.cache.convert_logical_block_mask(logical, torch.tensor(idx, device=DEV))
        assert mask.max_context == room
        for layer in range(2):
            q, k, v = s.rnd(B, 2, 1, s.D), s.rnd(B, 1, 1, s.D), s.rnd(B, 1, 1, s.D)
            K, V = s.cache.insert_kv(layer, k.to(DEV), v.to(DEV), input_pos=pos.view(-1, 1), batch_idx=mask.batch_idx)
            out, aux = A.compiled_flex_attn_decode(q.to(DEV), K, V, block_mask=mask, return_aux=AuxRequest(lse=True))
            got += [out, aux.lse]
            if sharing:
                keys = [tuple(torch.cat([old, new[i]], 1) for old, new in zip(s.keys[x][layer], (k, v))) for i, x in enumerate(idx)]
                s.expected(q, keys, pos.cpu()).check((out, aux.lse))
    assert len(calls) == 2 * shared
    if not shared:
        assert all(torch.equal(x, y) for x, y in zip(got[:4], got[4:]))


@pytest.mark.parametrize("B,shared", [(1536, True), (1537, False), (1700, False)])
def test_batches_of_any_size_decode(monkeypatch, B, shared):
    decode_alike(monkeypatch, B, 128, 2 * 1800, 1800, 32, shared=shared)


@pytest.mark.parametrize("room,shared", [(1 << 21, True), ((1 << 21) + 128, False)])
def test_contexts_of_any_size_decode(monkeypatch, room, shared):
    decode_alike(monkeypatch, 3, room, (1 << 14) + 2, 5, 128, shared=shared)


def test_a_first_use_inside_a_capture_clears_nothing_in_replays():
    """The buffers of a step whose first call is a graph's: a replay writes what the launch writes, not the whole buffers (some 70 MB
    for a cache of 1536 slots)."""
    s = Server(slots=400)
    cat = s.picture(133)
    idx = [cat, *s.fork(cat, 133, 2)]
    s.cache.step_tables(idx, [133] * 3, [134] * 3)
    pos = torch.full((3,), 133, dtype=torch.int32, device=DEV)
    mask, ids = s.mask(idx, pos), torch.tensor(idx, device=DEV)
    q, k, v = (s.rnd(3, h, 1, s.D).to(DEV) for h in (s.Hq, s.Hc, s.Hc))

    def step():
        K, V = s.cache.insert_kv(0, k, v, input_pos=pos.view(-1, 1), batch_idx=ids)
        return A.compiled_flex_attn_decode(q, K, V, block_mask=mask)

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    plan, workspace = s.cache.shared_decode_buffers(3, s.Hq, s.Hc, s.D)
    assert workspace.numel() > 1 << 20
    for _ in range(3):
        plan.fill_(0x5b)
        workspace.fill_(0x5b)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert bool((workspace[-4096:] == 0x5b).all()) and bool((plan[-256:] == 0x5b).all())
        want = step()
        assert torch.equal(out, want) and bool(torch.isfinite(want).all())


@pytest.mark.parametrize("dtype,D,heads,rep", [(torch.bfloat16, 128, 16, 2), (torch.float16, 64, 8, 4), (torch.float32, 64, 4, 2)])
@pytest.mark.parametrize("graph", [False, True])
def test_a_cache_whose_heads_are_copies(dtype, D, heads, rep, graph):
    """One cached head a query head, V (and K) the same in groups of `kv_rep`, as an engine caches them; the append left to the attention."""
    s = Server(Hc=heads, Hq=heads, D=D, dtype=dtype, kv_rep=rep, fuse_decode_append=True, layers=2, seed=12)
    rnd = s.rnd

    def copies(*shape):  # rows of K and V: groups of heads are alike; [.., heads, tokens, D]
        if len(shape) == 4 and shape[1] == heads:
            return rnd(shape[0], heads // rep, *shape[2:]).repeat_interleave(rep, 1)
        return rnd(*shape)

    s.rnd = copies
    cat, dog = s.picture(133), s.picture(70)
    idx = [cat, *s.fork(cat, 133, 4), dog, *s.fork(dog, 64, 2)]
    s.extend(idx, [1 + 5 * i for i in range(len(idx))])
    assert s.cache.v_copies_are_identical(0) and s.cache.v_copies_are_identical(1)
    if not graph:
        for batch in (idx, idx[::-1], idx[2:4]):
            s.decode(batch)
        s.check_pool()
        return
    lens = [s.length(x) for x in idx]
    for x, n in zip(idx, lens):
        s.cache.reserve(x, None, n + 3)
    pos = torch.tensor(lens, dtype=torch.int32, device=DEV)
    mask, ids = s.mask(idx, pos), torch.tensor(idx, device=DEV)
    q, k, v = (torch.zeros(2, len(idx), heads, 1, D, dtype=dtype, device=DEV) for _ in range(3))

    def step():
        got = []
        for layer in range(2):
            K, V = s.cache.insert_kv(layer, k[layer], v[layer], input_pos=pos.view(-1, 1), batch_idx=ids)
            out, aux = A.compiled_flex_attn_decode(q[layer], K, V, block_mask=mask, return_aux=AuxRequest(lse=True))
            got.append((out, aux.lse))
        return got

    step()
    torch.cuda.synchronize()
    captured = torch.cuda.CUDAGraph()
    with torch.cuda.graph(captured):
        made = step()
    for turn in range(3):
        for t in (q, k, v):
            for layer in range(2):
                t[layer].copy_(s.rnd(len(idx), heads, 1, D))
        captured.replay()
        torch.cuda.synchronize()
        for layer in range(2):
            for i, x in enumerate(idx):
                s.keys[x][layer] = tuple(torch.cat([old, new[layer, i].cpu()], 1) for old, new in zip(s.keys[x][layer], (k, v)))
            s.expected(q[layer].cpu(), [s.keys[x][layer] for x in idx], pos.cpu()).check(made[layer])
        pos.add_(1)
    s.check_pool()
