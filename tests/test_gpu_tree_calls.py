"""Attention of trees: positions of the caller's own, in front of a token's row in the step, plans of the other kind, buffers that
grow, caches whose heads are copies."""

import pytest
import torch

from falcon_perception_amd import ops
from falcon_perception_amd.attention import compiled_flex_attn_decode
from falcon_perception_amd.paged_attention import PagedKVCache
from tests.draft_cases import DraftBatch, random_tree
from tests.shared_cases import SharedBatch

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


class Early(DraftBatch):
    """Tokens whose row in the step is beyond their position: what their masks name in front of position 0 is no key."""

    def seen(self, b, j, max_context=None):
        pos, mask = int(self.pos[b, j]), int(self.masks[b, j])
        if pos < 0:
            return []
        base = pos - j
        keys = list(range(base)) + [base + i for i in range(j + 1) if mask >> i & 1]
        return [t for t in keys if 0 <= t and (max_context is None or t < max_context)]


@pytest.mark.parametrize("share", [False, True])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("dtype,Hq", [(BF16, 4), (F16, 16), (F32, 2)])
def test_positions_in_front_of_a_tokens_row(dtype, Hq, index, share):
    gen = torch.Generator().manual_seed(51)
    case = Early(52, [64], [(-1, 0, [-1] * 64), (0, 20, [-1] * 64), (-1, 30, [-1] * 33), (-1, 0, [-1] * 6)], Hq=Hq, Hc=2, D=64, P=32, dtype=dtype, S=64)
    case.masks = torch.randint(-(1 << 62), 1 << 62, (4, 64), generator=gen)
    case.masks[0, 60:] = torch.tensor([-1, 1, 0, -(1 << 63)])
    case.masks[3] = 0
    case.masks[3, :6] = torch.tensor([1, 2, 4, 8, 16, 32])  # each sees itself alone
    case.pos[0] = torch.randint(-1, 64, (64,), generator=gen, dtype=torch.int32)
    case.pos[1] = torch.randint(0, 84, (64,), generator=gen, dtype=torch.int32)
    case.pos[2] = torch.arange(64, dtype=torch.int32) // 2
    case.pos[3] = torch.where(torch.arange(64) < 6, torch.tensor([0, 0, 0, 2, 2, 2] + [-1] * 58), torch.tensor(-1)).int()
    case.on()
    tree = ops.DraftTree(case.masks_d, case.pos_d.to(index), case.pos_d)
    case.check(case.call(ops, share=share, tree=tree))
    for room in (3, 40):
        case.check(case.call(ops, share=share, tree=tree, max_context=room), max_context=room)


def test_infinities_that_such_a_token_does_not_see():
    """The value of a key is infinite: tokens whose mask names it, counted from the tree's first position, get to know and no others."""
    case = Early(53, [], [(-1, 0, [-1] * 8)], Hq=2, Hc=1, D=64, P=16, dtype=BF16).on()
    case.pos = torch.tensor([[0, 1, 1, 2, 2, 2, 6, 7]], dtype=torch.int32)
    case.pos_d = case.pos.cuda()
    case.masks = torch.tensor([[1, 0b11, 0b110, 0b1110, 0b11000, 0b100000, 0b1000010, 0b10000000]])
    case.masks_d = case.masks.cuda()
    case.check(case.call(ops))
    at = int(case.table[case.batch_idx[0], 0]) * 16 + 1  # position 1
    case.pool_d[1][:, at, 9] = float("inf")
    out = case.call(ops)[0][0, 0, :, 9].float().cpu()
    sees = [1 in case.seen(0, j) for j in range(8)]
    assert sees.count(True) >= 3 and sees.count(False) >= 3
    assert torch.isinf(out).tolist() == sees


def test_plans_of_the_other_kind_are_foreign():
    """A plan says what it is of: with more than 64 rows of a sequence the two kinds cut them differently."""
    gen = torch.Generator().manual_seed(54)
    case = DraftBatch(55, [], [(-1, 200, list(range(-1, 39))), (-1, 9, list(range(-1, 33)))], Hq=8, Hc=2, D=64, P=32, dtype=BF16).on()
    shape = dict(q_heads=8, cached_heads=2, head_dim=64)
    room = case.columns * 32
    tree = ops.DraftTree(case.masks_d, case.pos_d, case.pos_d)
    of_trees = ops.tree_decode_plan(case.batch_idx_d, tree, case.table_d, max_context=room, prefix_ids=case.ids_d, prefix_lens=case.lens_d, **shape)
    of_shared = ops.shared_decode_plan(case.batch_idx_d, case.pos_d, case.ids_d, case.lens_d, max_context=room, **shape)
    case.check(case.call(ops, plan=of_trees))
    case.check(SharedBatch.call(case, ops, plan=of_shared))
    for got in (case.call(ops, plan=of_shared), SharedBatch.call(case, ops, plan=of_trees)):
        assert torch.isnan(got[0].float()).all() and torch.isnan(got[1]).all()


def test_graphs_captured_before_the_buffers_grew():
    """A step of one request in a graph; larger steps afterwards, which need other buffers, and smaller ones, which take them; the graph between
    them all.  Every step against a cache of its own."""
    gen = torch.Generator().manual_seed(57)
    Hq, Hc, D, L = 8, 2, 64, 2
    make = lambda: PagedKVCache(60, 32, 9, Hc, D, L, BF16)
    cache, twins = make(), {}
    slots = [cache.allocate() for _ in range(8)]
    for s in slots:
        cache.reserve(s, None, 200)
    table = cache.page_table.clone()
    rnd = lambda *s: torch.randn(s, generator=gen).to(BF16).cuda()
    cache._kv.copy_(rnd(*cache._kv.shape))
    start = cache._kv.clone()

    def step(c, parents, cached, rows):
        c._kv.copy_(start)
        batch_idx = idx[:parents.shape[0]]
        mask = c.create_tree_mask(batch_idx, parents, cached)
        outs = []
        for layer, (q, k, v) in enumerate(rows):
            pools = c.insert_kv(layer, k, v, input_pos=mask.input_pos, batch_idx=batch_idx)
            outs += compiled_flex_attn_decode(q, *pools, block_mask=mask, return_lse=True)
        return outs

    def inputs(B, S):
        parents = torch.tensor([random_tree(gen, S, 1 + b % 4) for b in range(B)], dtype=torch.int32).cuda()
        cached = torch.randint(0, 130, (B,), generator=gen, dtype=torch.int32).cuda()
        return parents, cached, [(rnd(B, Hq, S, D), rnd(B, Hc, S, D), rnd(B, Hc, S, D)) for _ in range(L)]

    def alone(B, S, args):
        if (B, S) not in twins:
            twins[B, S] = make()
            twins[B, S].page_table.copy_(table)
        return step(twins[B, S], *args)

    idx = torch.tensor(slots, device="cuda")
    one = inputs(1, 3)
    step(cache, *one)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(cache, *one)
    for B, S in ((1, 3), (2, 5), (8, 20), (3, 7), (8, 64), (1, 1), (8, 20), (2, 64)):
        args = inputs(B, S)
        for x, y in zip(step(cache, *args), alone(B, S, args)):
            assert torch.equal(x, y)
        new = inputs(1, 3)
        for x, y in zip((one[0], one[1], *(t for r in one[2] for t in r)), (new[0], new[1], *(t for r in new[2] for t in r))):
            x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(captured, alone(1, 3, one)):
            assert torch.equal(x, y)
    assert len(cache._tree_buffers) == 1 and len(cache._retired_workspaces) >= 2


@pytest.mark.parametrize("sharing", [False, True])
@pytest.mark.parametrize("fuse", [False, True])
def test_a_cache_whose_heads_are_copies(fuse, sharing):
    """One cached head a query head, V copied in pairs: trees read every cached head and answer as a cache of the heads by themselves."""
    gen = torch.Generator().manual_seed(56)
    H, Hkv, D, L = 8, 4, 64, 2
    wide = PagedKVCache(40, 16, 5, H, D, L, BF16, kv_rep=2, prefix_sharing=sharing, fuse_decode_append=fuse)
    plain = PagedKVCache(40, 16, 5, H, D, L, BF16, kv_rep=1, prefix_sharing=sharing, fuse_decode_append=fuse)
    rnd = lambda *s: torch.randn(s, generator=gen).to(BF16).cuda()
    lens, S = [37, 5, 0], 6
    slots = []
    for cache in (wide, plain):
        slots.append([cache.allocate() for _ in lens])
        for s, n in zip(slots[-1], lens):
            cache.reserve(s, None, n + S)
    assert slots[0] == slots[1]
    batch_idx = torch.tensor(slots[0], device="cuda")
    pair = lambda t: t.repeat_interleave(2, 1)
    for i in range(max(lens)):
        have = torch.tensor([[i] if i < n else [-1] for n in lens], dtype=torch.int32).cuda()
        for layer in range(L):
            k, v = rnd(3, H, 1, D), pair(rnd(3, Hkv, 1, D))
            for cache in (wide, plain):
                cache.assign(layer, batch_idx, have, k, v)
                cache.flush()
    parents = torch.tensor([random_tree(gen, S, r) for r in (1, 2, 6)], dtype=torch.int32).cuda()
    cached = torch.tensor(lens, dtype=torch.int32).cuda()
    masks = [cache.create_tree_mask(batch_idx, parents, cached) for cache in (wide, plain)]
    for layer in range(L):
        k, v, q = rnd(3, H, S, D), pair(rnd(3, Hkv, S, D)), rnd(3, H, S, D)
        outs = []
        for cache, mask in zip((wide, plain), masks):
            pools = cache.insert_kv(layer, k, v, input_pos=mask.input_pos, batch_idx=batch_idx)
            outs.append(compiled_flex_attn_decode(q, *pools, block_mask=mask, return_lse=True))
        for x, y in zip(*outs):
            assert torch.equal(x, y)
        # against the definition, one request at a time
        for b, n in enumerate(lens):
            seen = masks[0].tree.masks[b].tolist()
            rows = torch.arange(n + S, device="cuda")
            at = wide.page_table[batch_idx[b], rows // 16] * 16 + rows % 16
            kk, vv = (wide.kv_cache[layer, i, 0][:, at].double().cpu() for i in range(2))
            hide = torch.tensor([[t >= n and not seen[j] >> (t - n) & 1 for t in range(n + S)] for j in range(S)])
            x = torch.bmm(q[b].double().cpu(), kk.transpose(1, 2).contiguous()) * D ** -0.5
            want = torch.bmm(torch.softmax(x.masked_fill(hide, -torch.inf), 2), vv)
            # rounded once to bf16; sums of 50 keys in 32 bits
            assert (outs[0][0][b].double().cpu() - want).abs().max() <= 2.0 ** -8 * want.abs().max() + 1e-4
