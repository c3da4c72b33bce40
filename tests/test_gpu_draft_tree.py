"""Trees of drafted tokens: what each sees, and attention over the paged cache against float64 (tolerances: DraftBatch.expect)."""

import pytest
import torch

from falcon_perception_amd import ops
from tests.draft_cases import DraftBatch, random_tree, tree_tensors
from tests.shared_cases import SharedBatch

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def chain(n):
    return list(range(-1, n - 1))


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("S", [1, 2, 5, 33, 63, 64])
def test_draft_tree(S, index):
    gen = torch.Generator().manual_seed(S)
    trees = [chain(S), [-1] * S, [-1] + [0] * (S - 1), [-2] * S, [0] * S, list(range(S)), [-1] + [S] * (S - 1), [-1, 5][:S] + [1] * (S - 2),
             [-(2 ** 31)] + [2 ** 31 - 1] * (S - 1), [-1, -2][:S] + list(range(1, S - 1))]
    trees += [random_tree(gen, S, 1 + i) for i in range(40)]
    cached = torch.randint(0, 100000, (len(trees),), generator=gen, dtype=index)
    cached[3], cached[4] = -1, 2 ** 31 - 65
    cached[12], cached[13], cached[14] = 0, 2 ** 31 - 64, -5
    if index == torch.int64:
        cached[15] = 1 << 40
    got = ops.draft_tree(torch.tensor(trees, dtype=torch.int32).cuda(), cached.cuda())
    for name, g, w in zip(got._fields, got, tree_tensors(trees, S, cached.tolist())):
        assert torch.equal(g.cpu(), w), name


def test_draft_tree_of_many_and_of_none():
    gen = torch.Generator().manual_seed(3)
    trees = [random_tree(gen, 7, 3) for _ in range(3001)]
    parents = torch.tensor(trees, dtype=torch.int32)
    wide = torch.full((3001, 9), 77, dtype=torch.int32)
    wide[:, 1:8] = parents
    cached = torch.arange(3001, dtype=torch.int32)
    got = ops.draft_tree(wide.cuda()[:, 1:8], torch.stack([cached, cached], 1).cuda()[:, 1])
    for g, w in zip(got, tree_tensors(trees, 7, cached.tolist())):
        assert torch.equal(g.cpu(), w)
    assert ops.draft_tree(parents[:0].cuda(), cached[:0].cuda()).masks.shape == (0, 7)


SHAPES = {
    "one_token": ([], [(-1, 0, [-1])]),
    "one_behind_a_key": ([], [(-1, 1, [-1])]),
    "chain": ([], [(-1, 77, chain(5)), (-1, 64, chain(3)), (-1, 300, chain(5)), (-1, 0, chain(4))]),
    "trees": ([], [(-1, 130, [-1, 0, 0, 0, 1, 1, 3]), (-1, 63, [-1, 0, 1, 0, 3, 2, 2]), (-1, 1, [-1, -1, -1]), (-1, 200, [-1]), (-1, 60, [-1, 0, 0, 0, 0, 0, 0])]),
    "holes": ([], [(-1, 90, [-1, -2, 0, 1, 2, 3, 4]), (-1, 20, [-2, -1, 1, 0, 2]), (-1, 55, [-1, 0, -2, -2, -2])]),
    "pictures": ([203, 64, 130], [(0, 5, chain(4)), (1, 1, [-1, 0, 0]), (0, 0, [-1, 0, 0, 1]), (2, 70, chain(6)), (-1, 33, chain(2)), (2, 0, [-1]), (0, 64, [-1, 0, 0, 0])]),
}


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D,Hq,Hc", [(128, 4, 2), (64, 8, 1), (128, 8, 2), (64, 2, 2)])
@pytest.mark.parametrize("shape", list(SHAPES))
def test_attention(shape, D, Hq, Hc, dtype):
    prefixes, sequences = SHAPES[shape]
    case = DraftBatch(21, prefixes, sequences, Hq=Hq, Hc=Hc, D=D, P=64, dtype=dtype).on()
    case.check(case.call(ops))
    case.check(case.call(ops, share=False))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("S,reach", [(64, 1), (64, 4), (64, 64), (63, 9), (17, 3), (33, 2)])
def test_large_trees(S, reach, dtype):
    """Up to 64 tokens of a sequence: several tiles of rows, masks whose last bit is the sign."""
    gen = torch.Generator().manual_seed(S * 100 + reach)
    seqs = [(-1, n, random_tree(gen, m, reach)) for n, m in ((150, S), (1, S), (0, S), (64, S - 1), (97, 1), (700, S))]
    case = DraftBatch(22, [], seqs, Hq=4, Hc=1, D=64, P=32, dtype=dtype, S=S).on()
    case.check(case.call(ops))
    case = DraftBatch(23, [100], [(0, n, t) for _, n, t in seqs], Hq=2, Hc=2, D=128, P=64, dtype=dtype, S=S).on()
    case.check(case.call(ops))


@pytest.mark.parametrize("P", [1, 16, 48, 100, 128, 256])
def test_page_sizes(P):
    gen = torch.Generator().manual_seed(P)
    seqs = [(g, n, random_tree(gen, m, 3)) for g, n, m in ((0, 5, 9), (1, 40, 3), (-1, 130, 20), (0, 99, 1), (-1, 47, 11), (1, 0, 20))]
    case = DraftBatch(24, [150, 97], seqs, Hq=4, Hc=2, D=128, P=P, dtype=BF16).on()
    case.check(case.call(ops))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_sink_gate_and_scale(dtype):
    gen = torch.Generator().manual_seed(5)
    case = DraftBatch(25, [100], [(0, 20, random_tree(gen, 6, 2)), (0, 90, chain(3)), (-1, 33, random_tree(gen, 5, 5)), (-1, 0, [-2, -1])], Hq=8, Hc=2, D=64,
                      P=64, dtype=dtype).on()
    sinks = torch.randn(8, generator=case.gen)
    case.check(case.call(ops, sinks=sinks.cuda(), scale=0.21), sinks=sinks, scale=0.21)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_what_a_token_does_not_see_has_no_part_in_it(bad, dtype):
    """Keys and values of a draft that others do not see, infinite or NaN: only those that see it get to know."""
    tree = [-1, 0, 0, 2, 1, 2, 0, 3]
    case = DraftBatch(26, [], [(-1, 70, tree), (-1, 3, tree)], Hq=4, Hc=2, D=64, P=32, dtype=dtype).on()
    want = case.call(ops)
    for b in range(2):
        t = int(case.cached[b]) + 2  # of draft 2, which 2, 3, 5 and 7 see
        at = int(case.table[case.batch_idx[b], t // 32]) * 32 + t % 32
        case.pool_d[1][:, at, 5] = bad
        case.pool_d[0][1, at] = bad
    got = case.call(ops)
    aware = [2, 3, 5, 7]
    others = [0, 1, 4, 6]
    for w, g in zip(want, got):
        assert torch.equal(w[:, :, others], g[:, :, others])
    # head 0 and 1 have clean keys: the infinite value shows in its element alone
    out = got[0][:, :2, aware].float()
    assert (torch.isnan(out[..., 5]) if bad != bad else out[..., 5] == bad).all()
    rest = [i for i in range(64) if i != 5]
    assert torch.equal(got[0][:, :2, aware][..., rest], want[0][:, :2, aware][..., rest])
    if bad != bad:
        assert torch.isnan(got[1][:, 2:, aware]).all()


def test_masks_of_the_callers_own():
    """Any mask serves, not trees alone; bits behind a token's own count for nothing; a token need not see itself."""
    case = DraftBatch(27, [], [(-1, 40, chain(6)), (-1, 0, chain(6)), (-1, 0, chain(6))], Hq=4, Hc=2, D=64, P=32, dtype=BF16).on()
    case.masks[0] = torch.tensor([0, 1, 2, 0b0101, -1, 0b100000])
    case.masks[1] = torch.tensor([0, 0b10, 0b11, 0, 0b1110000, -(1 << 63)])
    case.masks_d = case.masks.cuda()
    got = case.call(ops)
    case.check(got)
    assert torch.isneginf(got[1][1, :, [0, 3, 5]]).all() and (got[0][1, :, [0, 3, 5]] == 0).all()
    assert torch.isfinite(got[1][1, :, [1, 2, 4]]).all()


def test_int64_positions_and_max_context():
    gen = torch.Generator().manual_seed(6)
    case = DraftBatch(28, [100], [(0, 30, random_tree(gen, 12, 3)), (0, 4, chain(7)), (-1, 100, random_tree(gen, 12, 12))], Hq=4, Hc=2, D=128, P=64,
                      dtype=BF16).on()
    want = case.call(ops)
    got = case.call(ops, tree=ops.DraftTree(case.masks_d, case.pos_d.long(), case.pos_d))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for room in (137, 104, 64, 1):
        case.check(case.call(ops, max_context=room), max_context=room)


def test_a_chain_is_what_the_shared_kernel_computes():
    """Without branches the tokens see what they see in `paged_decode_shared`: both are within what rounding allows of the same values (they
    round the scale at different places)."""
    case = DraftBatch(29, [150], [(0, 30, chain(7)), (0, 0, chain(3)), (-1, 99, chain(7)), (-1, 0, chain(1))], Hq=4, Hc=2, D=128, P=64, dtype=BF16).on()
    case.check(case.call(ops))
    case.check(SharedBatch.call(case, ops))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("scale", [-0.3, 0.0, -1e-3, 2.0])
def test_scales(scale, dtype):
    gen = torch.Generator().manual_seed(11)
    case = DraftBatch(37, [70], [(0, 20, random_tree(gen, 40, 3)), (0, 200, chain(3)), (-1, 33, random_tree(gen, 12, 5))], Hq=4, Hc=2, D=64, P=64,
                      dtype=dtype).on()
    case.check(case.call(ops, scale=scale), scale=scale)


def test_strides_plan_and_workspace_of_the_caller():
    """q a slice of a projection, out rows of a projection's input, table rows of a wider table, one plan for several layers."""
    gen = torch.Generator().manual_seed(7)
    case = DraftBatch(30, [90], [(0, 20, random_tree(gen, 5, 2)), (0, 90, chain(5)), (-1, 33, random_tree(gen, 4, 4))], Hq=8, Hc=2, D=64, P=32, dtype=BF16).on()
    want = case.call(ops)
    tree = ops.draft_tree(case.parents_d, case.cached_d)
    wide = torch.randn(3, 5, 12, 64, device="cuda").to(BF16)
    wide[:, :, 2:10] = case.q_d.transpose(1, 2)
    out = torch.full((3, 5, 9, 64), 7.0, device="cuda", dtype=BF16)
    case.table_d = torch.cat([case.table_d, torch.full_like(case.table_d, 10 ** 12)], 1)[:, :case.columns]
    shape = dict(q_heads=8, cached_heads=2, head_dim=64)
    workspace = torch.full((ops.shared_decode_workspace_bytes(3, 5, **shape),), 255, dtype=torch.uint8, device="cuda")
    plan = torch.full((ops.shared_decode_plan_bytes(3, 5, **shape),), 255, dtype=torch.uint8, device="cuda")
    made = ops.tree_decode_plan(case.batch_idx_d, tree, case.table_d, max_context=case.columns * 32, prefix_ids=case.ids_d, prefix_lens=case.lens_d,
                                plan=plan, **shape)
    assert made is plan
    for _ in range(3):
        lse = torch.empty(3, 8, 5, device="cuda")
        got = case.call(ops, tree=tree, q=wide[:, :, 2:10].transpose(1, 2), out=out[:, :, :8].transpose(1, 2), lse=lse, plan=plan, workspace=workspace)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and got[1] is lse
    assert (out[:, :, 8] == 7).all()


def test_slots_outside_the_table_and_foreign_plans():
    case = DraftBatch(31, [], [(-1, 50, chain(4)), (-1, 9, chain(4)), (-1, 70, chain(4))], Hq=4, Hc=2, D=64, P=32, dtype=BF16).on()
    want = case.call(ops)
    good = case.batch_idx_d.clone()
    case.batch_idx_d[1] = case.max_batch
    got = case.call(ops)
    assert (got[0][1] == 0).all() and torch.isneginf(got[1][1]).all()
    assert torch.equal(got[0][[0, 2]], want[0][[0, 2]])
    shape = dict(q_heads=4, cached_heads=2, head_dim=64)
    plan = ops.tree_decode_plan(good, ops.DraftTree(case.masks_d, case.pos_d, case.pos_d), case.table_d, max_context=case.columns * 32, **shape)
    case.batch_idx_d = good.flip(0).contiguous()
    got = case.call(ops, share=False, plan=plan)
    assert torch.isnan(got[0][[0, 2]]).all() and torch.isnan(got[1][[0, 2]]).all()
    assert torch.equal(got[0][1], want[0][1])


def test_long_context_and_many_sequences():
    gen = torch.Generator().manual_seed(8)
    case = DraftBatch(32, [], [(-1, 9000, random_tree(gen, 12, 3)), (-1, 300, chain(5))], Hq=4, Hc=1, D=128, P=128, dtype=BF16).on()
    case.check(case.call(ops))
    seqs = [(b % 5 - 1, b % 9, random_tree(gen, 1 + b % 6, 2)) for b in range(700)]
    case = DraftBatch(33, [64, 70, 128, 31], seqs, Hq=2, Hc=1, D=64, P=16, dtype=BF16).on()
    case.check(case.call(ops))


@pytest.mark.parametrize("dtype,D,Hq,Hc", [(BF16, 128, 8, 1), (F16, 64, 16, 2), (F32, 128, 4, 2), (BF16, 128, 4, 1)])
def test_trees_of_several_tiles_of_rows(dtype, D, Hq, Hc):
    """Sequences of one to eight tiles of 64 rows, alone and in groups of as many, on long and short contexts: tiles of one sequence are cut at
    the same keys."""
    gen = torch.Generator().manual_seed(9)
    seqs = []
    for b in range(23):
        n = (64, 1, 33, 17, 0, 48, 9, 64)[b % 8]
        seqs.append((b % 4 - 1, (1500, 3, 0, 700, 64, 129, 2311)[b % 7], random_tree(gen, n, 1 + b % 5)))
    case = DraftBatch(35, [64, 300, 1024], seqs, Hq=Hq, Hc=Hc, D=D, P=64, dtype=dtype, S=64).on()
    case.check(case.call(ops))
    case.check(case.call(ops, share=False))


@pytest.mark.parametrize("B", [1024, 1030])
def test_the_most_sequences_of_several_tiles(B):
    gen = torch.Generator().manual_seed(10)
    seqs = [(-1, b % 5, random_tree(gen, (9, 1, 12)[b % 3], 2)) for b in range(B)]
    case = DraftBatch(36, [], seqs, Hq=8, Hc=1, D=64, P=16, dtype=BF16).on()
    case.check(case.call(ops))


@pytest.mark.parametrize("dtype,Hq", [(BF16, 4), (F32, 2), (F16, 16)])
def test_drafts_in_front_of_the_end_of_a_prefix(dtype, Hq):
    """Sequences that were set back: their tokens are at positions of the prefix that others read as theirs."""
    gen = torch.Generator().manual_seed(13)
    trees = [random_tree(gen, n, r) for n, r in ((9, 3), (17, 4), (40, 5), (64, 2), (1, 1), (30, 9))]
    case = DraftBatch(39, [192, 130], [(0, 20, trees[0]), (0, 64, trees[1]), (0, 0, trees[2]), (0, 7, trees[3]), (1, 0, trees[4]), (1, 65, trees[5])],
                      Hq=Hq, Hc=2, D=64, P=32, dtype=dtype, S=64)
    case.cached[1], case.cached[2], case.cached[3], case.cached[5] = 100, 64, 130, 0
    case.masks, case.pos, case.rope = tree_tensors(case.trees, case.S, case.cached.tolist())
    case.on()
    case.check(case.call(ops))
    case.check(case.call(ops, share=False))


def test_the_most_sequences():
    """Of one cached head: the plan's arrays fill the shared memory of a workgroup."""
    gen = torch.Generator().manual_seed(12)
    seqs = [((b % 9) - 3, b % 5, random_tree(gen, (9, 1, 12)[b % 3], 2)) for b in range(1536)]
    case = DraftBatch(38, [64, 130, 70, 200, 64, 300], seqs, Hq=8, Hc=1, D=64, P=16, dtype=BF16).on()
    case.check(case.call(ops))


def test_refusals():
    case = DraftBatch(34, [], [(-1, 5, chain(3))], Hq=4, Hc=2, D=64, P=32, dtype=BF16).on()
    T = ops.DraftTree
    with pytest.raises(RuntimeError, match="masks must be int64"):
        case.call(ops, tree=T(case.masks_d.int(), case.pos_d, case.pos_d))
    with pytest.raises(RuntimeError, match="input_pos must be"):
        case.call(ops, tree=T(case.masks_d, case.pos_d[:, :2], case.pos_d))
    with pytest.raises(RuntimeError, match="the tree is of"):
        case.call(ops, q=case.q_d[:, :, :2])
    with pytest.raises(RuntimeError, match="given together"):
        case.call(ops, share=False, prefix_ids=case.ids_d)
    with pytest.raises(RuntimeError, match="prefix_lens must be"):
        case.call(ops, share=False, prefix_ids=case.ids_d, prefix_lens=case.lens_d[1:])
    with pytest.raises(RuntimeError, match="batch_idx must be"):
        ops.tree_decode_plan(case.batch_idx_d[:0], T(case.masks_d, case.pos_d, case.pos_d), case.table_d, q_heads=4, cached_heads=2, head_dim=64, max_context=64)
    with pytest.raises(RuntimeError, match="S of 1 to 64"):
        ops.draft_tree(torch.zeros(1, 65, dtype=torch.int32, device="cuda"), case.cached_d)
    with pytest.raises(RuntimeError, match="parents must be int32"):
        ops.draft_tree(case.parents_d.long(), case.cached_d)
    with pytest.raises(RuntimeError, match="cached must be"):
        ops.draft_tree(case.parents_d, case.cached_d[:0])
