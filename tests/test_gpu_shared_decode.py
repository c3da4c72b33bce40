"""Attention of a batch whose sequences share prefixes, against float64 (tolerances: SharedBatch.expect)."""

import pytest
import torch

from falcon_perception_amd import ops
from tests.shared_cases import SharedBatch

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def one_each(groups, behind, n=1):
    return [(g, k, n) for g, k in zip(groups, behind)]


SHAPES = {
    # a single sequence, with and without a prefix; one key
    "one_key": ([], [(-1, 1, 1)]),
    "one_alone": ([], [(-1, 77, 1)]),
    "one_with_prefix": ([130], [(0, 5, 1)]),
    # all of the batch on one prefix that ends inside a page and a tile
    "picture": ([203], one_each([0] * 7, [1, 2, 17, 64, 65, 130, 33])),
    # groups of many sizes, loners between them, in no order
    "mixed": ([65, 257, 128, 1], one_each([2, -1, 0, 1, 2, -1, 1, 3, 0, 3, 2, -1, 3], [3, 300, 9, 70, 1, 1, 128, 5, 64, 63, 40, 129, 1])),
    # more rows than a tile of queries
    "many": ([300], one_each([0] * 75, [1 + 7 * i % 50 for i in range(75)])),
    # keys of the prefix only: the token itself is its last key
    "nothing_behind": ([192], [(0, 1, 1), (0, 1, 1), (0, 1, 1)]),
    "long": ([2111], one_each([0, 0, 0, -1], [700, 3, 1, 1500])),
}


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D,Hq,Hc", [(128, 4, 2), (64, 8, 1), (128, 8, 2), (64, 2, 2)])
@pytest.mark.parametrize("shape", list(SHAPES))
def test_a_token_each(shape, D, Hq, Hc, dtype):
    prefixes, sequences = SHAPES[shape]
    case = SharedBatch(11, prefixes, sequences, Hq=Hq, Hc=Hc, D=D, P=64, dtype=dtype).on()
    case.check(case.call(ops))


@pytest.mark.parametrize("P", [1, 16, 48, 100, 128, 256])
def test_page_sizes(P):
    case = SharedBatch(12, [150, 97], one_each([0, 1, 0, -1, 1, 0], [5, 40, 130, 99, 1, 17]), Hq=4, Hc=2, D=128, P=P, dtype=BF16).on()
    case.check(case.call(ops))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("D,Hq,Hc", [(128, 4, 2), (64, 8, 1), (64, 1, 1)])
@pytest.mark.parametrize("tokens", [2, 5, 17, 70])
def test_several_tokens(tokens, D, Hq, Hc, dtype):
    """Prompts of different lengths behind their pictures, padded to the longest; one sequence has no token at all."""
    seqs = [(0, tokens, tokens), (0, tokens + 3, 1), (-1, tokens, max(1, tokens // 2)), (1, 2 * tokens, tokens), (1, 9, min(9, tokens)),
            (0, 4, 0)]
    case = SharedBatch(13, [190, 64], seqs, Hq=Hq, Hc=Hc, D=D, P=32, dtype=dtype, S=tokens).on()
    case.check(case.call(ops))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_sink_gate_and_scale(dtype):
    case = SharedBatch(14, [100], one_each([0, 0, -1], [20, 90, 33]), Hq=8, Hc=2, D=64, P=64, dtype=dtype).on()
    sinks = torch.randn(8, generator=case.gen)
    case.check(case.call(ops, sinks=sinks.cuda(), scale=0.21), sinks=sinks, scale=0.21)


def test_rows_that_see_less_than_the_prefix():
    """A sequence whose position lies inside the shared prefix sees its keys up to there, and int64 positions are the same."""
    case = SharedBatch(15, [300], one_each([0] * 5, [3, 50, 9, 1, 1]), Hq=4, Hc=2, D=128, P=64, dtype=BF16).on()
    case.pos[1, 0], case.pos[2, 0], case.pos[3, 0] = 0, 131, 298
    case.pos_d = case.pos.cuda()
    got = case.call(ops)
    case.check(got)
    again = case.call(ops, pos=case.pos_d.long())
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


def test_no_token_and_slots_outside_the_table():
    case = SharedBatch(16, [100], one_each([0] * 4, [3, 50, 9, 20]), Hq=4, Hc=2, D=128, P=64, dtype=BF16).on()
    case.pos[1, 0] = -1
    case.pos_d = case.pos.cuda()
    case.batch_idx_d[2] = case.max_batch
    case.batch_idx_d[3] = -5
    got = case.call(ops)
    case.pos[2, 0] = case.pos[3, 0] = -1
    case.check(got)


def test_max_context_bounds_the_keys():
    case = SharedBatch(17, [100], one_each([0] * 4, [3, 50, 9, 200]), Hq=4, Hc=2, D=128, P=64, dtype=BF16).on()
    got = case.call(ops, max_context=109)
    case.check(got, pos=case.pos.clamp(max=108))


def test_smallest_length_of_a_group_counts():
    """Members whose prefix lengths differ share the smallest of them; an id of 0 or below shares with nobody."""
    case = SharedBatch(18, [300], one_each([0] * 6, [30, 50, 9, 1, 77, 6]), Hq=4, Hc=2, D=128, P=64, dtype=BF16)
    case.lens[case.batch_idx[2]] = 133
    case.lens[case.batch_idx[4]] = -3
    case.ids[case.batch_idx[4]] = 0
    case.ids[case.batch_idx[5]] = -3
    case.on()
    case.check(case.call(ops))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_strides(dtype):
    """q as a slice of a projection, out as rows of a projection's input, table rows of a wider table."""
    case = SharedBatch(19, [90], one_each([0, 0, -1, 0], [20, 90, 33, 4]), Hq=8, Hc=2, D=64, P=32, dtype=dtype).on()
    want = case.call(ops)
    wide = torch.randn(4, 1, 12, 64, device="cuda").to(dtype)
    wide[:, :, 2:10] = case.q_d.transpose(1, 2)
    out = torch.full((4, 1, 9, 64), 7.0, device="cuda", dtype=dtype)
    case.table_d = torch.cat([case.table_d, torch.full_like(case.table_d, 10 ** 12)], 1)[:, :case.columns]
    got = case.call(ops, q=wide[:, :, 2:10].transpose(1, 2), out=out[:, :, :8].transpose(1, 2))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert (out[:, :, 8] == 7).all()


def test_unmapped_pages_are_the_reserved_page():
    """As in paged_decode: a block without a page reads page 0."""
    case = SharedBatch(20, [], [(-1, 200, 1), (-1, 90, 1)], Hq=4, Hc=2, D=128, P=64, dtype=BF16)
    case.pool[:, :, :64] = torch.randn(case.pool[:, :, :64].shape, generator=case.gen).to(BF16)
    case.table[case.batch_idx[0], 1] = -1
    for i in range(2):
        case.keys[0][i][:, 64:128] = case.pool[i][:, :64]
    case.on()
    case.check(case.call(ops))


def test_equal_to_paged_decode():
    """The same step through the operator that reads every copy; the two differ by the order of their sums."""
    case = SharedBatch(21, [400, 129], one_each([0, 1, 0, -1, 1], [20, 90, 33, 4, 300]), Hq=8, Hc=4, D=128, P=128, dtype=BF16).on()
    got = case.call(ops)
    plain = ops.paged_decode(case.q_d, case.pool_d[0].nan_to_num(), case.pool_d[1].nan_to_num(), case.table_d, case.batch_idx_d,
                             case.pos_d.view(-1), 128, case.columns * 128)
    case.check(got)
    case.check(plain)


def test_scores_of_any_size():
    """Scores spread over hundreds: the running maximum moves, and most probabilities vanish."""
    for dtype in (BF16, F16, F32):
        case = SharedBatch(22, [300], one_each([0, 0, -1], [20, 90, 333]), Hq=4, Hc=2, D=128, P=64, dtype=dtype, spread=5.0).on()
        case.check(case.call(ops))


def test_an_empty_batch():
    case = SharedBatch(23, [], [(-1, 3, 1)], Hq=4, Hc=2, D=128, P=64, dtype=BF16).on()
    out, lse = ops.paged_decode_shared(case.q_d[:0], case.pool_d[0], case.pool_d[1], case.table_d, case.batch_idx_d[:0],
                                       case.pos_d[:0], case.ids_d, case.lens_d, 64, 64)
    assert out.shape == (0, 4, 1, 128) and lse.shape == (0, 4, 1)


def test_refusals():
    case = SharedBatch(24, [64], [(0, 3, 1), (0, 5, 1)], Hq=4, Hc=2, D=128, P=64, dtype=BF16).on()
    call = lambda **kw: case.call(ops, **kw)
    with pytest.raises(RuntimeError, match="workspace must be"):
        call(workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))
    with pytest.raises(RuntimeError, match="plan of 16 bytes is too small"):
        call(plan=torch.empty(16, dtype=torch.uint8, device="cuda"))
    with pytest.raises(RuntimeError, match="GPU only"):
        call(q=case.q)
    with pytest.raises(RuntimeError, match="dtype mismatch"):
        call(q=case.q_d.half())
    with pytest.raises(RuntimeError, match="of 2 sequences of 1 tokens"):
        call(q=case.q_d.repeat(1, 1, 2, 1))
    with pytest.raises(RuntimeError, match="query heads per cache head"):
        call(q=case.q_d.repeat(1, 3, 1, 1))
    with pytest.raises(RuntimeError, match="int32 or int64"):
        call(pos=case.pos_d.float())
    with pytest.raises(RuntimeError, match="sinks must be"):
        call(sinks=torch.zeros(3, device="cuda"))
    with pytest.raises(RuntimeError, match="max_context"):
        call(max_context=0)
    with pytest.raises(RuntimeError, match="out must be like q"):
        call(out=torch.empty(2, 4, 1, 64, dtype=BF16, device="cuda"))
    with pytest.raises(RuntimeError, match="head_dim"):
        ops.shared_decode_plan(case.batch_idx_d, case.pos_d, case.ids_d, case.lens_d, q_heads=4, cached_heads=2, head_dim=96,
                               max_context=64)
    with pytest.raises(RuntimeError, match="prefix_lens must be"):
        ops.shared_decode_plan(case.batch_idx_d, case.pos_d, case.ids_d, case.lens_d[1:], q_heads=4, cached_heads=2, head_dim=64,
                               max_context=64)


def test_a_plan_serves_all_layers_and_another_steps_plan_gives_nan():
    case = SharedBatch(25, [100], one_each([0, 0, -1, 0], [20, 90, 33, 4]), Hq=4, Hc=2, D=128, P=64, dtype=BF16).on()
    shape = dict(q_heads=4, cached_heads=2, head_dim=128, max_context=case.columns * 64)
    plan = ops.shared_decode_plan(case.batch_idx_d, case.pos_d, case.ids_d, case.lens_d, **shape)
    want = case.call(ops)
    ws = torch.empty(ops.shared_decode_workspace_bytes(4, 1, q_heads=4, cached_heads=2, head_dim=128), dtype=torch.uint8, device="cuda")
    for _ in range(3):
        got = case.call(ops, plan=plan, workspace=ws)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # one sequence has moved on: its row is NaN, the others' are what they are
    later = case.pos_d.clone()
    later[1] += 1
    got = case.call(ops, plan=plan, pos=later)
    assert got[0][1].isnan().all() and got[1][1].isnan().all()
    keep = [0, 2, 3]
    assert torch.equal(got[0][keep], want[0][keep])
    # a plan of another limit, and memory that holds none
    for other in (ops.shared_decode_plan(case.batch_idx_d, case.pos_d, case.ids_d, case.lens_d, **{**shape, "max_context": 7}),
                  torch.zeros_like(plan)):
        got = case.call(ops, plan=other)
        assert got[0].isnan().all() and got[1].isnan().all()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_values_hidden_from_some_rows(value, dtype):
    """A V row (and a K row) that is not finite reaches the tokens that see its key and no other."""
    seqs = [(0, 20, 20), (0, 7, 3), (-1, 90, 15)]
    case = SharedBatch(26, [130], seqs, Hq=8, Hc=2, D=64, P=64, dtype=dtype, S=20).on()
    want = case.call(ops)
    case.check(want)
    # the key of token 11 of sequence 0 and of token 4 of sequence 2
    for b, t in ((0, 130 + 11), (2, 75 + 4)):
        page = int(case.table[case.batch_idx[b], t // 64])
        case.pool_d[1][1, page * 64 + t % 64, 5] = value
    got = case.call(ops)
    touched = torch.zeros_like(want[0], dtype=torch.bool)
    touched[0, 4:, 11:, 5] = True
    touched[2, 4:, 4:, 5] = True
    assert torch.equal(torch.where(touched, 0, got[0]), torch.where(touched, 0, want[0]))
    hit = got[0][touched]
    hit = hit[~(want[0][touched] == 0)]  # padding tokens of sequence 2
    assert (hit.isnan() if value != value else hit == value).all()
    assert torch.equal(got[1], want[1])


def test_graph_replays():
    """Plan and two layers captured once; the step's lengths, groups and rows change between the replays."""
    case = SharedBatch(27, [300, 200], one_each([0, 0, 1, -1, 1, 0], [20, 90, 33, 400, 5, 64]), Hq=4, Hc=2, D=128, P=64, dtype=BF16).on()
    shape = dict(q_heads=4, cached_heads=2, head_dim=128)
    ws = torch.empty(ops.shared_decode_workspace_bytes(6, 1, **shape), dtype=torch.uint8, device="cuda")
    plan = torch.empty(ops.shared_decode_plan_bytes(6, 1, **shape), dtype=torch.uint8, device="cuda")
    case.q2 = torch.randn(case.q.shape, generator=case.gen).to(BF16).cuda()

    def step():
        ops.shared_decode_plan(case.batch_idx_d, case.pos_d, case.ids_d, case.lens_d, max_context=case.columns * 64, plan=plan, **shape)
        return case.call(ops, plan=plan, workspace=ws), case.call(ops, q=case.q2, plan=plan, workspace=ws)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        made = step()
    pos, lens, ids = case.pos.clone(), case.lens.clone(), case.ids.clone()
    for turn in range(4):
        case.pos_d.copy_((pos - 3 * turn).clamp(min=-1))
        case.lens_d.copy_((lens - 40 * turn).clamp(min=0))
        case.ids_d.copy_(ids if turn % 2 == 0 else ids * 0)
        graph.replay()
        torch.cuda.synchronize()
        eager = step()
        for a, b in zip(made, eager):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        case.check(eager[0], pos=case.pos_d.cpu())


def test_another_stream_and_many_pages():
    """Page ids that do not fit LDS at once (pages of one token), on a stream of its own."""
    case = SharedBatch(28, [2500], one_each([0, 0, -1], [20, 1700, 3000]), Hq=2, Hc=1, D=64, P=1, dtype=F16).on()
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        got = case.call(ops)
    torch.cuda.synchronize()
    case.check(got)


@pytest.mark.parametrize("B", [257, 1000])
def test_many_sequences(B):
    groups = [b % 41 - 1 for b in range(B)]
    case = SharedBatch(29, [64 + 3 * g for g in range(40)], one_each(groups, [1 + b % 90 for b in range(B)]), Hq=2, Hc=1, D=64, P=32,
                       dtype=BF16).on()
    case.check(case.call(ops))


def test_long_prefixes_and_uneven_heads():
    """Three cached heads: the cut is for a number of workgroups that divides nothing evenly."""
    case = SharedBatch(30, [5000, 1333], one_each([0, 1, 0, 0, 1], [700, 3, 1, 50, 2222]), Hq=6, Hc=3, D=128, P=128, dtype=BF16).on()
    case.check(case.call(ops))


@pytest.mark.parametrize("D,Hq,Hc,dtype", [(128, 4, 2, BF16), (64, 16, 2, F16), (128, 8, 2, F32)])
def test_prefixes_of_several_tiles_beside_others(D, Hq, Hc, dtype):
    """Groups whose rows fill several tiles are cut by themselves, small ones and own keys together; some are too short for that."""
    groups = [0] * 90 + [1] * 70 + [2] * 3 + [3] * 40 + [-1] * 7
    order = torch.randperm(len(groups), generator=torch.Generator().manual_seed(3)).tolist()
    groups = [groups[i] for i in order]
    case = SharedBatch(31, [1500, 640, 2000, 70], one_each(groups, [1 + 13 * i % 60 for i in range(len(groups))]), Hq=Hq, Hc=Hc, D=D,
                       P=64, dtype=dtype).on()
    case.check(case.call(ops))


def test_tokens_in_any_places():
    """Tokens need not come first in their rows: -1 may stand anywhere."""
    case = SharedBatch(32, [190, 300], [(0, 70, 70), (0, 70, 70), (1, 80, 70), (-1, 90, 70), (1, 71, 70)], Hq=4, Hc=2, D=64, P=32,
                       dtype=BF16, S=70)
    case.pos[torch.rand(case.pos.shape, generator=case.gen) < 0.4] = -1
    case.pos[1] = -1
    case.pos[2, :66] = -1
    case.on()
    case.check(case.call(ops))
    case.check(case.call(ops, pos=case.pos_d.long()))


def test_far_pages():
    """Pages behind 2^32 bytes of a plane, and rows whose number passes 2^24."""
    P, D, n_pages = 128, 128, 150_000
    case = SharedBatch(33, [300], one_each([0, 0, -1], [20, 90, 400]), Hq=4, Hc=1, D=D, P=P, dtype=BF16)
    pool = torch.empty(2, 1, n_pages * P, D, dtype=BF16, device="cuda")
    shift = n_pages - case.n_pages
    pool[:, :, shift * P:] = case.pool.cuda()
    pool[:, :, :P] = float("nan")
    case.on()
    case.pool_d = pool
    case.table_d[case.table_d > 0] += shift
    case.check(case.call(ops))
    src, dst, rows = (torch.tensor([v], device="cuda") for v in (n_pages - 1, n_pages - 2, 100))
    ops.copy_pages(pool, src, dst, rows.int(), P)
    a, b = pool[:, :, (n_pages - 2) * P:(n_pages - 2) * P + 100], pool[:, :, (n_pages - 1) * P:(n_pages - 1) * P + 100]
    assert torch.equal(a.view(torch.int16), b.view(torch.int16))


@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_a_query_that_is_not_finite(value):
    """It spoils its own row only."""
    case = SharedBatch(34, [200], one_each([0] * 40, [1 + i for i in range(40)]), Hq=4, Hc=2, D=128, P=64, dtype=BF16).on()
    want = case.call(ops)
    case.q_d[7, 1] = value
    got = case.call(ops)
    keep = torch.ones(40, 4, dtype=torch.bool, device="cuda")
    keep[7, 1] = False
    assert torch.equal(got[0].squeeze(2)[keep], want[0].squeeze(2)[keep]) and torch.equal(got[1].squeeze(2)[keep], want[1].squeeze(2)[keep])
    assert got[0][7, 1].isnan().all()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_an_infinite_value_that_all_rows_see(dtype):
    """Infinity, whatever the weight of its key: the first is far below the largest."""
    case = SharedBatch(35, [150], one_each([0] * 20, [1 + i for i in range(20)]), Hq=4, Hc=1, D=64, P=32, dtype=dtype)
    k = case.keys[0][0]
    far = int((k[0, :128].double() @ case.q[0, 0, 0].double()).argmin())  # in a page that all of them map
    page = int(case.table[case.batch_idx[0], far // 32])
    case.pool[1][0, page * 32 + far % 32, 3] = float("inf")
    case.pool[1][0, page * 32 + far % 32, 4] = float("-inf")
    assert (case.table[case.batch_idx, far // 32] == page).all()
    case.q *= 3  # weights down to e^-20 and below
    case.on()
    want = torch.tensor([float("inf"), float("-inf")], dtype=dtype, device="cuda")
    out = case.call(ops)[0]
    assert (out[..., 3:5] == want).all()
    assert out[..., [0, 1, 2, 5]].isfinite().all()


def test_the_same_slot_twice():
    case = SharedBatch(36, [200], one_each([0, 0, -1], [30, 9, 50]), Hq=4, Hc=2, D=128, P=64, dtype=BF16).on()
    want = case.call(ops)
    order = [2, 0, 1, 0, 2]
    case.q_d, case.batch_idx_d = case.q_d[order], case.batch_idx_d[order]
    got = case.call(ops, pos=case.pos_d[order])
    assert torch.equal(got[1], want[1][order]) or torch.allclose(got[1], want[1][order], atol=2e-6)
    assert torch.equal(got[0][1], got[0][3]) and torch.equal(got[0][0], got[0][4])


def test_rows_that_are_not_aligned():
    case = SharedBatch(37, [90], one_each([0, 0], [20, 90]), Hq=4, Hc=2, D=64, P=32, dtype=BF16).on()
    want = case.call(ops)
    wide = torch.zeros(2, 4, 1, 67, dtype=BF16, device="cuda")
    wide[..., 3:] = case.q_d
    got = case.call(ops, q=wide[..., 3:])
    assert torch.equal(got[0], want[0])


@pytest.mark.parametrize("with_plan", [False, True])
def test_a_context_of_more_than_32_bits_is_refused(with_plan):
    case = SharedBatch(24, [64], [(0, 3, 1), (0, 5, 1)], Hq=4, Hc=2, D=128, P=64, dtype=BF16).on()
    kw = {}
    if with_plan:
        shape = dict(q_heads=4, cached_heads=2, head_dim=128)
        kw = dict(plan=torch.zeros(ops.shared_decode_plan_bytes(2, 1, **shape), dtype=torch.uint8, device="cuda"),
                  workspace=torch.zeros(ops.shared_decode_workspace_bytes(2, 1, **shape), dtype=torch.uint8, device="cuda"))
        with pytest.raises(RuntimeError, match="does not fit 32 bits"):
            ops.shared_decode_plan(case.batch_idx_d, case.pos_d, case.ids_d, case.lens_d, max_context=(1 << 32) + 200, plan=kw["plan"], **shape)
    with pytest.raises(RuntimeError, match="does not fit 32 bits"):
        case.call(ops, max_context=(1 << 32) + 200, **kw)
