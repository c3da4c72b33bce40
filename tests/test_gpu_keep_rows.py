"""Cached rows of the drafts that stand, moved together: bit for bit against plain indexing."""

import pytest
import torch

from falcon_perception_amd import ops

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def expected(pool, table, batch_idx, cached, path, P):
    before, after = pool.clone(), pool.clone()
    n_slots = pool.shape[-2]
    named = set()

    def row(slot, t):
        blk = t // P
        page = int(table[slot, blk]) if blk < table.shape[1] else -1
        return page * P + t % P if 0 <= page < n_slots // P else -1

    for slot, base, line in zip(batch_idx.tolist(), cached.tolist(), path.tolist()):
        if not 0 <= slot < table.shape[0] or not 0 <= base < 2 ** 31 or slot in named:
            named.add(slot)
            continue
        named.add(slot)
        last = -1
        for i, p in enumerate(line):
            if not last < p < len(line):
                break
            last = p
            src, dst = row(slot, base + p), row(slot, base + i)
            if p > i and src >= 0 and dst >= 0:
                after[..., dst, :] = before[..., src, :]
    return after


def random_path(gen, S, n):
    rows = torch.randperm(S, generator=gen)[:n].sort().values.int()
    if n:
        rows[0] = 0 if n > 1 else rows[0]
    path = torch.full((S,), -1, dtype=torch.int32)
    path[:n] = rows.sort().values
    return path


class Cache:
    def __init__(self, seed, B, S, *, planes=(3, 2, 1, 2), D=64, P=16, dtype=BF16, longest=100, columns=None):
        gen = torch.Generator().manual_seed(seed)
        blocks = -(-(longest + S) // P)
        n_pages = B * blocks + 3
        self.pool = torch.randn(*planes, n_pages * P, D, generator=gen).to(dtype)
        self.table = torch.full((B + 3, columns or blocks + 1), -1, dtype=torch.int64)
        self.batch_idx = (torch.randperm(B + 2, generator=gen) + 1)[:B]
        pages = torch.randperm(n_pages - 1, generator=gen) + 1
        self.cached = torch.randint(0, longest + 1, (B,), generator=gen, dtype=torch.int32)
        for i, slot in enumerate(self.batch_idx.tolist()):
            self.table[slot, :blocks] = pages[i * blocks:(i + 1) * blocks][:self.table.shape[1]]
        self.path = torch.stack([random_path(gen, S, int(torch.randint(0, S + 1, (1,), generator=gen))) for _ in range(B)])
        self.P, self.gen = P, gen

    def run(self, **kw):
        a = dict(table=self.table, batch_idx=self.batch_idx, cached=self.cached, path=self.path)
        a.update(kw)
        pool = self.pool.cuda()
        ops.keep_rows(pool, a["table"].cuda(), a["batch_idx"].cuda(), a["cached"].cuda(), a["path"].cuda(), self.P)
        want = expected(self.pool, a["table"], a["batch_idx"], a["cached"], a["path"], self.P)
        assert torch.equal(pool.cpu(), want)
        return pool


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D", [8, 64, 72, 128])
@pytest.mark.parametrize("S", [1, 2, 7, 33, 64])
def test_paths(S, D, dtype):
    Cache(S + D, 9, S, D=D, dtype=dtype).run()


@pytest.mark.parametrize("P", [1, 3, 16, 100, 128])
def test_page_sizes(P):
    Cache(P, 7, 20, P=P).run()


@pytest.mark.parametrize("planes", [(1,), (5,), (28, 2, 1, 8), (301,)])
def test_planes(planes):
    Cache(4, 5, 12, planes=planes).run()


@pytest.mark.parametrize("D,dtype", [(64, BF16), (128, F32), (1024, F32), (2048, F16)])
def test_rows_that_are_written_over_and_read(D, dtype):
    """Every row moves down by one or two: each is the place of one and the source of another, in several turns of a plane."""
    case = Cache(5, 6, 64, D=D, dtype=dtype, longest=40)
    for b in range(6):
        step = 1 + b % 2
        line = torch.arange(64, dtype=torch.int32) + step
        line[0] = b // 3
        line[64 - step:] = -1
        case.path[b] = line
    case.run()


def test_paths_that_do_not_rise():
    case = Cache(6, 8, 6)
    case.path[:] = torch.tensor([[0, 2, 2, 5, -1, -1], [0, 3, 1, 4, -1, -1], [-1, 2, 3, 4, 5, -1], [2, 4, 6, 5, -1, -1], [1, 2, 3, 4, 5, 7],
                                 [0, 1, 2, 3, 4, 5], [0, 4, -1, 5, -1, -1], [5, 2 ** 31 - 1, -1, -1, -1, -1]], dtype=torch.int32)
    case.run()


def test_bad_entries():
    """Slots outside the table, named twice, lengths that are none, pages that are none or outside the pool, rows past the table."""
    case = Cache(7, 12, 8, longest=40, P=4)
    case.batch_idx[1] = -1
    case.batch_idx[2] = case.table.shape[0]
    case.batch_idx[5] = case.batch_idx[4]
    case.cached[6] = -3
    case.table[case.batch_idx[7], :] = -1
    case.table[case.batch_idx[8], 3:6] = 10 ** 12
    case.table[case.batch_idx[9], 2:9:2] = -1
    case.cached[10] = 2 ** 31 - 1
    case.cached[11] = case.table.shape[1] * 4 - 3
    case.run()
    case.run(cached=case.cached.long())
    far = case.cached.long()
    far[3], far[0] = 1 << 40, -(1 << 40)
    case.run(cached=far)


def test_tables_of_other_widths_and_strides():
    case = Cache(8, 5, 10, columns=3)
    case.run()
    wide = torch.full((case.table.shape[0], 9), 10 ** 12, dtype=torch.int64)
    wide[:, 2:5] = case.table
    pool = case.pool.cuda()
    long = case.path.repeat_interleave(2, 1).cuda()[:, ::2]
    ops.keep_rows(pool, wide.cuda()[:, 2:5], case.batch_idx.cuda(), case.cached.cuda(), long, case.P)
    assert torch.equal(pool.cpu(), expected(case.pool, case.table, case.batch_idx, case.cached, case.path, case.P))


def test_many_sequences():
    Cache(9, 1200, 4, planes=(2,), longest=10, P=8).run()


def test_offsets_past_32_bits():
    """The last pages of a plane of 9 GB, rows whose byte offsets need 64 bits; any bit pattern is kept."""
    n_slots, D, P = 1 << 25, 128, 128
    pool = torch.empty(1, n_slots, D, dtype=BF16, device="cuda")
    pages = n_slots // P
    table = torch.tensor([[0, 0], [pages - 1, pages - 2]], device="cuda")
    rows = torch.randint(-2 ** 15, 2 ** 15, (2 * P, D), dtype=torch.int16)
    pool[0, -2 * P:] = rows.view(BF16).cuda()
    path = torch.tensor([[0, 3, 7, -1, -1, -1, -1, -1]], dtype=torch.int32).cuda()  # (entries are rows of the step: below its 8)
    ops.keep_rows(pool, table, torch.tensor([1], device="cuda"), torch.tensor([P - 2], device="cuda"), path, P)
    want = rows.clone()
    line = lambda t: (P if t < P else 0) + t % P  # the last page comes first in the text
    for i, p in ((1, 3), (2, 7)):
        want[line(P - 2 + i)] = rows[line(P - 2 + p)]
    assert torch.equal(pool[0, -2 * P:].view(torch.int16).cpu(), want)


def test_nothing_moves():
    case = Cache(10, 4, 8)
    case.path[:] = torch.arange(8)
    assert torch.equal(case.run().cpu(), case.pool)
    ops.keep_rows(case.pool.cuda(), case.table.cuda(), case.batch_idx[:0].cuda(), case.cached[:0].cuda(), case.path[:0].cuda(), 16)
    ops.keep_rows(case.pool[:0].cuda(), case.table.cuda(), case.batch_idx.cuda(), case.cached.cuda(), case.path.cuda(), 16)


def test_refusals():
    case = Cache(11, 2, 4)
    pool, table, idx, cached, path = (t.cuda() for t in (case.pool, case.table, case.batch_idx, case.cached, case.path))
    for args, text in [((pool[..., ::2], table, idx, cached, path, 16), "contiguous"), ((pool, table.int(), idx, cached, path, 16), "page_table must be"),
                       ((pool, table, idx.int(), cached, path, 16), "batch_idx must be"), ((pool, table, idx, cached.float(), path, 16), "cached must be"),
                       ((pool, table, idx, cached, path.long(), 16), "path must be int32"), ((pool, table, idx, cached, path, 0), "page_size 0"),
                       ((pool, table, idx, cached[:1], path, 16), "cached must be"), ((pool.double(), table, idx, cached, path, 16), "unsupported")]:
        with pytest.raises(RuntimeError, match=text):
            ops.keep_rows(*args)
