"""Tables, rows and slot map of a step, and the copy of pages: whole numbers and bytes, equal to a plain loop's."""

import random

import pytest
import torch

from falcon_perception_amd import ops

pytestmark = pytest.mark.gpu


def plain(slots, old, new, parents, free, count, table, P, max_rows, multiple):
    """The step as a host loop that takes pages as `PagedKVCache.reserve` does."""
    table = table.clone()
    free = list(free[:count])
    rows, starts, copies = [], [0], []
    for s, o, n, p in zip(slots, old, new, parents):
        have = o // P if p > 0 else -(-o // P)
        need = max(0, -(-n // P) - have)
        taken = free[len(free) - need:]
        del free[len(free) - need:]
        if p > 0:
            table[s, :have] = table[p, :have]
        table[s, have:have + need] = torch.tensor(taken, dtype=torch.int64)
        copies.append((int(table[p, have]), taken[0], o % P) if p > 0 and o % P else (-1, -1, 0))
        rows += [(s, t, int(table[s, t // P]) * P + t % P) for t in range(o, n)]
        rows += [(0, 0, 0)] * (-(n - o) % multiple)
        starts.append(len(rows))
    rows += [(0, 0, 0)] * (max_rows - len(rows))
    return table, rows, starts, len(free), copies


def make(seed, B, *, old_hi, add_hi, P, forks=0, parents=1, max_batch=None, spare=5):
    """Requests, a table that maps what they have, and a free list."""
    r = random.Random(seed)
    max_batch = max_batch or B + parents + 3
    order = list(range(1, max_batch))
    r.shuffle(order)
    slots, parent_slots = order[:B], order[B:B + parents]
    lens = [r.randint(1, max(1, old_hi)) for _ in range(parents)]
    old, new, par = [], [], []
    for b in range(B):
        p = r.randrange(parents) if b < forks else -1
        o = lens[p] - (r.randint(0, lens[p] - 1) if r.random() < 0.3 else 0) if p >= 0 else r.randint(0, old_hi)
        old.append(o)
        new.append(o + r.randint(0, add_hi))
        par.append(parent_slots[p] if p >= 0 else r.choice([0, -4]))
    mix = list(range(B))
    r.shuffle(mix)
    old, new, par = ([x[i] for i in mix] for x in (old, new, par))
    columns = -(-(old_hi + add_hi) // P) + 1
    table = torch.full((max_batch, columns), -1, dtype=torch.int64)
    table[0] = 0
    pages = list(range(1, 20 + sum(-(-n // P) + 2 for n in new + lens)))
    r.shuffle(pages)
    for s, n in list(zip(parent_slots, lens)) + [(s, o) for s, o, p in zip(slots, old, par) if p <= 0]:
        for c in range(-(-n // P)):
            table[s, c] = pages.pop()
    return slots, old, new, par, pages, len(pages), table


def run(case, P, max_rows, multiple=1, lens=torch.int32, inverse=None, pad_free=3):
    slots, old, new, par, free, count, table = case
    dev = lambda x, t: torch.tensor(x, dtype=t, device="cuda")
    t = table.cuda()
    made = ops.step_tables(dev(slots, torch.int64), dev(old, lens), dev(new, lens), dev(free + [10 ** 9] * pad_free, torch.int64),
                           dev([count], torch.int32), t, P, max_rows, parents=dev(par, torch.int64), row_multiple=multiple,
                           inverse=inverse)
    return t, made


def check(case, P, max_rows, multiple=1, lens=torch.int32):
    slots, old, new, par, free, count, table = case
    t, made = run(case, P, max_rows, multiple, lens)
    made.check()
    want, rows, starts, left, copies = plain(slots, old, new, par, free, count, table, P, max_rows, multiple)
    assert torch.equal(t.cpu(), want)
    got = list(zip(made.batch_idx.tolist(), made.input_pos.tolist(), made.slot_map.tolist()))
    assert got == rows
    assert made.row_starts.tolist() == starts and made.free_left.tolist() == [left]
    assert list(zip(made.copy_src.tolist(), made.copy_dst.tolist(), made.copy_rows.tolist())) == copies


@pytest.mark.parametrize("B,old_hi,add_hi,P,forks,multiple", [
    (1, 0, 1, 128, 0, 1), (1, 300, 40, 64, 1, 1), (64, 4000, 1, 128, 0, 1), (65, 700, 90, 16, 30, 128), (7, 5, 3, 1, 4, 5),
    (300, 100, 400, 48, 120, 1), (257, 2000, 0, 100, 100, 16), (1000, 900, 60, 128, 333, 1),
])
@pytest.mark.parametrize("lens", [torch.int32, torch.int64])
def test_step(B, old_hi, add_hi, P, forks, multiple, lens):
    case = make(B + P, B, old_hi=old_hi, add_hi=add_hi, P=P, forks=forks, parents=5)
    rows = sum(-(-(n - o) // multiple) * multiple for o, n in zip(case[1], case[2]))
    check(case, P, rows + 37, multiple, lens)
    check(case, P, rows, multiple, lens)


def test_the_most_requests():
    check(make(3, 4096, old_hi=40, add_hi=5, P=16, forks=2000, parents=50, max_batch=9000), 16, 30000)


def test_the_most_requests_and_slots_and_many_rows():
    """A workgroup a CU, several turns of four rows a thread."""
    check(make(7, 4096, old_hi=60, add_hi=160, P=64, forks=900, parents=50, max_batch=1 << 17), 64, 400001)


def test_no_requests_and_no_rows():
    slots, old, new, par, free, count, table = make(4, 3, old_hi=40, add_hi=0, P=16)
    check((slots, old, old, par, free, count, table), 16, 0)
    check(([], [], [], [], free, count, table), 16, 5)


def test_only_the_new_blocks_are_written():
    """What a table holds behind the blocks of a request, and in the rows of others, stays."""
    case = make(5, 20, old_hi=400, add_hi=70, P=32, forks=8, parents=3)
    table = case[-1]
    table[table < 0] = 777
    check(case, 32, 3000)


def test_the_inverse_table():
    case = make(6, 20, old_hi=400, add_hi=70, P=32, forks=8, parents=3)
    slots, old, new, par, free, count, table = case
    pages = max(free) + 1
    inverse = torch.full((table.shape[0], pages), -1, dtype=torch.int64, device="cuda")
    t, made = run(case, 32, 3000, inverse=inverse)
    made.check()
    want = torch.full((table.shape[0], pages), -1, dtype=torch.int64)
    for s, o, n, p in zip(slots, old, new, par):
        for c in range(0 if p > 0 else -(-o // 32), -(-n // 32)):
            want[s, int(t[s, c])] = c
    assert torch.equal(inverse.cpu(), want)


@pytest.mark.parametrize("what,bit", [("pages", 1), ("columns", 2), ("rows", 4), ("slot", 8), ("zero", 8), ("twice", 8), ("shrinks", 8),
                                      ("negative", 8), ("parent", 8), ("nested", 8), ("count", 8), ("far", 8)])
def test_a_refused_step_changes_nothing(what, bit):
    slots, old, new, par, free, count, table = make(7, 9, old_hi=200, add_hi=70, P=16, forks=3, parents=2)
    max_rows, lens = 2000, torch.int64
    plain_one = next(b for b in range(9) if par[b] <= 0)
    fork = next(b for b in range(9) if par[b] > 0)
    if what == "pages":
        need = sum(-(-n // 16) - (o // 16 if p > 0 else -(-o // 16)) for o, n, p in zip(old, new, par))
        count = need - 1
    elif what == "columns":
        new[plain_one] = table.shape[1] * 16 + 1
    elif what == "rows":
        max_rows = sum(new) - sum(old) - 1
    elif what == "slot":
        slots[plain_one] = table.shape[0]
    elif what == "zero":
        slots[plain_one] = 0
    elif what == "twice":
        slots[8] = slots[0]
    elif what == "shrinks":
        old[plain_one] += 5
        new[plain_one] = old[plain_one] - 1
    elif what == "negative":
        old[plain_one] = -1
    elif what == "parent":
        par[fork] = table.shape[0]
    elif what == "nested":
        par[fork] = slots[plain_one]
    elif what == "count":
        count = len(free) + 4
    elif what == "far":
        new[plain_one] = 2 ** 31
    t, made = run((slots, old, new, par, free, count, table), 16, max_rows, lens=lens)
    assert int(made.status) & bit
    with pytest.raises(RuntimeError, match="step_tables: "):
        made.check()
    assert torch.equal(t.cpu(), table) and made.free_left.tolist() == [count]
    for rows in (made.batch_idx, made.input_pos, made.slot_map, made.row_starts, made.copy_rows):
        assert not rows.any()
    assert (made.copy_src == -1).all() and (made.copy_dst == -1).all()


def test_the_next_step_takes_free_left():
    slots, old, new, par, free, count, table = make(8, 30, old_hi=200, add_hi=40, P=16)
    dev = lambda x, t: torch.tensor(x, dtype=t, device="cuda")
    t, left, fr = table.cuda(), dev([count], torch.int32), dev(free, torch.int64)
    want, have = table, count
    for _ in range(3):
        made = ops.step_tables(dev(slots, torch.int64), dev(old, torch.int32), dev(new, torch.int32), fr, left, t, 16, 1200)
        want, _, _, have, _ = plain(slots, old, new, [0] * 30, free, have, want, 16, 1200, 1)
        left = made.check().free_left
        assert torch.equal(t.cpu(), want) and int(left) == have
        old, new = new, [n + 1 for n in new]


def test_step_tables_refusals():
    slots, old, new, par, free, count, table = make(9, 4, old_hi=200, add_hi=40, P=16)
    dev = lambda x, t: torch.tensor(x, dtype=t, device="cuda")
    args = [dev(slots, torch.int64), dev(old, torch.int32), dev(new, torch.int32), dev(free, torch.int64), dev([count], torch.int32),
            table.cuda()]
    def call(i=None, t=None, P=16, rows=10, **kw):
        return ops.step_tables(*(t if j == i else a for j, a in enumerate(args)), P, rows, **kw)
    for i, t, match in [(0, args[0].int(), "slots must be"), (1, args[1][:3], "old_lens must be"), (2, args[2].long(), "new_lens must be"),
                        (3, args[3].int(), "free_pages must be"), (4, args[4].long(), "free_count must be"),
                        (5, args[5].int(), "page_table must be"), (0, args[0].cpu(), "GPU only")]:
        with pytest.raises(RuntimeError, match=match):
            call(i, t)
    with pytest.raises(RuntimeError, match="row_multiple 0"):
        call(row_multiple=0)
    with pytest.raises(RuntimeError, match="page_size=0"):
        call(P=0)
    with pytest.raises(RuntimeError, match="inverse must be"):
        call(inverse=torch.zeros(3, 4, dtype=torch.int64, device="cuda"))


# --------------------------------------------------------------------------------------------------- copy of pages

def copied(pool, src, dst, rows, P):
    want = pool.clone()
    pages, valid = pool.shape[-2] // P, []
    for s, d, n in zip(src, dst, rows):
        valid.append(0 <= s < pages and 0 <= d < pages and n > 0)
    sources = {s for s, v in zip(src, valid) if v}
    taken = set()
    for s, d, n, v in zip(src, dst, rows, valid):
        if not v:
            continue
        if d not in sources and d not in taken:
            n = min(n, P)
            want[..., d * P:d * P + n, :] = pool[..., s * P:s * P + n, :]
        taken.add(d)
    return want


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("P,D,src,dst,rows", [
    (64, 128, [3], [5], [64]), (64, 64, [3, 3, 1], [5, 7, 2], [1, 63, 30]), (48, 64, [-1, 4, 4], [-1, 9, 2], [0, 48, 5]),
    (16, 128, [1, 2, 3, 4, 5], [6, 6, 1, 4, 7], [16, 9, 4, 3, 99]), (100, 64, [2, 11, 2, 0], [12, 3, -2, 8], [50, 20, 10, -1]),
    (1, 64, list(range(5)), [11, 10, 9, 8, 7], [1] * 5),
])
def test_copy_pages(P, D, src, dst, rows, dtype):
    gen = torch.Generator().manual_seed(5)
    pool = torch.randn(3, 2, 1, 2, 12 * P + 1, D, generator=gen).to(dtype)
    pool[..., ::7, 3] = float("nan")
    got = pool.cuda()
    dev = lambda x, t: torch.tensor(x, dtype=t, device="cuda")
    ops.copy_pages(got, dev(src, torch.int64), dev(dst, torch.int64), dev(rows, torch.int32), P)
    bits = torch.int32 if dtype == torch.float32 else torch.int16
    assert torch.equal(got.cpu().view(bits), copied(pool, src, dst, rows, P).view(bits))


def test_copy_many_pages():
    P, D, n = 16, 64, 700
    gen = torch.Generator().manual_seed(6)
    pool = torch.randn(2, 2 * n * P, D, generator=gen)
    order = torch.randperm(2 * n, generator=gen)
    src, dst = order[:n], order[n:]
    dst[650] = dst[3]
    rows = torch.randint(0, P + 1, (n,), generator=gen, dtype=torch.int32)
    got = pool.cuda()
    ops.copy_pages(got, src.cuda(), dst.cuda(), rows.cuda(), P)
    assert torch.equal(got.cpu(), copied(pool, src.tolist(), dst.tolist(), rows.tolist(), P))
    ops.copy_pages(got, src.cuda()[:0], dst.cuda()[:0], rows.cuda()[:0], P)


@pytest.mark.parametrize("change", [dict(rows=(1 << 32) + 10), dict(row_multiple=(1 << 32) + 1), dict(P=(1 << 32) + 16), dict(P=-(1 << 33))])
def test_numbers_of_more_than_32_bits_are_refused(change):
    slots, old, new, par, free, count, table = make(9, 4, old_hi=200, add_hi=40, P=16)
    dev = lambda x, t: torch.tensor(x, dtype=t, device="cuda")
    sizes = dict(P=16, rows=200, row_multiple=1) | change
    with pytest.raises(RuntimeError, match="does not fit 32 bits"):
        ops.step_tables(dev(slots, torch.int64), dev(old, torch.int32), dev(new, torch.int32), dev(free, torch.int64),
                        dev([count], torch.int32), table.cuda(), sizes["P"], sizes["rows"], row_multiple=sizes["row_multiple"])
    if "P" in change:
        one = torch.tensor([1], device="cuda")
        with pytest.raises(RuntimeError, match="does not fit 32 bits" if change["P"] > 0 else "page_size"):
            ops.copy_pages(torch.zeros(2, 64, 64, device="cuda"), one, one, one.int(), change["P"])


def test_copy_pages_refusals():
    pool = torch.zeros(2, 64, 64, device="cuda")
    one = torch.tensor([1], device="cuda")
    rows = one.int()
    for args, match in [((pool.transpose(0, 1), one, one, rows, 16), "contiguous"), ((pool, one.int(), one, rows, 16), "src must be"),
                        ((pool, one, one, one, 16), "rows must be"), ((pool, one, one.repeat(2), rows, 16), "dst must be"),
                        ((pool, one, one, rows, 0), "page_size"), ((pool.cpu(), one, one, rows, 16), "GPU only"),
                        ((pool.double(), one, one, rows, 16), "unsupported KV dtype")]:
        with pytest.raises(RuntimeError, match=match):
            ops.copy_pages(*args)


def test_steps_and_copies_from_a_graph():
    """Captured once, replayed over lengths that change: every replay is what the eager call makes of them."""
    P, slots = 16, [3, 1, 4, 7]
    dev = lambda x, t: torch.tensor(x, dtype=t, device="cuda")
    table = torch.full((9, 12), -1, dtype=torch.int64, device="cuda")
    table[0] = 0
    table[5, :4] = dev([40, 41, 42, 43], torch.int64)
    free, count = dev(list(range(1, 30)), torch.int64), dev([29], torch.int32)
    pool = torch.randn(2, 2, 50 * P, 64, device="cuda")
    old, new, parents = dev([0, 0, 37, 50], torch.int32), dev([0, 0, 0, 0], torch.int32), dev([0, 0, 5, 5], torch.int64)
    ids = dev(slots, torch.int64)

    def step(table, pool):
        made = ops.step_tables(ids, old, new, free, count, table, P, 200, parents=parents, row_multiple=8)
        ops.copy_pages(pool, made.copy_src, made.copy_dst, made.copy_rows, P)
        return made

    new.copy_(dev([5, 30, 40, 50], torch.int32))
    step(table.clone(), pool.clone())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        made = step(table, pool)
    for lens in ([5, 30, 40, 50], [1, 1, 37, 90], [100, 0, 80, 51], [300, 0, 80, 51], [0, 0, 37, 50]):
        new.copy_(dev(lens, torch.int32))
        before = table.clone(), pool.clone()
        graph.replay()
        torch.cuda.synchronize()
        want = step(*before)
        for a, b in zip(made, want):
            assert torch.equal(a, b)
        assert torch.equal(table, before[0]) and torch.equal(pool, before[1])
        assert bool(made.status) == (lens[0] == 300)


def test_under_inference_mode():
    case = make(11, 20, old_hi=400, add_hi=70, P=32, forks=8, parents=3)
    with torch.inference_mode():
        check(case, 32, 3000)
        t, made = run(case, 32, 3000)
        assert made.batch_idx.is_inference() and made.free_left.is_inference()
    t, made = run(case, 32, 3000)
    assert not made.batch_idx.is_inference()
    made.batch_idx[0] = 5  # an ordinary tensor
    assert made.batch_idx._version == 1 or made.batch_idx.requires_grad is False


@pytest.mark.parametrize("B,rows,native", [(1, 0, True), (3, 7, True), (20, 3001, True), (21, 3002, True), (5, 4, False), (33, 1001, False)])
def test_the_returned_tensors_are_apart(monkeypatch, B, rows, native):
    """Nine tensors in two allocations: writing to one changes none of the others, and each counts its own versions."""
    slots, old, new, par, free, count, table = make(12, B, old_hi=200, add_hi=1 if rows < 100 else 40, P=16)
    if rows < 100:
        new = list(old)
    if not native:
        monkeypatch.setattr(ops, "_current", lambda t: -1)
    dev = lambda x, t: torch.tensor(x, dtype=t, device="cuda")
    made = ops.step_tables(dev(slots, torch.int64), dev(old, torch.int32), dev(new, torch.int32), dev(free, torch.int64), dev([count], torch.int32),
                           table.cuda(), 16, rows).check()
    sizes = dict(batch_idx=rows, input_pos=rows, slot_map=rows, row_starts=B + 1, free_left=1, copy_src=B, copy_dst=B, copy_rows=B, status=1)
    for i, (name, t) in enumerate(made._asdict().items()):
        assert t.shape == (sizes[name],) and t._version == 0
        before = [x.clone() for x in made]
        t.fill_(i + 70)
        assert t._version == 1 and bool((t == i + 70).all())
        for j, (x, y) in enumerate(zip(made, before)):
            assert j == i or (torch.equal(x, y) and x._version == (j < i))
