"""Requests that fork from a cached picture, as an engine serves them: fork, prompts, decode steps, release."""

import pytest
import torch
from torch.nn.attention.flex_attention import AuxRequest, BlockMask

from falcon_perception_amd import attention as A
from falcon_perception_amd.paged_attention import PagedKVCache
from tests.shared_cases import SharedBatch

pytestmark = pytest.mark.gpu
DEV = "cuda"


class Server:
    """A cache, and every sequence's keys and values on the host."""

    def __init__(self, *, prefix_sharing=True, n_pages=120, P=32, slots=20, Hc=2, Hq=4, D=64, layers=3, dtype=torch.bfloat16, seed=0,
                 **kw):
        self.gen = torch.Generator().manual_seed(seed)
        self.cache = PagedKVCache(n_pages, P, slots, Hc, D, layers, dtype, device=DEV, prefix_sharing=prefix_sharing, **kw)
        self.cache.free_pages = (torch.randperm(n_pages - 1, generator=self.gen) + 1).tolist()
        self.Hc, self.Hq, self.D, self.P, self.layers, self.dtype = Hc, Hq, D, P, layers, dtype
        self.keys: dict[int, list] = {}  # slot -> per layer (k, v) [Hc, L, D]

    def rnd(self, *shape):
        return torch.randn(shape, generator=self.gen).to(self.dtype)

    def length(self, slot):
        return self.keys[slot][0][0].shape[1]

    def forget(self, slot):
        self.cache.erase(slot)
        del self.keys[slot]

    def picture(self, n):
        slot = self.cache.allocate()
        self.keys[slot] = [(self.rnd(self.Hc, 0, self.D), self.rnd(self.Hc, 0, self.D)) for _ in range(self.layers)]
        self.extend([slot], [n])
        return slot

    def fork(self, parent, n, count=1):
        slots = self.cache.fork(parent, n, count)
        for slot in slots:
            self.keys[slot] = [(k[:, :n], v[:, :n]) for k, v in self.keys[parent]]
        return slots

    def extend(self, slots, more, row_multiple=1):
        """A packed prefill step of `more` tokens for each slot; returns its tables."""
        old = [self.length(s) for s in slots]
        made = self.cache.step_tables(slots, old, [o + m for o, m in zip(old, more)], row_multiple=row_multiple).check()
        L = made.batch_idx.shape[0]
        starts = made.row_starts.tolist()
        for layer in range(self.layers):
            k, v = self.rnd(1, self.Hc, L, self.D), self.rnd(1, self.Hc, L, self.D)
            self.cache.insert_kv(layer, k.to(DEV), v.to(DEV), input_pos=made.input_pos[None], batch_idx=made.batch_idx[None])
            for s, m, at in zip(slots, more, starts):
                self.keys[s][layer] = tuple(torch.cat([old, new[0, :, at:at + m]], 1) for old, new in zip(self.keys[s][layer], (k, v)))
        return made

    def mask(self, slots, pos, room=None):
        B, room = len(slots), room or 16 * self.P
        whole = self.cache.create_causal_blockmask(B=1, L=room)
        n = (pos.view(B, 1, 1) // self.P + 1).int()
        logical = BlockMask.from_kv_blocks(n, whole.kv_indices[:, :, :1].expand(B, 1, 1, -1).contiguous(), None, None, BLOCK_SIZE=whole.BLOCK_SIZE,
                                           mask_mod=lambda b, h, q, kv: q + pos[b] >= kv, seq_lengths=(1, room))
        return self.cache.convert_logical_block_mask(logical, torch.tensor(slots, device=DEV))

    def decode(self, slots, sinks=None):
        """One token for each slot through every layer, checked."""
        lens = [self.length(s) for s in slots]
        for s, n in zip(slots, lens):
            self.cache.reserve(s, None, n + 1)
        pos = torch.tensor(lens, dtype=torch.int32, device=DEV)
        mask, idx = self.mask(slots, pos), torch.tensor(slots, device=DEV)
        for layer in range(self.layers):
            q, k, v = self.rnd(len(slots), self.Hq, 1, self.D), self.rnd(len(slots), self.Hc, 1, self.D), self.rnd(len(slots), self.Hc, 1, self.D)
            K, V = self.cache.insert_kv(layer, k.to(DEV), v.to(DEV), input_pos=pos.view(-1, 1), batch_idx=idx)
            out, aux = A.compiled_flex_attn_decode(q.to(DEV), K, V, block_mask=mask, return_aux=AuxRequest(lse=True),
                                                   sinks=None if sinks is None else sinks.to(DEV))
            for i, s in enumerate(slots):
                self.keys[s][layer] = (torch.cat([self.keys[s][layer][0], k[i]], 1), torch.cat([self.keys[s][layer][1], v[i]], 1))
            self.expected(q, [self.keys[s][layer] for s in slots], pos.cpu()).check((out, aux.lse), sinks=sinks)

    def expected(self, q, keys, pos):
        case = SharedBatch.__new__(SharedBatch)
        case.Hq, case.Hc, case.D, case.dtype, case.B, case.S = self.Hq, self.Hc, self.D, self.dtype, q.shape[0], 1
        case.q, case.keys, case.pos = q, keys, pos.view(-1, 1)
        return case

    def check_pool(self):
        """Every cached row of every sequence, through its row of the page table."""
        table, pool = self.cache.page_table.cpu(), self.cache.kv_cache.cpu()
        for slot, layers in self.keys.items():
            L = self.length(slot)
            at = torch.tensor([int(table[slot, t // self.P]) * self.P + t % self.P for t in range(L)], dtype=torch.int64)
            assert self.cache.page_table_cpu[slot] == [p for p in table[slot].tolist() if p >= 0]
            for layer, (k, v) in enumerate(layers):
                assert torch.equal(pool[layer, 0, 0][:, at], k) and torch.equal(pool[layer, 1, 0][:, at], v)
        if self.cache.physical_to_logical is not None:
            back = self.cache.physical_to_logical.cpu()
            for slot in self.keys:
                want = torch.full_like(back[slot], -1)
                for c, page in enumerate(self.cache.page_table_cpu[slot]):
                    want[page] = c
                assert torch.equal(back[slot], want)


@pytest.mark.parametrize("prefix_sharing", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_a_serving_run(prefix_sharing, dtype):
    s = Server(prefix_sharing=prefix_sharing, dtype=dtype)
    free = s.cache.num_free_pages
    cat, dog = s.picture(133), s.picture(96)  # one ends inside a page, one does not
    a = s.fork(cat, 133, 4)
    b = s.fork(dog, 96, 3)
    s.check_pool()
    s.extend(a + b, [3, 17, 1, 40, 5, 64, 9], row_multiple=128)
    s.check_pool()
    alone = s.picture(70)
    batch = [a[2], b[0], cat, alone, a[0], b[2], a[1], b[1], a[3], dog]
    for _ in range(3):
        s.decode(batch)
    s.check_pool()
    # the picture's own sequence ends first, a fork of a fork lives on
    s.forget(cat)
    late = s.fork(a[1], 140)
    s.forget(a[0])
    s.decode([a[1], *late, a[2], b[0], dog])
    s.check_pool()
    for slot in list(s.keys):
        s.forget(slot)
    assert s.cache.num_free_pages == free and sorted(s.cache.free_pages) == list(range(1, 120))
    assert not s.cache._page_slots and not s.cache._prefixes
    if prefix_sharing:
        assert not s.cache.prefix_ids.any()


def test_lines_of_forks():
    """What two slots are said to share, they share: forks at several lengths, of forks, of a sequence that has grown."""
    s = Server(n_pages=300, slots=40)
    root = s.picture(200)
    one = s.fork(root, 100, 2)
    two = s.fork(root, 170)
    s.extend(one + two, [80, 90, 5])
    three = s.fork(one[0], 150, 2)  # shares 100 with the root, 150 with one[0]
    four = s.fork(three[0], 64)
    s.extend(three + four + [root], [33, 1, 70, 55])
    five = s.fork(root, 255)
    ids, lens = s.cache.prefix_ids.tolist(), s.cache.prefix_lens.tolist()
    slots = list(s.keys)
    assert len({ids[x] for x in slots}) == 1 and ids[root] > 0
    for x in slots:
        for y in slots:
            n = min(lens[x], lens[y])
            assert all(torch.equal(s.keys[x][0][i][:, :n], s.keys[y][0][i][:, :n]) for i in range(2))
    for batch in (slots, one, three + four, [root, *five]):
        s.decode(batch)
    other = s.picture(200)
    s.fork(other, 100)
    assert s.cache.prefix_ids[other] != ids[root]


def test_step_tables_reserves_as_reserve_does():
    s, plain = Server(seed=5), Server(seed=5)
    slots = [s.cache.allocate() for _ in range(5)]
    assert slots == [plain.cache.allocate() for _ in range(5)]
    lens = [0, 0, 0, 0, 0]
    s.cache.reserve(slots[3], None, 70)  # more than its first step needs
    plain.cache.reserve(slots[3], None, 70)
    for more in ([40, 1, 0, 32, 100], [1, 1, 1, 1, 1], [64, 0, 31, 90, 0]):
        new = [a + b for a, b in zip(lens, more)]
        made = s.cache.step_tables(slots, lens, new, row_multiple=16).check()
        for slot, n in zip(slots, new):
            plain.cache.reserve(slot, None, n)
        for name in ("page_table_cpu", "capacity", "free_pages", "free_batch_idx"):
            assert getattr(s.cache, name) == getattr(plain.cache, name)
        assert torch.equal(s.cache.page_table, plain.cache.page_table)
        assert torch.equal(s.cache.physical_to_logical, plain.cache.physical_to_logical)
        rows = [(a, b) for a, b in zip(made.batch_idx.tolist(), made.input_pos.tolist()) if a]
        assert rows == [(slot, t) for slot, a, b in zip(slots, lens, new) for t in range(a, b)]
        lens = new


def test_a_table_without_its_inverse():
    s = Server(max_blocks_per_seq=9)
    cat = s.picture(133)
    forks = s.fork(cat, 133, 3)
    s.extend(forks, [3, 90, 1])
    s.decode([forks[1], cat, forks[0]])
    s.check_pool()


def test_refusals_change_nothing():
    s = Server(n_pages=20, slots=8, max_blocks_per_seq=10)
    cat = s.picture(133)
    before = ([list(x) for x in s.cache.page_table_cpu], list(s.cache.free_pages), list(s.cache.free_batch_idx), list(s.cache.capacity))
    for call, error in [(lambda: s.cache.fork(cat, 161), RuntimeError), (lambda: s.cache.fork(cat, 0), RuntimeError),
                        (lambda: s.cache.fork(0, 5), RuntimeError), (lambda: s.cache.fork(8, 5), RuntimeError),
                        (lambda: s.cache.fork(cat, 133, 7), RuntimeError), (lambda: s.cache.step_tables([cat], [133], [700]), RuntimeError),
                        (lambda: s.cache.step_tables([cat], [133], [321]), RuntimeError),
                        (lambda: s.cache.step_tables([cat, cat], [133, 133], [134, 134]), ValueError),
                        (lambda: s.cache.step_tables([cat], [133], [132]), ValueError), (lambda: s.cache.step_tables([0], [0], [1]), ValueError),
                        (lambda: s.cache.step_tables([cat], [200], [201]), RuntimeError),
                        (lambda: s.cache.step_tables([cat], [133], [140], row_multiple=0), ValueError),
                        (lambda: s.cache.step_tables([cat], [133, 1], [140]), ValueError)]:
        with pytest.raises(error):
            call()
        assert before == ([list(x) for x in s.cache.page_table_cpu], list(s.cache.free_pages), list(s.cache.free_batch_idx),
                          list(s.cache.capacity))
    assert s.cache.fork(cat, 133, 0) == []
    pages = s.cache.num_free_pages
    s.cache.free_pages, kept = s.cache.free_pages[:2], s.cache.free_pages[2:]
    with pytest.raises(RuntimeError, match="Cannot reserve 3 pages"):
        s.cache.fork(cat, 133, 3)
    s.cache.free_pages += kept
    assert s.cache.num_free_pages == pages
    s.check_pool()


def test_steps_that_one_launch_does_not_serve_change_nothing():
    s = Server(n_pages=20, slots=4200, max_blocks_per_seq=2)
    cat = s.picture(40)
    before = ([list(x) for x in s.cache.page_table_cpu], list(s.cache.free_pages), list(s.cache.free_batch_idx), list(s.cache.capacity))
    many = [i for i in range(1, 4199) if i != cat][:4097]
    for call, error, text in [(lambda: s.cache.step_tables(many, [0] * 4097, [0] * 4097), RuntimeError, "at most 4096"),
                              (lambda: s.cache.fork(cat, 32, 4097), RuntimeError, "at most 4096"),
                              (lambda: s.cache.step_tables(many[:3], [0] * 3, [1] * 3, row_multiple=1 << 30), ValueError, "31 bits"),
                              (lambda: s.cache.step_tables(many[:3], [0] * 3, [0] * 3, row_multiple=1 << 32), ValueError, "31 bits")]:
        with pytest.raises(error, match=text):
            call()
        assert before == ([list(x) for x in s.cache.page_table_cpu], list(s.cache.free_pages), list(s.cache.free_batch_idx),
                          list(s.cache.capacity))
    s.check_pool()


def test_pages_whose_rows_are_not_whole_chunks_are_not_forked():
    cache = PagedKVCache(16, 16, 5, 2, 4, 1, torch.bfloat16, device="cuda")
    slot = cache.allocate()
    cache.reserve(slot, None, 40)
    before = (list(cache.free_pages), list(cache.free_batch_idx))
    with pytest.raises(RuntimeError, match="cannot be copied"):
        cache.fork(slot, 20)
    assert before == (cache.free_pages, cache.free_batch_idx)


def test_decode_from_a_graph():
    """A decode step captured before any fork serves the forks that come later, also when they go."""
    s = Server(slots=12)
    B, slots = 5, []
    idx = torch.zeros(B, dtype=torch.int64, device=DEV)
    pos = torch.zeros(B, dtype=torch.int32, device=DEV)
    q, k, v = (torch.zeros(s.layers, B, h, 1, s.D, dtype=s.dtype, device=DEV) for h in (s.Hq, s.Hc, s.Hc))

    def step():
        got = []
        whole = s.cache.create_causal_blockmask(B=1, L=16 * s.P)
        logical = BlockMask.from_kv_blocks((pos.view(B, 1, 1) // s.P + 1).int(), whole.kv_indices[:, :, :1].expand(B, 1, 1, -1).contiguous(), None,
                                           None, BLOCK_SIZE=whole.BLOCK_SIZE, mask_mod=lambda b, h, x, kv: x + pos[b] >= kv,
                                           seq_lengths=(1, 16 * s.P))
        mask = s.cache.convert_logical_block_mask(logical, idx)
        for layer in range(s.layers):
            K, V = s.cache.insert_kv(layer, k[layer], v[layer], input_pos=pos.view(B, 1), batch_idx=idx)
            out, aux = A.compiled_flex_attn_decode(q[layer], K, V, block_mask=mask, return_aux=AuxRequest(lse=True))
            got.append((out, aux.lse))
        return got

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        made = step()
    s.cache.flush()
    cat, dog = s.picture(150), s.picture(64)
    a = s.fork(cat, 150, 3)
    for slots in ([cat, *a, dog], [dog, *a, cat], [a[0], dog, a[1], cat, a[2]]):
        lens = [s.length(x) for x in slots]
        for x, n in zip(slots, lens):
            s.cache.reserve(x, None, n + 1)
        idx.copy_(torch.tensor(slots))
        pos.copy_(torch.tensor(lens))
        for t in (q, k, v):
            t.copy_(s.rnd(*t.shape))
        graph.replay()
        torch.cuda.synchronize()
        for layer in range(s.layers):
            for i, x in enumerate(slots):
                s.keys[x][layer] = tuple(torch.cat([old, new[layer, i].cpu()], 1) for old, new in zip(s.keys[x][layer], (k, v)))
            s.expected(q[layer].cpu(), [s.keys[x][layer] for x in slots], pos.cpu()).check(made[layer])
        s.check_pool()
    s.forget(a[1])
    new = s.picture(90)  # takes the slot
    assert new == a[1]
    s.decode([new, cat, a[0], a[2]])


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.float16, 64), (torch.float32, 64)])
def test_prompts_attend_over_a_forked_prefix(dtype, D):
    """A packed prefill step of forks is bit for bit that of sequences which were given the same prefix each for itself."""
    n, prompts, layers, Hc, Hq = 133, [3, 17, 40], 2, 2, 4
    gen = torch.Generator().manual_seed(5)
    rnd = lambda *shape: torch.randn(shape, generator=gen).to(dtype).to(DEV)
    first = [(rnd(1, Hc, n, D), rnd(1, Hc, n, D)) for _ in range(layers)]
    new, q = None, None
    got = []
    for forked in (True, False):
        cache = PagedKVCache(60, 32, 9, Hc, D, layers, dtype, device=DEV, prefix_sharing=forked)
        heads = 1 if forked else 3
        slots = [cache.allocate() for _ in range(heads)]
        made = cache.step_tables(slots, [0] * heads, [n] * heads).check()
        for layer, (k, v) in enumerate(first):
            cache.insert_kv(layer, k.repeat(1, 1, heads, 1), v.repeat(1, 1, heads, 1), input_pos=made.input_pos[None], batch_idx=made.batch_idx[None])
        if forked:
            slots = cache.fork(slots[0], n, 3)
        made = cache.step_tables(slots, [n] * 3, [n + p for p in prompts], row_multiple=128).check()
        L = made.batch_idx.shape[0]
        if new is None:
            new, q = [(rnd(1, Hc, L, D), rnd(1, Hc, L, D)) for _ in range(layers)], rnd(1, Hq, L, D)
        mask = cache.create_prefill_blockmask(made.batch_idx[None], torch.ones(1, L, dtype=torch.int64, device=DEV), 998, 999, validate=True)
        for layer, (k, v) in enumerate(new):
            K, V = cache.insert_kv(layer, k, v, input_pos=made.input_pos[None], batch_idx=made.batch_idx[None])
            out, aux = A.compiled_flex_attn_prefill(q, K, V, block_mask=mask, return_aux=AuxRequest(lse=True))
            got.append((out, aux.lse, made.row_starts.tolist(), made.input_pos, made.batch_idx > 0))
    starts = got[0][2]
    assert starts == [0, 128, 256, 384]
    for a, b in zip(got[:layers], got[layers:]):
        assert a[2] == b[2] and torch.equal(a[3], b[3]) and torch.equal(a[4], b[4])
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    # the first row of a prompt sees the prefix and itself: in float64, within what probabilities of the type and sums may be off
    u = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -16}[dtype]
    for layer in range(layers):
        for at in starts[:3]:
            k, v = (torch.cat([first[layer][i], new[layer][i][:, :, at:at + 1]], 2)[0].double().repeat_interleave(Hq // Hc, 0) for i in range(2))
            scores = (k @ q[0, :, at, :, None].double())[..., 0] / D ** 0.5
            p = torch.softmax(scores, -1)
            want, mass = (p[..., None] * v).sum(1), (p[..., None] * v.abs()).sum(1)
            assert bool(((got[layer][0][0, :, at].double() - want).abs() <= 3 * u * mass).all())


def test_one_sequence_decodes_as_without_sharing():
    """A step of one sequence, alone and between steps of several, is that of a cache without prefix_sharing bit for bit."""
    outs = []
    for sharing in (True, False):
        s = Server(prefix_sharing=sharing, seed=9)
        seen = []
        cat = s.picture(133)
        forks = s.fork(cat, 133, 2)
        s.decode([forks[0]])
        s.decode([forks[0], cat, forks[1]])
        s.decode([cat])
        pos = torch.tensor([s.length(cat)], dtype=torch.int32, device=DEV)
        s.cache.reserve(cat, None, int(pos) + 1)
        mask, idx, gen = s.mask([cat], pos), torch.tensor([cat], device=DEV), torch.Generator().manual_seed(3)
        rnd = lambda heads: torch.randn(1, heads, 1, s.D, generator=gen).to(s.dtype).to(DEV)
        for layer in range(s.layers):
            K, V = s.cache.insert_kv(layer, rnd(s.Hc), rnd(s.Hc), input_pos=pos.view(-1, 1), batch_idx=idx)
            out, aux = A.compiled_flex_attn_decode(rnd(s.Hq), K, V, block_mask=mask, return_aux=AuxRequest(lse=True))
            seen += [out, aux.lse]
        outs.append(seen)
    assert all(torch.equal(x, y) for x, y in zip(*outs))
