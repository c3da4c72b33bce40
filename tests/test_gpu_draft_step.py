"""Steps of drafted tokens through the cache: append, attention, verification and the kept rows together."""

import threading

import pytest
import torch

from falcon_perception_amd import _native as N
from falcon_perception_amd import ops
from falcon_perception_amd.attention import compiled_flex_attn_decode
from falcon_perception_amd.paged_attention import PagedKVCache
from tests.draft_cases import random_tree

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
V = 97


class Model:
    """A small model whose layers are attention alone: everything a token adds follows from its id and its place in the text, so that the
    same text gives the same keys whether its tokens came as drafts or one by one."""

    def __init__(self, seed, layers, Hq, Hc, D, dtype):
        gen = torch.Generator().manual_seed(seed)
        rnd = lambda *s: torch.randn(s, generator=gen).cuda()
        self.layers, self.Hq, self.Hc, self.D, self.dtype = layers, Hq, Hc, D, dtype
        self.q, self.k, self.v = rnd(layers, V, Hq, D), rnd(layers, V, Hc, D), rnd(layers, V, Hc, D)
        self.turn = rnd(4096, D) * 0.3
        self.head = rnd(Hq * D, V) * (Hq * D) ** -0.5 * 4

    def rows(self, what, layer, tokens, places):
        """[B, H, S, D]"""
        x = what[layer][tokens] + self.turn[places.long()][:, :, None] * (what is not self.v)
        return x.transpose(1, 2).contiguous().to(self.dtype)

    def step(self, cache, mask, tokens):
        """Logits [B, S, V] of a step of drafts."""
        x = 0
        for layer in range(self.layers):
            k, v = (self.rows(w, layer, tokens, mask.rope_pos) for w in (self.k, self.v))
            pools = cache.insert_kv(layer, k, v, input_pos=mask.input_pos, batch_idx=mask.batch_idx)
            q = self.rows(self.q, layer, tokens, mask.rope_pos)
            out = compiled_flex_attn_decode(q, *pools, block_mask=mask)
            x = x + out.float()
        return x.transpose(1, 2).flatten(2) @ self.head

    def whole(self, text):
        """Logits behind every token of a text, without a cache, in 64 bits."""
        t = torch.tensor(text, device="cuda")
        n, G = len(text), self.Hq // self.Hc
        places = torch.arange(n, device="cuda")[None]
        x = 0
        for layer in range(self.layers):
            q, k, v = (self.rows(w, layer, t[None], places)[0].double() for w in (self.q, self.k, self.v))
            k, v = (y.repeat_interleave(G, 0) for y in (k, v))
            s = torch.bmm(q, k.mT.contiguous()) * self.D ** -0.5
            s = s.masked_fill(torch.ones(n, n, device="cuda").triu(1).bool(), -torch.inf)
            x = x + torch.bmm(torch.softmax(s, 2), v)
        return x.transpose(0, 1).flatten(1) @ self.head.double()


def start(cache, model, texts, gen):
    """Slots with the texts cached but for their last tokens."""
    slots = []
    for text in texts:
        slot = cache.allocate()
        cache.reserve(slot, None, len(text) + 80)
        slots.append(slot)
    batch_idx = torch.tensor(slots, device="cuda")
    for i in range(max(len(t) - 1 for t in texts)):
        have = torch.tensor([[i] if i < len(t) - 1 else [-1] for t in texts], dtype=torch.int32).cuda()
        tokens = torch.tensor([[t[min(i, len(t) - 1)]] for t in texts]).cuda()
        for layer in range(model.layers):
            k, v = (model.rows(w, layer, tokens, have.clamp(min=0)) for w in (model.k, model.v))
            cache.assign(layer, batch_idx, have, k, v)
            cache.flush()
    return batch_idx


@pytest.mark.parametrize("drafts", ["any", "likely"])
@pytest.mark.parametrize("sharing", [False, True])
@pytest.mark.parametrize("dtype,D,Hq,Hc,fuse", [(F32, 64, 4, 2, False), (BF16, 128, 2, 2, True), (F16, 64, 8, 1, True)])
def test_steps_of_drafts(dtype, D, Hq, Hc, fuse, sharing, drafts):
    """Greedy and drawn requests answer as if their text had been read whole: after every step the text's own logits, to what rounding the
    rows of three layers allows, say the same next token, and the cache holds the text's keys in its order."""
    gen = torch.Generator().manual_seed(31)
    model = Model(1, 3, Hq, Hc, D, dtype)
    cache = PagedKVCache(60, 16, 9, Hc, D, 3, dtype, prefix_sharing=sharing, fuse_decode_append=fuse)
    cache.free_pages = (torch.randperm(59, generator=gen) + 1).tolist()
    texts = [torch.randint(0, V, (n,), generator=gen).tolist() for n in (17, 1, 40, 2)]
    batch_idx = start(cache, model, texts, gen)
    heat = torch.tensor([0.0, 1.0, 0.0, 0.7], device="cuda")
    accepted_all = 0
    for turn in range(6):
        S = (7, 1, 12, 4, 9, 2)[turn]
        trees, tokens = torch.full((4, S), -2, dtype=torch.int32), torch.zeros(4, S, dtype=torch.int64)
        for b, text in enumerate(texts):
            n = S if b != 2 else max(1, S // 2)
            tree = random_tree(gen, n, 1 + b)
            trees[b, :n] = torch.tensor(tree, dtype=torch.int32)
            tokens[b, 0] = text[-1]
            for j in range(1, n):  # the model's own likely tokens, or any
                behind, at = [], j
                line = []
                while tree[at] >= 0:
                    at = tree[at]
                    line.append(int(tokens[b, at]))
                best = model.whole(text[:-1] + line[::-1])[-1]
                rank = j % 3 if drafts == "any" else tree[:j].count(tree[j]) % 3
                tokens[b, j] = int(best.topk(3).indices[rank]) if torch.rand((), generator=gen) < 0.8 else int(torch.randint(0, V, (), generator=gen))
        cached = torch.tensor([len(t) - 1 for t in texts], dtype=torch.int32).cuda()
        mask = cache.create_tree_mask(batch_idx, trees.cuda(), cached)
        logits = model.step(cache, mask, tokens.cuda())
        u = torch.rand(4, S, generator=gen)
        got = ops.verify_drafts(logits, tokens.cuda(), trees.cuda(), u.cuda(), temperatures=heat)
        cache.keep_drafts(mask, got.path)
        for b, text in enumerate(texts):
            n = int(got.accepted[b])
            accepted_all += n
            answer = got.tokens[b, :n + 1].tolist()
            texts[b] = text + answer
            want = model.whole(texts[b][:-1])[len(text) - 1:]
            # the logits at the tokens that stand are those of the text read whole: rows rounded to the type, as here, outputs too
            rows = torch.tensor(got.path[b, :n + 1].tolist(), device="cuda")
            u_half = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}[dtype]
            bound = (3 * 4 * u_half + 2.0 ** -15) * model.head.abs().sum(0).max().item()
            assert (logits[b, rows].double() - want).abs().max() <= bound
            if heat[b] == 0:
                top = want.topk(2).values
                sure = top[:, 0] - top[:, 1] > 2 * bound
                assert all(int(want[i].argmax()) == answer[i] for i in range(n + 1) if sure[i])
        for b, text in enumerate(texts):  # what the next step finds in front of it
            t = torch.tensor([text[:-1]], device="cuda")
            at = torch.arange(t.shape[1], device="cuda")
            where = cache.page_table[batch_idx[b], at // 16] * 16 + at % 16
            for layer in range(3):
                for i, w in enumerate((model.k, model.v)):
                    assert torch.equal(cache.kv_cache[layer, i, 0][:, where], model.rows(w, layer, t, at[None])[0])
    assert accepted_all >= (10 if drafts == "likely" else 1)


def captured_step(cache, model, mask, tokens, uniforms, heat):
    logits = model.step(cache, mask, tokens)
    got = ops.verify_drafts(logits, tokens, mask.parents, uniforms, temperatures=heat)
    cache.keep_drafts(mask, got.path)
    return logits, got


def test_a_captured_step():
    """The whole step in a graph, replayed between eager steps with other trees, lengths and random numbers in the same tensors."""
    gen = torch.Generator().manual_seed(32)
    model = Model(2, 3, 4, 2, 64, BF16)
    make = lambda: PagedKVCache(80, 16, 9, 2, 64, 3, BF16)
    cache, twin = make(), make()
    texts = [torch.randint(0, V, (n,), generator=gen).tolist() for n in (30, 5, 18)]
    batch_idx, twin_idx = start(cache, model, texts, gen), start(twin, model, texts, gen)
    assert torch.equal(batch_idx, twin_idx)
    S = 6
    parents = torch.zeros(3, S, dtype=torch.int32, device="cuda")
    tokens = torch.zeros(3, S, dtype=torch.int64, device="cuda")
    cached = torch.zeros(3, dtype=torch.int32, device="cuda")
    uniforms, heat = torch.zeros(3, S, device="cuda"), torch.tensor([1.0, 0.0, 0.8], device="cuda")
    workspace = torch.empty(ops.verify_workspace_bytes(3, S, V), dtype=torch.uint8, device="cuda")

    def fill(seed):
        g = torch.Generator().manual_seed(seed)
        parents.copy_(torch.tensor([random_tree(g, S, 1 + b) for b in range(3)], dtype=torch.int32))
        tokens.copy_(torch.randint(0, V, (3, S), generator=g))
        cached.copy_(torch.tensor([20 + seed % 7, 4, 17 - seed % 5], dtype=torch.int32))
        uniforms.copy_(torch.rand(3, S, generator=g))

    def run(c):
        mask = c.create_tree_mask(batch_idx, parents, cached)
        logits = model.step(c, mask, tokens)
        got = ops.verify_drafts(logits, tokens, parents, uniforms, temperatures=heat, workspace=workspace)
        c.keep_drafts(mask, got.path)
        return logits, got

    fill(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(cache)
    torch.cuda.current_stream().wait_stream(side)
    run(twin)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits, got = run(cache)
    for seed in range(1, 9):
        fill(seed)
        graph.replay()
        torch.cuda.synchronize()
        want_logits, want = run(twin)
        assert torch.equal(logits, want_logits)
        for x, y in zip(got, want):
            assert torch.equal(x, y)
        assert torch.equal(cache.kv_cache, twin.kv_cache)
        if seed % 3 == 0:  # an eager step in between, on the graph's own cache
            fill(100 + seed)
            for x, y in zip(run(cache)[1], run(twin)[1]):
                assert torch.equal(x, y)


def test_two_graphs_and_other_streams():
    """verify_drafts: two graphs with a workspace each, replayed on two streams at once, and an eager call on a third."""
    gen = torch.Generator().manual_seed(33)
    B, S, Vb = 16, 4, 5003
    sets = []
    for i in range(3):
        logits = (3 * torch.randn(B, S, Vb, generator=gen)).cuda()
        parents = torch.tensor([random_tree(gen, S, 2) for _ in range(B)], dtype=torch.int32).cuda()
        tokens = logits.argmax(2).roll(1, 1).contiguous()
        u = torch.rand(B, S, generator=gen).cuda()
        ws = torch.empty(ops.verify_workspace_bytes(B, S, Vb), dtype=torch.uint8, device="cuda")
        sets.append((logits, tokens, parents, u, ws))
    call = lambda s: ops.verify_drafts(*s[:4], workspace=s[4])
    want = [[t.clone() for t in call(s)] for s in sets]
    torch.cuda.synchronize()
    graphs, results = [], []
    for s in sets[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            results.append(call(s))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(3)]
    for turn in range(20):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        with torch.cuda.stream(streams[2]):
            third = call(sets[2])
        torch.cuda.synchronize()
        for got, w in zip([*results, third], want):
            for x, y in zip(got, w):
                assert torch.equal(x, y)


def test_threads():
    """The calls from two threads at once, a stream and buffers each."""
    gen = torch.Generator().manual_seed(34)
    B, S, Vb = 8, 5, 3001
    logits = (3 * torch.randn(B, S, Vb, generator=gen)).cuda()
    parents = torch.tensor([random_tree(gen, S, 3) for _ in range(B)], dtype=torch.int32).cuda()
    cached = torch.arange(B, dtype=torch.int32).cuda()
    tokens = torch.randint(0, Vb, (B, S), generator=gen).cuda()
    u = torch.rand(B, S, generator=gen).cuda()
    want, tree = ops.verify_drafts(logits, tokens, parents, u), ops.draft_tree(parents, cached)
    torch.cuda.synchronize()
    wrong = []

    def work():
        st = torch.cuda.Stream()
        ws = torch.empty(ops.verify_workspace_bytes(B, S, Vb), dtype=torch.uint8, device="cuda")
        with torch.cuda.stream(st):
            for _ in range(200):
                got, t = ops.verify_drafts(logits, tokens, parents, u, workspace=ws), ops.draft_tree(parents, cached)
                st.synchronize()
                if not all(torch.equal(x, y) for x, y in zip([*got, *t], [*want, *tree])):
                    wrong.append(1)

    threads = [threading.Thread(target=work) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_masks_and_steps_that_do_not_fit():
    model = Model(3, 1, 4, 2, 64, BF16)
    cache = PagedKVCache(20, 16, 4, 2, 64, 1, BF16)
    parents = torch.tensor([[-1, 0]], dtype=torch.int32).cuda()
    slot = cache.allocate()
    cache.reserve(slot, None, 40)
    batch_idx = torch.tensor([slot], device="cuda")
    mask = cache.create_tree_mask(batch_idx, parents, torch.tensor([3], dtype=torch.int32).cuda())
    q = torch.zeros(1, 4, 2, 64, dtype=BF16, device="cuda")
    with pytest.raises(RuntimeError, match="before PagedKVCache.insert_kv"):
        compiled_flex_attn_decode(q, *cache._pools[0], block_mask=mask)
    k = torch.zeros(1, 2, 1, 64, dtype=BF16, device="cuda")
    pools = cache.insert_kv(0, k, k, input_pos=torch.tensor([[3]], device="cuda"), batch_idx=batch_idx)
    with pytest.raises(RuntimeError, match="must follow the insert_kv"):
        compiled_flex_attn_decode(q, *pools, block_mask=mask)
    with pytest.raises(RuntimeError, match="score_mod"):
        compiled_flex_attn_decode(q, *pools, score_mod=lambda *a: a[0], block_mask=mask)
    with pytest.raises(RuntimeError, match="batch_idx must be"):
        cache.create_tree_mask(batch_idx, parents[:0], torch.tensor([3], dtype=torch.int32).cuda())


class Other(torch.Tensor):
    pass


def spread(t):
    """The same values with a gap behind every element of the last axis."""
    return torch.stack([t, t], -1).flatten(-2)[..., ::2]


def host_args():
    gen = torch.Generator().manual_seed(35)
    B, S, Hq, Hc, D, P, Vb = 3, 4, 4, 2, 64, 16, 500
    dev = lambda t: t.cuda()
    a = dict(parents=dev(torch.tensor([random_tree(gen, S, 2) for _ in range(B)], dtype=torch.int32)), cached=dev(torch.tensor([5, 0, 30], dtype=torch.int32)),
             bidx=dev(torch.tensor([2, 3, 1])), table=dev(torch.randperm(12, generator=gen).view(4, 3)), q=dev(torch.randn(B, Hq, S, D, generator=gen)),
             pool=dev(torch.randn(2, Hc, 12 * P, D, generator=gen)), sinks=dev(torch.randn(Hq, generator=gen)), ids=dev(torch.zeros(4, dtype=torch.int32)),
             logits=dev(torch.randn(B, S, Vb, generator=gen)), tokens=dev(torch.randint(0, Vb, (B, S), generator=gen)), u=dev(torch.rand(B, S, generator=gen)),
             heat=dev(torch.rand(B, generator=gen)), probs=dev(torch.softmax(torch.randn(B, S, Vb, generator=gen), 2).to(BF16)),
             path=dev(torch.tensor([[0, 2, 3, -1], [0, 3, -1, -1], [0, 1, 3, -1]], dtype=torch.int32)), P=P, room=48, scale=0.125)
    shape = dict(q_heads=Hq, cached_heads=Hc, head_dim=D)
    a["plan"] = torch.empty(ops.shared_decode_plan_bytes(B, S, **shape), dtype=torch.uint8, device="cuda")
    a["ws"] = torch.empty(ops.shared_decode_workspace_bytes(B, S, **shape), dtype=torch.uint8, device="cuda")
    a["vws"] = torch.empty(ops.verify_workspace_bytes(B, S, Vb), dtype=torch.uint8, device="cuda")
    tree = ops.draft_tree(a["parents"], a["cached"])
    a.update(masks=tree.masks, pos=tree.input_pos, pk=a["pool"][0], pv=a["pool"][1], lens=a["ids"].clone())
    return a


def host_calls(a):
    h, end = N.host(), (torch.cuda.current_device(), N.raw_stream(torch.cuda.current_device()))
    return dict(
        draft_tree=lambda: h.draft_tree(a["parents"], a["cached"], *end),
        tree_plan=lambda: h.tree_plan(a["bidx"], a["masks"], a["pos"], a["table"], 4, 2, 64, a["room"], a["ids"], a["lens"], a["plan"], *end),
        tree=lambda: h.tree(a["q"], a["pk"], a["pv"], a["table"], a["bidx"], a["masks"], a["pos"], a["P"], a["room"], a["scale"], a["sinks"], a["plan"],
                            a["ws"], *end),
        verify=lambda: h.verify(a["logits"], a["tokens"], a["parents"], a["u"], a["heat"], a["probs"], a["vws"], *end),
        keep=lambda: h.keep(a["pool"], a["table"], a["bidx"], a["cached"], a["path"], a["P"], *end))


LEFT = [("draft_tree", "parents", spread), ("draft_tree", "parents", lambda t: t.long()), ("draft_tree", "parents", lambda t: t[0]),
        ("draft_tree", "cached", lambda t: t.float()), ("draft_tree", "cached", lambda t: t[:1]), ("draft_tree", "cached", lambda t: t.cpu()),
        ("tree_plan", "masks", lambda t: t.int()), ("tree_plan", "pos", lambda t: t[:1]), ("tree_plan", "bidx", lambda t: t.int()),
        ("tree_plan", "table", spread), ("tree_plan", "ids", lambda t: None), ("tree_plan", "lens", lambda t: t[:2]), ("tree_plan", "plan", lambda t: t.float()),
        ("tree_plan", "room", lambda t: 1 << 40), ("tree", "q", spread), ("tree", "q", lambda t: t.half()), ("tree", "q", lambda t: t[0]),
        ("tree", "q", lambda t: t.as_subclass(Other)), ("tree", "q", lambda t: torch.zeros(t.numel() + 1, device="cuda")[1:].view(t.shape)),
        ("tree", "pv", lambda t: t[:, 1:]), ("tree", "table", lambda t: t.int()), ("tree", "bidx", lambda t: t[:1]), ("tree", "masks", spread),
        ("tree", "pos", lambda t: t.float()), ("tree", "sinks", lambda t: t[:1]), ("tree", "ws", lambda t: t.float()), ("tree", "P", lambda t: 1 << 33),
        ("verify", "logits", spread), ("verify", "logits", lambda t: t.double()), ("verify", "logits", lambda t: t[0]), ("verify", "tokens", lambda t: t.int()),
        ("verify", "parents", spread), ("verify", "u", lambda t: t.double()), ("verify", "heat", lambda t: t[:1]), ("verify", "probs", lambda t: t[:, :, :9]),
        ("verify", "probs", spread), ("verify", "vws", lambda t: t.float()), ("keep", "pool", spread), ("keep", "pool", lambda t: t.double()),
        ("keep", "table", lambda t: t.int()), ("keep", "bidx", spread), ("keep", "cached", lambda t: t[:1]), ("keep", "path", lambda t: t.long()),
        ("keep", "path", spread), ("keep", "P", lambda t: 0)]


@pytest.mark.parametrize("i", range(len(LEFT)))
def test_what_the_calls_in_cpp_do_not_recognise_is_left_alone(i):
    call, name, other = LEFT[i]
    a = host_args()
    before = a["pool"].clone()
    a[name] = other(a[name])
    assert host_calls(a)[call]() is None
    if name != "pool":
        assert torch.equal(a["pool"], before)


def test_the_calls_in_cpp_return_what_ops_does(monkeypatch):
    a = host_args()
    calls = host_calls(a)
    got = [calls["draft_tree"](), calls["tree_plan"](), calls["tree"](), calls["verify"]()]
    assert got[1] is True and None not in got
    pool = a["pool"].clone()
    assert calls["keep"]() is True
    moved = a["pool"].clone()
    a["pool"].copy_(pool)

    class Nothing:  # ops.py by itself
        draft_tree = tree_plan = tree = verify = keep = staticmethod(lambda *a: None)

    monkeypatch.setattr(N, "host", lambda: Nothing)
    tree = ops.draft_tree(a["parents"], a["cached"])
    plan = ops.tree_decode_plan(a["bidx"], tree, a["table"], q_heads=4, cached_heads=2, head_dim=64, max_context=48, prefix_ids=a["ids"],
                                prefix_lens=a["lens"], plan=a["plan"])
    want = [tree, plan, ops.paged_decode_tree(a["q"], a["pk"], a["pv"], a["table"], a["bidx"], tree, 16, 48, scale=0.125, sinks=a["sinks"], plan=plan,
                                              workspace=a["ws"]),
            ops.verify_drafts(a["logits"], a["tokens"], a["parents"], a["u"], temperatures=a["heat"], draft_probs=a["probs"], workspace=a["vws"])]
    for g, w in zip(got, want):
        if g is not True:
            for x, y in zip(g, w):
                assert x.dtype == y.dtype and x.shape == y.shape and x.stride() == y.stride() and torch.equal(x, y)
    ops.keep_rows(a["pool"], a["table"], a["bidx"], a["cached"], a["path"], 16)
    assert torch.equal(a["pool"], moved) and not torch.equal(moved, pool)
    for name in ("draft_tree", "tree_plan", "tree", "verify", "keep"):
        monkeypatch.undo()
        with pytest.raises(TypeError, match="arguments expected"):
            getattr(N.host(), name)(1, 2)


def test_what_the_library_refuses_is_raised():
    a = host_args()
    a["vws"] = a["vws"][:64]
    with pytest.raises(RuntimeError, match="is needed"):
        host_calls(a)["verify"]()
    a["plan"] = a["plan"][:64]
    with pytest.raises(RuntimeError, match="the plan needs"):
        host_calls(a)["tree_plan"]()
    with pytest.raises(RuntimeError, match="too small"):
        host_calls(a)["tree"]()


def test_results_do_not_overlap():
    a = host_args()
    for made in (ops.draft_tree(a["parents"], a["cached"]), ops.verify_drafts(a["logits"], a["tokens"], a["parents"], a["u"], workspace=a["vws"])):
        copies = [t.clone() for t in made]
        for i, t in enumerate(made):
            version = [x._version for x in made]
            t.fill_(7)
            assert [x._version - v for x, v in zip(made, version)] == [int(k == i) for k in range(len(made))]
            for k, (x, c) in enumerate(zip(made, copies)):
                if k > i:
                    assert torch.equal(x, c)
