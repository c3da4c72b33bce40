"""The work of answering with drafted tokens over the paged cache, as a list of measurable cases.

A step of a model that is given drafted tokens appends their keys behind the cached ones, attends, decides which drafts
stand and puts the rows of those together:

* `attend`: the drafts of a sequence form a tree; each sees the cached keys, its ancestors and itself.  The tree is worked
  out once a step, then every layer attends;
* `verify`: the target's probabilities and given random numbers say which drafts stand, and draw the token behind them;
* `keep`: the cached rows of the drafts that stand move together, in all layers.

Rows have the values the path meets in a model: q and k are RMS-normalised rows (norm sqrt(head_dim)), v is N(0, 1),
pages come from a shuffled free list; logits are N(0, 3^2) with a few likely tokens a row, drafts are drawn from a
distribution near the target's, or are its likely tokens.  Lengths and trees follow from the case alone; everything else
follows from the seed.
"""

import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
DEVICE = "cuda"


def _ops():
    package = os.path.join(os.getcwd(), "falcon-perception_amd")
    if package not in sys.path:
        sys.path.insert(1, package)
    from falcon_perception_amd import ops

    return ops


# ------------------------------------------------------------------------------------------------------------- cases

def _attend(name, *, batch, groups, prefix_lo, prefix_hi, own_lo, own_hi, drafts_lo, drafts, branch, q_heads, cached_heads,
            head_dim, page_size, dtype, layers, sinks, room):
    case = dict(kind="attend", batch=batch, groups=groups, prefix_lo=prefix_lo, prefix_hi=prefix_hi, own_lo=own_lo,
                own_hi=own_hi, drafts_lo=drafts_lo, drafts=drafts, branch=branch, q_heads=q_heads,
                cached_heads=cached_heads, head_dim=head_dim, page_size=page_size, dtype=dtype, layers=layers,
                sinks=sinks, room=room)
    return case if name is None else dict(name=name, **case)


def _verify(name, *, batch, drafts_lo, drafts, branch, vocab, dtype, probs, greedy, temperature):
    case = dict(kind="verify", batch=batch, drafts_lo=drafts_lo, drafts=drafts, branch=branch, vocab=vocab, dtype=dtype,
                probs=probs, greedy=greedy, temperature=temperature)
    return case if name is None else dict(name=name, **case)


def _keep(name, *, batch, drafts, kept_lo, kept_hi, layers, cached_heads, head_dim, page_size, dtype, old_lo, old_hi):
    case = dict(kind="keep", batch=batch, drafts=drafts, kept_lo=kept_lo, kept_hi=kept_hi, layers=layers,
                cached_heads=cached_heads, head_dim=head_dim, page_size=page_size, dtype=dtype, old_lo=old_lo,
                old_hi=old_hi)
    return case if name is None else dict(name=name, **case)


def listed():
    return [
        # A first try in float32: three short conversations with four drafts each, pages of 64 tokens; what a step costs
        # before the first key.
        _attend("tree_three_f32", batch=3, groups=0, prefix_lo=0, prefix_hi=0, own_lo=70, own_hi=311, drafts_lo=5,
                drafts=5, branch=1, q_heads=8, cached_heads=8, head_dim=64, page_size=64, dtype="f32", layers=2,
                sinks=False, room=4096),
        # A full server of the default model: 64 requests, each with a chain of four drafts behind its last token.
        _attend("chain_serving", batch=64, groups=0, prefix_lo=0, prefix_hi=0, own_lo=1088, own_hi=4096, drafts_lo=2,
                drafts=5, branch=1, q_heads=16, cached_heads=8, head_dim=128, page_size=128, dtype="bf16", layers=4,
                sinks=False, room=8192),
        # Sixteen requests with trees of up to 32 tokens, the sink gate.
        _attend("tree_serving", batch=16, groups=0, prefix_lo=0, prefix_hi=0, own_lo=513, own_hi=8000, drafts_lo=17,
                drafts=32, branch=3, q_heads=16, cached_heads=8, head_dim=128, page_size=128, dtype="bf16", layers=4,
                sinks=True, room=8192),
        # Pages of text: 64 requests on long contexts, trees of 24 tokens, four query heads per cached head.
        _attend("tree_long", batch=64, groups=0, prefix_lo=0, prefix_hi=0, own_lo=4352, own_hi=12288, drafts_lo=24,
                drafts=24, branch=2, q_heads=32, cached_heads=8, head_dim=128, page_size=128, dtype="bf16", layers=2,
                sinks=False, room=16384),
        # The small variants in half precision: 37 requests on four pictures, eight query heads per cached head, an odd
        # page size, trees of odd sizes.
        _attend("tree_pictures_f16", batch=37, groups=4, prefix_lo=577, prefix_hi=2311, own_lo=1, own_hi=700,
                drafts_lo=1, drafts=13, branch=4, q_heads=32, cached_heads=4, head_dim=64, page_size=48, dtype="f16",
                layers=4, sinks=True, room=4100),
        # One request of a chat, four drafts from its own text: the latency of a step's decision.
        _verify("verify_one", batch=1, drafts_lo=5, drafts=5, branch=1, vocab=65536, dtype="bf16", probs="none",
                greedy=0, temperature=0.8),
        # A full server whose drafts a smaller model drew: 64 chains of up to seven, float32 logits, its probabilities.
        _verify("verify_drawn", batch=64, drafts_lo=3, drafts=8, branch=1, vocab=65536, dtype="f32", probs="f32",
                greedy=0, temperature=0.9),
        # Trees of likely tokens, some of the requests greedy.
        _verify("verify_trees", batch=32, drafts_lo=17, drafts=33, branch=3, vocab=65536, dtype="bf16", probs="none",
                greedy=9, temperature=1.0),
        # An odd vocabulary in half precision, the draft's probabilities in half precision, too.
        _verify("verify_odd", batch=7, drafts_lo=1, drafts=4, branch=1, vocab=50021, dtype="f16", probs="f16",
                greedy=2, temperature=0.7),
        # Three requests, a small float32 cache.
        _keep("keep_three_f32", batch=3, drafts=5, kept_lo=2, kept_hi=4, layers=2, cached_heads=8, head_dim=64,
              page_size=64, dtype="f32", old_lo=40, old_hi=100),
        # A full server's trees, in all 28 layers of the engine's cache.
        _keep("keep_serving", batch=64, drafts=32, kept_lo=1, kept_hi=7, layers=28, cached_heads=16, head_dim=128,
              page_size=128, dtype="bf16", old_lo=64, old_hi=200),
    ]


# ------------------------------------------------------------------------------------------------------- drawn cases

def _log(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


# what a drawn case may cost at most: a little less than the largest listed ones
_MOST = {"attend": (4.0e9, 4.0e11), "verify": (1.5e8, 1.0e9), "keep": (2.0e8, 1.0)}


def draw(rng):
    while True:
        kind = rng.choice(["attend", "attend", "verify", "verify", "keep"])
        case = {"attend": _draw_attend, "verify": _draw_verify, "keep": _draw_keep}[kind](rng)
        w = work(case)
        if w["bytes"] <= _MOST[kind][0] and w["flops"] <= _MOST[kind][1] and _pool_bytes(case) < 8.0e9:
            return case


def _draw_attend(rng):
    cached = rng.choice([2, 4, 8])
    batch = _log(rng, 1, 128)
    groups = min(batch, _log(rng, 1, 8)) if rng.random() < 0.4 else 0
    prefix_hi = _log(rng, 65, 8000) if groups else 0
    own_hi = _log(rng, 1, 12000)
    drafts = _log(rng, 1, 64)
    need = prefix_hi + own_hi + drafts
    return _attend(None, batch=batch, groups=groups, prefix_lo=_log(rng, 64, prefix_hi) if groups else 0,
                   prefix_hi=prefix_hi, own_lo=rng.randint(0, own_hi), own_hi=own_hi, drafts_lo=rng.randint(0, drafts),
                   drafts=drafts, branch=rng.choice([1, 1, 2, 3, 8]), q_heads=cached * rng.choice([1, 2, 2, 4, 8]),
                   cached_heads=cached, head_dim=rng.choice([64, 128, 128]),
                   page_size=rng.choice([16, 48, 64, 128, 128, 256]), dtype=rng.choice(["bf16", "bf16", "f16", "f32"]),
                   layers=rng.choice([1, 2, 4]), sinks=rng.random() < 0.25, room=rng.choice([need, 16384, 32768]))


def _draw_verify(rng):
    batch, drafts = _log(rng, 1, 256), _log(rng, 1, 64)
    probs = rng.choice(["none", "none", "f32", "same"])
    dtype = rng.choice(["bf16", "f16", "f32", "f32"])
    return _verify(None, batch=batch, drafts_lo=rng.randint(0, drafts), drafts=drafts,
                   branch=1 if probs != "none" else rng.choice([1, 2, 3, 8]), vocab=_log(rng, 1000, 150000), dtype=dtype,
                   probs=dtype if probs == "same" else probs, greedy=rng.choice([0, 0, rng.randint(0, batch), batch]),
                   temperature=round(rng.uniform(0.3, 1.5), 2))


def _draw_keep(rng):
    drafts, page_size = _log(rng, 1, 64), rng.choice([16, 48, 64, 128, 128, 256])
    kept_hi = rng.randint(1, min(drafts, 12))
    old_hi = rng.randint(1, 3 * page_size)
    return _keep(None, batch=_log(rng, 1, 128), drafts=drafts, kept_lo=rng.randint(0, kept_hi), kept_hi=kept_hi,
                 layers=_log(rng, 1, 28), cached_heads=rng.choice([2, 4, 8, 16]), head_dim=rng.choice([64, 128]),
                 page_size=page_size, dtype=rng.choice(["bf16", "f16", "f32"]), old_lo=rng.randint(0, old_hi),
                 old_hi=old_hi)


# ------------------------------------------------------------------------------------------------ lengths and trees

def _spread(n, lo, hi):
    """n whole numbers over lo .. hi, in no order."""
    if n == 1:
        return [(lo + hi) // 2]
    return [lo + int((hi - lo) * ((0.5 + 0.6180339887498949 * i) % 1.0) + 0.5) for i in range(n)]


def _attend_lengths(case):
    """Keys of the prefixes, and per sequence: (group or -1, shared keys, own cached keys, drafts)."""
    prefixes = _spread(case["groups"], case["prefix_lo"], case["prefix_hi"]) if case["groups"] else []
    behind = _spread(case["batch"], case["own_lo"], case["own_hi"])
    counts = _spread(case["batch"], case["drafts_lo"], case["drafts"])[::-1]
    out = []
    for b in range(case["batch"]):
        g = b % case["groups"] if case["groups"] else -1
        out.append((g, prefixes[g] if g >= 0 else 0, behind[b], counts[b]))
    return prefixes, out


def _parents(b, n, branch):
    """The tree of sequence b: the parent of each of its n tokens, -1 of the first.  Every other one is uneven."""
    line = []
    for j in range(n):
        if j == 0 or branch == 1 or b % 2 == 0:
            line.append(-1 if j == 0 else (j - 1) // branch)
        else:
            line.append(max(0, j - 1 - (7 * b + 5 * j + j * j) % (2 * branch)))
    return line


def _depths(line):
    depth = []
    for p in line:
        depth.append(0 if p < 0 else depth[p] + 1)
    return depth


def _kept(case):
    """Per sequence: (cached keys, kept rows).  The rows that move come from behind all that stay."""
    olds = _spread(case["batch"], case["old_lo"], case["old_hi"])
    counts = _spread(case["batch"], case["kept_lo"], case["kept_hi"])
    out = []
    for b, (old, n) in enumerate(zip(olds, counts)):
        room = case["drafts"] - n  # rows behind the kept ones, from which those that move come
        still = max(min(n, 1 + (b % 3 if n > 2 else 0)), n - room)
        step = max(1, room // max(1, n - still))
        out.append((old, [i if i < still else n + (i - still) * step + (b % step if room >= (n - still) * step else 0)
                          for i in range(n)]))
    return out


def _pool_bytes(case):
    if case["kind"] == "verify":
        return 0
    page = case["page_size"]
    if case["kind"] == "attend":
        prefixes, seqs = _attend_lengths(case)
        pages = sum(p // page for p in prefixes) + sum(s[2] // page + 3 for s in seqs)
    else:
        pages = case["batch"] * ((case["old_hi"] + case["drafts"]) // page + 1)
    return pages * page * case["layers"] * 2.0 * case["cached_heads"] * case["head_dim"] * (4 if case["dtype"] == "f32" else 2)


def work(case):
    size = {"bf16": 2, "f16": 2, "f32": 4}[case["dtype"]]
    if case["kind"] == "keep":
        rows = sum(1 for _, path in _kept(case) for i, p in enumerate(path) if p != i)
        return {"bytes": 2.0 * rows * case["layers"] * 2 * case["cached_heads"] * case["head_dim"] * size
                + 12.0 * case["batch"] + 4.0 * case["batch"] * case["drafts"], "flops": 0.0}
    if case["kind"] == "verify":
        rows = sum(_spread(case["batch"], case["drafts_lo"], case["drafts"])[::-1])
        probs = {"none": 0, "bf16": 2, "f16": 2, "f32": 4}[case["probs"]]
        return {"bytes": rows * case["vocab"] * float(size) + case["batch"] * (case["vocab"] * float(probs) + 8)
                + case["batch"] * case["drafts"] * 28.0, "flops": 2.0 * rows * case["vocab"]}
    prefixes, seqs = _attend_lengths(case)
    keys = sum(prefixes) + sum(s[2] + s[3] for s in seqs)
    tokens = sum(s[3] for s in seqs)
    pairs = 0
    for b, (_, shared, behind, n) in enumerate(seqs):
        pairs += n * (shared + behind) + sum(d + 1 for d in _depths(_parents(b, n, case["branch"])))
    row = case["head_dim"] * size
    return {"bytes": float(case["layers"] * (2 * keys * case["cached_heads"] * row + 2 * tokens * case["q_heads"] * row
                                             + 4 * tokens * case["q_heads"] + 8 * keys // case["page_size"])
                           + 20 * case["batch"] * case["drafts"]),
            "flops": 4.0 * case["layers"] * pairs * case["q_heads"] * case["head_dim"]}


# ------------------------------------------------------------------------------------------------------------ inputs

def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    order = torch.Generator().manual_seed(seed + 1)
    return {"attend": _prepare_attend, "verify": _prepare_verify, "keep": _prepare_keep}[case["kind"]](case, gen, order)


def _randn(gen, shape, dtype):
    out = torch.empty(shape, dtype=dtype, device=DEVICE)
    flat = out.view(-1)
    for i in range(0, flat.numel(), 1 << 28):  # in pieces: float32 copies of a large pool are not kept
        part = flat[i:i + (1 << 28)]
        part.copy_(torch.randn(part.numel(), generator=gen, device=DEVICE))
    return out


def _unit_rows(x):
    """RMS-normalised rows, as the model hands q and k to the cache."""
    flat = x.view(-1, x.shape[-1])
    for i in range(0, flat.shape[0], 1 << 21):
        part = flat[i:i + (1 << 21)]
        f = part.float()
        part.copy_(f * torch.rsqrt(f.square().mean(dim=-1, keepdim=True)))
    return x


def _prepare_attend(case, gen, order):
    dtype, page = DTYPES[case["dtype"]], case["page_size"]
    prefixes, seqs = _attend_lengths(case)
    columns = -(-case["room"] // page)
    whole = [p // page for p in prefixes]  # pages of a prefix that are shared; the one it ends in is everybody's own
    wanted = [-(-(shared + behind + n) // page) - (whole[g] if g >= 0 else 0) for g, shared, behind, n in seqs]
    n_pages = 1 + sum(whole) + sum(wanted) + 3
    pages = (torch.randperm(n_pages - 1, generator=order) + 1).tolist()
    take = lambda n: [pages.pop() for _ in range(n)]
    shared_pages = [take(n) for n in whole]
    B, slots = case["batch"], (torch.randperm(case["batch"], generator=order) + 1).tolist()
    table = torch.full((B + 1, columns), -1, dtype=torch.int64)
    table[0] = 0
    ids, lens = torch.zeros(B + 1, dtype=torch.int32), torch.zeros(B + 1, dtype=torch.int32)
    parents = torch.full((B, case["drafts"]), -2, dtype=torch.int32)
    cached = torch.zeros(B, dtype=torch.int32)
    first, tails = {}, []
    rows = torch.randperm(B, generator=order).tolist()  # the batch is in no order of its groups
    batch_idx = torch.zeros(B, dtype=torch.int64)
    for b, (g, shared, behind, n) in enumerate(seqs):
        s, r = slots[b], rows[b]
        line = (shared_pages[g] if g >= 0 else []) + take(wanted[b])
        table[s, :len(line)] = torch.tensor(line, dtype=torch.int64)
        batch_idx[r] = s
        cached[r] = shared + behind
        parents[r, :n] = torch.tensor(_parents(b, n, case["branch"]), dtype=torch.int32)
        if g >= 0:
            ids[s], lens[s] = g + 1, shared
            if shared % page:
                if g in first:
                    tails.append((first[g], line[whole[g]], shared % page))
                elif len(line) > whole[g]:
                    first[g] = line[whole[g]]
    L, Hc, D = case["layers"], case["cached_heads"], case["head_dim"]
    pool = torch.empty((L, 2, Hc, n_pages * page, D), dtype=dtype, device=DEVICE)
    for layer in range(L):
        for t in range(2):
            pool[layer, t] = _randn(gen, (Hc, n_pages * page, D), dtype)
        _unit_rows(pool[layer, 0])
    paged = pool.view(L, 2, Hc, n_pages, page, D)
    for src, dst, n in tails:
        paged[:, :, :, dst, :n] = paged[:, :, :, src, :n]
    q = _unit_rows(_randn(gen, (L, B, case["q_heads"], case["drafts"], D), dtype))
    shares = case["groups"] > 0
    state = dict(case=case, pool=pool, q=q, table=table.to(DEVICE), batch_idx=batch_idx.to(DEVICE),
                 parents=parents.to(DEVICE), cached=cached.to(DEVICE), ids=ids.to(DEVICE) if shares else None,
                 lens=lens.to(DEVICE) if shares else None, keys=max(s[1] + s[2] for s in seqs) + case["drafts"],
                 sinks=torch.randn(case["q_heads"], generator=gen, device=DEVICE) if case["sinks"] else None)
    if own:  # what a program keeps for all its steps
        ops, shape = _ops(), dict(q_heads=case["q_heads"], cached_heads=Hc, head_dim=D)
        state["plan"] = torch.empty(ops.shared_decode_plan_bytes(B, case["drafts"], **shape), dtype=torch.uint8,
                                    device=DEVICE)
        state["workspace"] = torch.empty(ops.shared_decode_workspace_bytes(B, case["drafts"], **shape),
                                         dtype=torch.uint8, device=DEVICE)
    return state


def _prepare_verify(case, gen, order):
    B, S, V, dtype = case["batch"], case["drafts"], case["vocab"], DTYPES[case["dtype"]]
    rand = lambda *shape: torch.rand(shape, generator=gen, device=DEVICE)
    randn = lambda *shape: torch.randn(shape, generator=gen, device=DEVICE)
    greedy = torch.zeros(B, dtype=torch.bool)
    greedy[torch.randperm(B, generator=order)[:case["greedy"]]] = True
    temperatures = torch.where(greedy, 0.0, case["temperature"]).to(DEVICE)
    counts = _spread(B, case["drafts_lo"], case["drafts"])[::-1]
    parents = torch.full((B, S), -2, dtype=torch.int32)
    for b, n in enumerate(counts):
        parents[b, :n] = torch.tensor(_parents(b, n, case["branch"]), dtype=torch.int32)
    logits = torch.empty((B, S, V), dtype=dtype, device=DEVICE)
    likely = torch.randint(0, V, (B, S, 8), generator=gen, device=DEVICE)  # of every row; the drafts are among them
    # (the likely tokens' logits over the sum of the others': about exp(4.5) a token)
    heights = math.log(V) + 4.5 - torch.tensor([-0.5, 0.3, 1.0, 1.7, 2.3, 3.0, 3.6, 4.2], device=DEVICE)
    probs = torch.empty((B, S, V), dtype=DTYPES[case["probs"]], device=DEVICE) if case["probs"] != "none" else None
    tokens = torch.randint(0, V, (B, S), generator=gen, device=DEVICE)
    place = torch.zeros((B, S), dtype=torch.int64)  # which of its parent's likely tokens a draft is
    for b, n in enumerate(counts):
        seen = {}
        for j in range(1, n):
            p = int(parents[b, j])
            place[b, j] = seen.get(p, 0) % 8
            seen[p] = seen.get(p, 0) + 1
    place = place.to(DEVICE)
    for b in range(B):
        x = 3.0 * randn(S, V)
        x.scatter_(1, likely[b], heights + 0.7 * randn(S, 8))
        logits[b] = x.to(dtype)
        if probs is not None:  # a smaller model's, near the target's; its drafts are drawn from them
            y = (logits[b].float() + 0.8 * randn(S, V)) / case["temperature"]
            probs[b] = torch.softmax(y, -1).to(probs.dtype)
            tokens[b, 1:] = (torch.log(probs[b, :-1].float()) - torch.log(-torch.log(rand(S - 1, V)))).argmax(-1)
    if probs is None:
        b = torch.arange(B, device=DEVICE)[:, None]
        tokens[:, 1:] = likely[b, parents[:, 1:].to(DEVICE).long().clamp(min=0), place[:, 1:]]
    state = dict(case=case, logits=logits, tokens=tokens, parents=parents.to(DEVICE), uniforms=rand(B, S),
                 temperatures=temperatures, probs=probs)
    if own:
        state["workspace"] = torch.empty(_ops().verify_workspace_bytes(B, S, V), dtype=torch.uint8, device=DEVICE)
    return state


def _prepare_keep(case, gen, order):
    page, B = case["page_size"], case["batch"]
    per = (case["old_hi"] + case["drafts"]) // page + 1
    pages = (torch.randperm(B * per + 2, generator=order) + 1).tolist()
    slots = (torch.randperm(B + 2, generator=order) + 1).tolist()[:B]
    table = torch.full((B + 3, per + 2), -1, dtype=torch.int64)
    table[0] = 0
    path = torch.full((B, case["drafts"]), -1, dtype=torch.int32)
    cached = torch.zeros(B, dtype=torch.int32)
    for b, (old, line) in enumerate(_kept(case)):
        table[slots[b], :per] = torch.tensor([pages.pop() for _ in range(per)], dtype=torch.int64)
        cached[b] = old
        path[b, :len(line)] = torch.tensor(line, dtype=torch.int32)
    pool = _randn(gen, (case["layers"], 2, 1, case["cached_heads"], (B * per + 3) * page, case["head_dim"]),
                  DTYPES[case["dtype"]])
    return dict(case=case, pool=pool, table=table.to(DEVICE), batch_idx=torch.tensor(slots, device=DEVICE),
                cached=cached.to(DEVICE), path=path.to(DEVICE))


# -------------------------------------------------------------------------------------------------------------- runs

def run(state):
    return {"attend": _run_attend, "verify": _run_verify, "keep": _run_keep}[state["case"]["kind"]](state)


def _run_attend(state):
    case = state["case"]
    if own:
        ops = _ops()
        tree = ops.draft_tree(state["parents"], state["cached"])
        plan = ops.tree_decode_plan(state["batch_idx"], tree, state["table"], q_heads=case["q_heads"],
                                    cached_heads=case["cached_heads"], head_dim=case["head_dim"],
                                    max_context=case["room"], prefix_ids=state["ids"], prefix_lens=state["lens"],
                                    plan=state["plan"])
        result = [tree.masks, tree.input_pos, tree.rope_pos]
        for layer in range(case["layers"]):
            result += ops.paged_decode_tree(state["q"][layer], state["pool"][layer, 0], state["pool"][layer, 1],
                                            state["table"], state["batch_idx"], tree, case["page_size"], case["room"],
                                            prefix_ids=state["ids"], prefix_lens=state["lens"], sinks=state["sinks"],
                                            plan=plan, workspace=state["workspace"])
        return result
    masks, input_pos, rope_pos = _plain_tree(state["parents"], state["cached"])
    result = [masks, input_pos, rope_pos]
    for layer in range(case["layers"]):
        result += _plain_attend(state["q"][layer], state["pool"][layer], state["table"], state["batch_idx"], masks,
                                state["cached"], case["page_size"], state["keys"], state["sinks"])
    return result


def _plain_tree(parents, cached):
    """Which drafts each token sees (bit i: draft i), its row behind the cached keys and its place in the text."""
    B, S = parents.shape
    masks = torch.zeros((B, S), dtype=torch.int64, device=parents.device)
    depth = torch.zeros((B, S), dtype=torch.int64, device=parents.device)
    for j in range(S):
        p = parents[:, j].long()
        at = p.clamp(0, max(j - 1, 0))[:, None]
        above = masks.gather(1, at)[:, 0]
        there = (p == -1) | ((p >= 0) & (p < j) & (above != 0))
        masks[:, j] = torch.where(there, torch.where(p >= 0, above, 0) | (1 << j if j < 63 else -(1 << 63)), 0)
        depth[:, j] = torch.where(there & (p >= 0), depth.gather(1, at)[:, 0] + 1, 0)
    here = masks != 0
    rows = cached[:, None] + torch.arange(S, device=parents.device)
    return masks, torch.where(here, rows, -1).int(), torch.where(here, cached[:, None] + depth, 0).int()


def _plain_attend(q, pool, table, batch_idx, masks, cached, page, keys, sinks):
    """Every sequence over the keys that its row of the page table names, a few sequences at a time."""
    B, Hq, S, D = q.shape
    Hc = pool.shape[1]
    t = torch.arange(keys, device=q.device)
    slots = table[batch_idx][:, (t // page).clamp(max=table.shape[1] - 1)].clamp(min=0) * page + t % page  # [B, keys]
    out, lse = torch.empty_like(q), torch.empty((B, Hq, S), device=q.device)
    per = max(1, (1 << 26) // (keys * Hc * D))
    for b in range(0, B, per):
        rows = slots[b:b + per]
        n = rows.shape[0]
        k, v = (pool[i][:, rows].transpose(0, 1).float() for i in range(2))  # [n, Hc, keys, D]
        scores = q[b:b + per].float().reshape(n, Hc, Hq // Hc * S, D) @ k.transpose(2, 3).contiguous() * D ** -0.5
        behind = t - cached[b:b + per, None]  # [n, keys]
        bit = (masks[b:b + per, :, None] >> behind.clamp(0, 63)[:, None]) & 1
        seen = torch.where(behind[:, None] < 0, masks[b:b + per, :, None] != 0, (bit != 0) & (behind[:, None] < S))
        scores = scores.view(n, Hq, S, keys).masked_fill(~seen[:, None], -math.inf)
        top = scores.amax(dim=3, keepdim=True).clamp(min=-3.0e38)
        p = torch.exp(scores - top)
        total = p.sum(dim=3, keepdim=True)
        o = (p.view(n, Hc, -1, keys) @ v).view(n, Hq, S, D) / total
        o = o.masked_fill(total == 0, 0.0)
        part = top.squeeze(3) + torch.log(total.squeeze(3))
        if sinks is not None:
            o = o * (1.0 / (1.0 + torch.exp(sinks[:, None] - part)))[..., None]
            o = o.masked_fill(total == 0, 0.0)
        out[b:b + per] = o.to(q.dtype)
        lse[b:b + per] = part
    return out, lse


def _run_verify(state):
    if own:
        return list(_ops().verify_drafts(state["logits"], state["tokens"], state["parents"], state["uniforms"],
                                         temperatures=state["temperatures"], draft_probs=state["probs"],
                                         workspace=state["workspace"]))
    return _plain_verify(state["logits"], state["tokens"], state["parents"], state["uniforms"], state["temperatures"],
                         state["probs"])


def _plain_verify(logits, tokens, parents, uniforms, temperatures, probs):
    """In 64 bits: a decision lies next to a border wherever 32 would be used."""
    B, S, V = logits.shape
    dev, parents = logits.device, parents.long()
    peak, total = (torch.empty((B, S), dtype=torch.float64, device=dev) for _ in range(2))
    best = torch.empty((B, S), dtype=torch.int64, device=dev)
    heat = torch.where(temperatures > 0, temperatures, 1.0).double()

    def weights(x, top, heat):
        return torch.where(x == top, 1.0, torch.exp((x - top) / heat)).masked_fill(x == -math.inf, 0.0)

    def values(x):
        return x.double().masked_fill(torch.isnan(x), -math.inf)

    per = max(1, (1 << 27) // (S * V))
    for b in range(0, B, per):
        x = values(logits[b:b + per])
        peak[b:b + per] = x.amax(-1)
        best[b:b + per] = torch.where(x == peak[b:b + per, :, None], torch.arange(V, device=dev), V).amin(-1)
        total[b:b + per] = weights(x, peak[b:b + per, :, None], heat[b:b + per, None, None]).sum(-1)
    best = torch.where(peak == -math.inf, -1, best)

    rows = torch.arange(B, device=dev)
    at = parents.clamp(min=0, max=S - 1)
    known = (tokens >= 0) & (tokens < V)
    named = tokens.clamp(0, V - 1)
    weight = weights(values(logits[rows[:, None], at, named]), peak.gather(1, at), heat[:, None]).masked_fill(~known, 0.0)
    share = None if probs is None else probs[rows[:, None], at, named].double()
    earlier = torch.arange(S, device=dev)
    twin = ((parents[:, :, None] == parents[:, None]) & (tokens[:, :, None] == tokens[:, None]) & (earlier[:, None] > earlier)).any(2)
    weight = weight.masked_fill(twin, 0.0)

    node = torch.zeros(B, dtype=torch.int64, device=dev)
    count = torch.zeros(B, dtype=torch.int64, device=dev)
    refused = torch.zeros(B, dtype=torch.float64, device=dev)
    tested = torch.zeros(B, dtype=torch.bool, device=dev)
    path = torch.full((B, S + 1), -1, dtype=torch.int64, device=dev)
    there = parents[:, 0] == -1
    path[:, 0] = torch.where(there, 0, -1)
    u, greedy = uniforms.double(), ~(temperatures > 0)
    for j in range(1, S):
        child = there & (parents[:, j] == node)
        z = total.gather(1, node[:, None])[:, 0]
        if probs is None:
            takes = u[:, j] * (z - refused) < weight[:, j]
        else:
            takes = (u[:, j] * share[:, j] * z < weight[:, j]) & ~tested
        takes = torch.where(greedy, tokens[:, j] == best.gather(1, node[:, None])[:, 0], takes)
        takes &= child & known[:, j]
        tested = torch.where(child, ~takes, tested)
        refused = torch.where(takes, 0.0, refused + torch.where(child, weight[:, j], 0.0))
        node = torch.where(takes, j, node)
        count = count + takes
        path.scatter_(1, torch.where(takes, count, S)[:, None], j)
    path = path[:, :S]

    x = values(logits[rows, node])
    w = weights(x, peak.gather(1, node[:, None]), heat[:, None])
    if probs is None:
        out = (parents == node[:, None]) & known & (earlier > node[:, None])
        w = w.scatter_reduce(1, torch.where(out, named, 0), torch.where(out, 0.0, math.inf).double(), "amin")
    else:
        left = (w / total.gather(1, node[:, None]) - probs[rows, node].double()).clamp(min=0.0)
        w = torch.where((tested & (left.sum(-1) > 0))[:, None], left, w)
    sums = torch.cumsum(w, 1)
    drawn = torch.searchsorted(sums, (u[:, :1] * sums[:, -1:]), right=True)[:, 0]
    last = torch.where(w > 0, torch.arange(V, device=dev), -1).amax(1)
    drawn = torch.where(greedy, best.gather(1, node[:, None])[:, 0], torch.minimum(drawn, last))

    answer = torch.full((B, S), -1, dtype=torch.int64, device=dev)
    ahead = path[:, 1:]
    answer[:, :S - 1] = torch.where(ahead >= 0, tokens.gather(1, ahead.clamp(min=0)), -1)
    answer.scatter_(1, count[:, None], torch.where(there, drawn, -1)[:, None])

    # what the target thinks of each answered token: the log of its share where it stands
    stands = torch.where(path >= 0, path, 0)
    picked = values(logits[rows[:, None], stands, answer.clamp(min=0)])
    top = peak.gather(1, stands)
    says = torch.where(picked == top, 0.0, (picked - top) / heat[:, None]) - torch.log(total.gather(1, stands))
    return [count.int(), path.int(), answer, torch.where(answer >= 0, says, 0.0).float()]


def _run_keep(state):
    page = state["case"]["page_size"]
    if own:
        _ops().keep_rows(state["pool"], state["table"], state["batch_idx"], state["cached"], state["path"], page)
        return state["pool"]
    pool, path = state["pool"], state["path"].long()
    flat = pool.view(-1, *pool.shape[-2:])
    line = state["table"][state["batch_idx"]]
    cached = state["cached"].long()[:, None]
    to = torch.arange(path.shape[1], device=path.device).expand_as(path)
    moved = path > to  # the others stand for the first row, which stays
    src, dst = (line.gather(1, (cached + torch.where(moved, i, 0)) // page) * page + (cached + torch.where(moved, i, 0)) % page
                for i in (path, to))
    flat[:, dst] = flat[:, src]
    return pool


# ------------------------------------------------------------------------------------------------------- 64-bit values

def exact(case, seed):
    """The moved pool; out and lse of every layer; logarithms of the answer's probabilities.  Decisions and trees are whole
    numbers."""
    state = prepare(case, seed)
    if case["kind"] == "verify":
        return [None, None, None, _exact_verify(state)]
    page = case["page_size"]
    if case["kind"] == "keep":
        pool, table = state["pool"].double(), state["table"].tolist()
        for slot, old, line in zip(*(state[name].tolist() for name in ("batch_idx", "cached", "path"))):
            where = lambda t: table[slot][t // page] * page + t % page
            for i, p in enumerate(line):
                if p > i:
                    pool[..., where(old + i), :] = pool[..., where(old + p), :]
        return pool
    lines, group = state["table"].cpu(), case["q_heads"] // case["cached_heads"]
    slots, trees, olds = (state[name].tolist() for name in ("batch_idx", "parents", "cached"))
    result = [None, None, None]
    for layer in range(case["layers"]):
        q = state["q"][layer]
        out = torch.zeros(q.shape, dtype=torch.float64, device=DEVICE)
        lse = torch.full(q.shape[:3], -math.inf, dtype=torch.float64, device=DEVICE)
        for b, slot in enumerate(slots):
            n = sum(p > -2 for p in trees[b])
            if n == 0:
                continue
            hidden = torch.ones((n, olds[b] + n), dtype=torch.bool)
            hidden[:, :olds[b]] = False
            for j in range(n):
                at = j
                while at >= 0:
                    hidden[j, olds[b] + at] = False
                    at = trees[b][at]
            ids = lines[slot, :-(-hidden.shape[1] // page)].tolist()
            k, v = (torch.cat([state["pool"][layer, i][:, p * page:(p + 1) * page] for p in ids], 1)[:, :hidden.shape[1]]
                    .double().repeat_interleave(group, 0) for i in range(2))  # one a query head
            scores = torch.bmm(q[b, :, :n].double(), k.mT.contiguous()) / math.sqrt(case["head_dim"])
            scores.masked_fill_(hidden.to(DEVICE), -math.inf)
            lse[b, :, :n] = torch.logsumexp(scores, 2)
            out[b, :, :n] = torch.bmm(torch.softmax(scores, 2), v)
        if state["sinks"] is not None:
            out *= torch.sigmoid(lse - state["sinks"].double()[:, None])[..., None]
        result += [out, lse]
    return result


def _exact_verify(state):
    """One request after the other, one token after the other."""
    B, S, V = state["logits"].shape
    result = torch.zeros((B, S), dtype=torch.float64)
    trees, names, chances, heats = (state[n].tolist() for n in ("parents", "tokens", "uniforms", "temperatures"))
    for b in range(B):
        node, depth = 0, 0
        while trees[b][0] == -1:
            row = state["logits"][b, node].double()
            says = torch.log_softmax(row / (heats[b] if heats[b] > 0 else 1.0), 0)
            left, stands = torch.exp(says), None
            for j in [j for j in range(1, S) if trees[b][j] == node]:
                name = names[b][j]
                if heats[b] <= 0:
                    takes = name == int(row.argmax())
                elif state["probs"] is None:
                    takes = chances[b][j] * float(left.sum()) < float(left[name])
                else:
                    takes = chances[b][j] * float(state["probs"][b, node, name].double()) < float(left[name])
                if takes:
                    stands = j
                    break
                if state["probs"] is None:
                    left[name] = 0.0
                elif heats[b] > 0:
                    rest = (left - state["probs"][b, node].double()).clamp(min=0.0)
                    left = rest if float(rest.sum()) > 0 else left
                    break
            if stands is None:
                if heats[b] <= 0:
                    name = int(row.argmax())
                else:
                    sums = torch.cumsum(left, 0)
                    name = int((sums <= chances[b][0] * sums[-1]).sum())
                    name = min(name, int(left.nonzero()[-1]))
            else:
                name = names[b][stands]
            result[b, depth] = says[name]
            if stands is None:
                break
            node, depth = stands, depth + 1
    return result.to(DEVICE)
