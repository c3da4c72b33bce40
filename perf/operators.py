"""The work of serving many requests on one cached prefix, as a list of measurable cases.

Requests about one picture (or one page of text) have the same first keys.  An engine that serves them together does
three things beside the calls it makes already:

* `tables`: the page tables and the packed rows of a step, from the lengths of its requests, some of which fork from a
  cached prefix;
* `copy`: the page in which a forked prefix ends is copied for every request that will write behind it, in all layers;
* `attend`: the new tokens of the batch attend over the shared keys, which are read once for all, and over their own.

Rows have the values the path meets in a model: q and k are RMS-normalised rows (norm sqrt(head_dim)), v is N(0, 1),
pages come from a shuffled free list.  Lengths are spread over their range by a fixed low-discrepancy sequence, so
`work` knows them from the case alone; everything else follows from the seed.
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

def _attend(name, *, batch, groups, loners, prefix_lo, prefix_hi, own_lo, own_hi, tokens, q_heads, cached_heads,
            head_dim, page_size, dtype, layers, sinks, room):
    case = dict(kind="attend", batch=batch, groups=groups, loners=loners, prefix_lo=prefix_lo, prefix_hi=prefix_hi,
                own_lo=own_lo, own_hi=own_hi, tokens=tokens, q_heads=q_heads, cached_heads=cached_heads,
                head_dim=head_dim, page_size=page_size, dtype=dtype, layers=layers, sinks=sinks, room=room)
    return case if name is None else dict(name=name, **case)


def _tables(name, *, batch, forks, parents, old_lo, old_hi, add_lo, add_hi, page_size, columns, row_multiple):
    case = dict(kind="tables", batch=batch, forks=forks, parents=parents, old_lo=old_lo, old_hi=old_hi, add_lo=add_lo,
                add_hi=add_hi, page_size=page_size, columns=columns, row_multiple=row_multiple)
    return case if name is None else dict(name=name, **case)


def _copy(name, *, pages, pool_pages, rows_lo, rows_hi, layers, cached_heads, head_dim, page_size, dtype):
    case = dict(kind="copy", pages=pages, pool_pages=pool_pages, rows_lo=rows_lo, rows_hi=rows_hi, layers=layers,
                cached_heads=cached_heads, head_dim=head_dim, page_size=page_size, dtype=dtype)
    return case if name is None else dict(name=name, **case)


def listed():
    return [
        # A first try: three questions about one small picture in float32, pages of 64 tokens; the latency of a token.
        _attend("attend_three_f32", batch=3, groups=1, loners=0, prefix_lo=261, prefix_hi=261, own_lo=9, own_hi=61,
                tokens=1, q_heads=8, cached_heads=8, head_dim=64, page_size=64, dtype="f32", layers=2, sinks=False,
                room=4096),
        # Sixteen questions about one picture of 1030 tokens; the page in which the prefix ends is each one's own.
        _attend("attend_picture", batch=16, groups=1, loners=0, prefix_lo=1030, prefix_hi=1030, own_lo=11, own_hi=190,
                tokens=1, q_heads=16, cached_heads=8, head_dim=128, page_size=128, dtype="bf16", layers=4, sinks=False,
                room=8192),
        # A full server: 64 requests on nine pictures, a few of them alone, and up to 2800 tokens of text each.
        _attend("attend_serving", batch=64, groups=9, loners=5, prefix_lo=1024, prefix_hi=4096, own_lo=64, own_hi=2800,
                tokens=1, q_heads=16, cached_heads=8, head_dim=128, page_size=128, dtype="bf16", layers=4, sinks=False,
                room=8192),
        # Pages of text read by many users: 192 requests on eight long prefixes, four query heads per cached head.
        _attend("attend_long", batch=192, groups=8, loners=0, prefix_lo=4096, prefix_hi=12288, own_lo=256, own_hi=4096,
                tokens=1, q_heads=32, cached_heads=8, head_dim=128, page_size=128, dtype="bf16", layers=2, sinks=False,
                room=16384),
        # The small variants in half precision, eight query heads per cached head, the sink gate, an odd page size.
        _attend("attend_group8_f16", batch=37, groups=4, loners=3, prefix_lo=577, prefix_hi=2311, own_lo=1, own_hi=700,
                tokens=1, q_heads=32, cached_heads=4, head_dim=64, page_size=48, dtype="f16", layers=4, sinks=True,
                room=4100),
        # The prompts of 40 requests, 3 to 24 tokens each, behind the pictures they ask about: the first step after the
        # fork.
        _attend("attend_prompts", batch=40, groups=5, loners=0, prefix_lo=1030, prefix_hi=4102, own_lo=3, own_hi=24,
                tokens=24, q_heads=16, cached_heads=8, head_dim=128, page_size=128, dtype="bf16", layers=4, sinks=False,
                room=8192),
        # One token for each of 64 running requests: a few of them need a page.
        _tables("tables_decode", batch=64, forks=0, parents=0, old_lo=1088, old_hi=4096, add_lo=1, add_hi=1,
                page_size=128, columns=64, row_multiple=1),
        # The prompts of 48 requests that fork from four cached pictures, rows padded to 128 a sequence.
        _tables("tables_fork", batch=48, forks=48, parents=4, old_lo=577, old_hi=4102, add_lo=5, add_hi=300,
                page_size=64, columns=128, row_multiple=128),
        # The admission of a whole queue: 1000 requests, some on cached prefixes, 2 million rows.
        _tables("tables_queue", batch=1000, forks=300, parents=40, old_lo=0, old_hi=2000, add_lo=64, add_hi=4000,
                page_size=128, columns=128, row_multiple=1),
        # One request forks; the last page of its prefix is copied through eight layers in float32.
        _copy("copy_one_f32", pages=1, pool_pages=16, rows_lo=37, rows_hi=37, layers=8, cached_heads=8, head_dim=64,
              page_size=64, dtype="f32"),
        # 24 requests fork in the engine's own cache of 28 layers.
        _copy("copy_forks", pages=24, pool_pages=60, rows_lo=6, rows_hi=121, layers=28, cached_heads=16, head_dim=128,
              page_size=128, dtype="bf16"),
    ]


# ------------------------------------------------------------------------------------------------------- drawn cases

def _log(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


# what a drawn case may cost at most: a little less than the largest listed ones
_MOST = {"attend": (3.0e9, 6.0e10), "tables": (6.0e7, 1.0), "copy": (6.0e8, 1.0)}


def draw(rng):
    while True:
        kind = rng.choice(["attend", "attend", "attend", "tables", "copy"])
        case = {"attend": _draw_attend, "tables": _draw_tables, "copy": _draw_copy}[kind](rng)
        w = work(case)
        if w["bytes"] <= _MOST[kind][0] and w["flops"] <= _MOST[kind][1]:
            return case


def _draw_attend(rng):
    cached = rng.choice([2, 4, 8])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    tokens = 1 if rng.random() < 0.7 else _log(rng, 2, 40)
    batch = _log(rng, 1, 192)
    loners = rng.randint(0, batch // 3) if rng.random() < 0.5 else 0
    groups = min(batch - loners, _log(rng, 1, 12))
    prefix_hi = _log(rng, 65, 12000)
    prefix_lo = _log(rng, 64, prefix_hi)
    own_hi = max(tokens, _log(rng, 1, 4000))
    own_lo = _log(rng, 1, own_hi)
    need = prefix_hi + own_hi
    return _attend(None, batch=batch, groups=groups, loners=loners, prefix_lo=prefix_lo, prefix_hi=prefix_hi,
                   own_lo=own_lo, own_hi=own_hi, tokens=tokens, q_heads=cached * rng.choice([1, 2, 2, 4, 8]),
                   cached_heads=cached, head_dim=rng.choice([64, 128, 128]),
                   page_size=rng.choice([16, 48, 64, 128, 128, 256]), dtype=dtype, layers=rng.choice([1, 2, 4]),
                   sinks=rng.random() < 0.25, room=rng.choice([need, 16384]))


def _draw_tables(rng):
    batch = _log(rng, 1, 1000)
    forks = rng.randint(0, batch) if rng.random() < 0.6 else 0
    page_size = rng.choice([16, 48, 64, 128, 128, 256])
    add_hi = 1 if rng.random() < 0.3 else _log(rng, 1, 4000)
    old_hi = _log(rng, 1, 12000)
    return _tables(None, batch=batch, forks=forks, parents=min(forks, _log(rng, 1, 40)),
                   old_lo=rng.randint(0, old_hi), old_hi=old_hi, add_lo=_log(rng, 1, add_hi), add_hi=add_hi,
                   page_size=page_size, columns=-(-(old_hi + add_hi) // page_size) + rng.randint(0, 64),
                   row_multiple=rng.choice([1, 1, 16, 128]))


def _draw_copy(rng):
    page_size = rng.choice([16, 48, 64, 128, 128, 256])
    pages = _log(rng, 1, 64)
    rows_hi = rng.randint(1, page_size)
    return _copy(None, pages=pages, pool_pages=2 * pages + rng.randint(2, 30), rows_lo=rng.randint(1, rows_hi),
                 rows_hi=rows_hi, layers=_log(rng, 1, 28), cached_heads=rng.choice([2, 4, 8, 16]),
                 head_dim=rng.choice([64, 128]), page_size=page_size, dtype=rng.choice(["bf16", "f16", "f32"]))


# ----------------------------------------------------------------------------------------------------------- lengths

def _spread(n, lo, hi):
    """n whole numbers over lo .. hi, in no order."""
    if n == 1:
        return [(lo + hi) // 2]
    return [lo + int((hi - lo) * ((0.5 + 0.6180339887498949 * i) % 1.0) + 0.5) for i in range(n)]


def _attend_lengths(case):
    """Per sequence: (group or -1, shared keys, own keys, query tokens).  The query tokens are the last of the own keys."""
    prefixes = _spread(case["groups"], case["prefix_lo"], case["prefix_hi"]) if case["groups"] else []
    behind = _spread(case["batch"], case["own_lo"], case["own_hi"])
    shared = case["batch"] - case["loners"]
    out = []
    for b in range(case["batch"]):
        g = b % case["groups"] if b < shared and case["groups"] else -1
        length = prefixes[g] if g >= 0 else 0
        out.append((g, length, behind[b], min(case["tokens"], behind[b])))
    return prefixes, out


def _table_lengths(case):
    """Parents' lengths, and per request (parent or -1, old length, new length)."""
    parents = _spread(case["parents"], max(1, case["old_lo"]), max(1, case["old_hi"])) if case["parents"] else []
    old = _spread(case["batch"], case["old_lo"], case["old_hi"])
    add = _spread(case["batch"], case["add_lo"], case["add_hi"])[::-1]
    out = []
    for b in range(case["batch"]):
        p = b % case["parents"] if b < case["forks"] and case["parents"] else -1
        o = parents[p] if p >= 0 else old[b]
        out.append((p, o, o + add[b]))
    return parents, out


def _table_sizes(case):
    """(new pages, shared blocks, rows with their padding) of all requests."""
    page, multiple = case["page_size"], case["row_multiple"]
    fresh = blocks = rows = 0
    for p, o, n in _table_lengths(case)[1]:
        have = o // page if p >= 0 else -(-o // page)
        fresh += max(0, -(-n // page) - have)
        blocks += have if p >= 0 else 0
        rows += -(-(n - o) // multiple) * multiple
    return fresh, blocks, rows


def work(case):
    size = {"bf16": 2, "f16": 2, "f32": 4}.get(case.get("dtype"), 0)
    if case["kind"] == "copy":
        rows = sum(_spread(case["pages"], case["rows_lo"], case["rows_hi"]))
        return {"bytes": 2.0 * rows * case["layers"] * 2 * case["cached_heads"] * case["head_dim"] * size, "flops": 0.0}
    if case["kind"] == "tables":
        fresh, blocks, rows = _table_sizes(case)
        return {"bytes": 20.0 * rows + 16.0 * (fresh + blocks) + 48.0 * case["batch"], "flops": 0.0}
    prefixes, seqs = _attend_lengths(case)
    keys = sum(prefixes) + sum(s[2] for s in seqs)
    tokens = sum(s[3] for s in seqs)
    # token i of n sees all keys but the n - 1 - i behind it
    pairs = sum(n * (shared + behind) - n * (n - 1) // 2 for _, shared, behind, n in seqs)
    row = case["head_dim"] * size
    return {"bytes": float(case["layers"] * (2 * keys * case["cached_heads"] * row + 2 * tokens * case["q_heads"] * row
                                             + 4 * tokens * case["q_heads"] + 8 * keys // case["page_size"])),
            "flops": 4.0 * case["layers"] * pairs * case["q_heads"] * case["head_dim"]}


# ------------------------------------------------------------------------------------------------------------ inputs

def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    order = torch.Generator().manual_seed(seed + 1)
    return {"attend": _prepare_attend, "tables": _prepare_tables, "copy": _prepare_copy}[case["kind"]](case, gen, order)


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
    wanted = [-(-(shared + behind) // page) - (whole[g] if g >= 0 else 0) for g, shared, behind, _ in seqs]
    n_pages = 1 + sum(whole) + sum(wanted) + 3
    pages = (torch.randperm(n_pages - 1, generator=order) + 1).tolist()
    take = lambda n: [pages.pop() for _ in range(n)]
    shared_pages = [take(n) for n in whole]
    B, slots = case["batch"], (torch.randperm(case["batch"], generator=order) + 1).tolist()
    table = torch.full((B + 1, columns), -1, dtype=torch.int64)
    table[0] = 0
    ids, lens = torch.zeros(B + 1, dtype=torch.int32), torch.zeros(B + 1, dtype=torch.int32)
    pos = torch.full((B, case["tokens"]), -1, dtype=torch.int32)
    first, tails = {}, []
    rows = torch.randperm(B, generator=order).tolist()  # the batch is in no order of its groups
    batch_idx = torch.zeros(B, dtype=torch.int64)
    for b, (g, shared, behind, n) in enumerate(seqs):
        s, r = slots[b], rows[b]
        line = (shared_pages[g] if g >= 0 else []) + take(wanted[b])
        table[s, :len(line)] = torch.tensor(line)
        batch_idx[r] = s
        pos[r, :n] = torch.arange(shared + behind - n, shared + behind)
        if g >= 0:
            ids[s], lens[s] = g + 1, shared
            if shared % page:
                if g in first:
                    tails.append((first[g], line[whole[g]], shared % page))
                else:
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
    q = _unit_rows(_randn(gen, (L, B, case["q_heads"], case["tokens"], D), dtype))
    state = dict(case=case, pool=pool, q=q, table=table.to(DEVICE), batch_idx=batch_idx.to(DEVICE), pos=pos.to(DEVICE),
                 ids=ids.to(DEVICE), lens=lens.to(DEVICE), keys=max(s[1] + s[2] for s in seqs),
                 sinks=torch.randn(case["q_heads"], generator=gen, device=DEVICE) if case["sinks"] else None)
    if own:  # what a program keeps for all its steps
        ops, shape = _ops(), dict(q_heads=case["q_heads"], cached_heads=Hc, head_dim=D)
        state["plan"] = torch.empty(ops.shared_decode_plan_bytes(B, case["tokens"], **shape), dtype=torch.uint8,
                                    device=DEVICE)
        state["workspace"] = torch.empty(ops.shared_decode_workspace_bytes(B, case["tokens"], **shape),
                                         dtype=torch.uint8, device=DEVICE)
    return state


def _prepare_tables(case, gen, order):
    page = case["page_size"]
    lengths, requests = _table_lengths(case)
    fresh, _, rows = _table_sizes(case)
    wanted = [-(-n // page) for n in lengths] + [-(-o // page) if p < 0 else 0 for p, o, _ in requests]
    spare = 17
    pages = (torch.randperm(sum(wanted) + fresh + spare, generator=order) + 1).tolist()
    slots = (torch.randperm(len(wanted), generator=order) + 1).tolist()
    table = torch.full((len(wanted) + 1, case["columns"]), -1, dtype=torch.int64)
    table[0] = 0
    for slot, n in zip(slots, wanted):
        table[slot, :n] = torch.tensor([pages.pop() for _ in range(n)], dtype=torch.int64)
    free = torch.zeros(len(pages) + 5, dtype=torch.int64)
    free[:len(pages)] = torch.tensor(pages)
    parent_slots, request_slots = slots[:len(lengths)], slots[len(lengths):]
    dev = lambda x, t: torch.tensor(x, dtype=t, device=DEVICE)
    return dict(case=case, table=table.to(DEVICE), free=free.to(DEVICE), count=dev([len(pages)], torch.int32),
                slots=dev(request_slots, torch.int64), old=dev([r[1] for r in requests], torch.int32),
                new=dev([r[2] for r in requests], torch.int32),
                parents=dev([parent_slots[r[0]] if r[0] >= 0 else 0 for r in requests], torch.int64), rows=rows + 64)


def _prepare_copy(case, gen, order):
    n = case["pages"]
    pages = (torch.randperm(case["pool_pages"] - 1, generator=order) + 1).tolist()
    dst = pages[:n]
    src = [pages[n + i % max(1, (len(pages) - n) // 2)] for i in range(n)]  # several forks of one prefix have one source
    pool = _randn(gen, (case["layers"], 2, 1, case["cached_heads"], case["pool_pages"] * case["page_size"],
                        case["head_dim"]), DTYPES[case["dtype"]])
    rows = _spread(n, case["rows_lo"], case["rows_hi"])
    return dict(case=case, pool=pool, src=torch.tensor(src, device=DEVICE), dst=torch.tensor(dst, device=DEVICE),
                rows=torch.tensor(rows, dtype=torch.int32, device=DEVICE))


# -------------------------------------------------------------------------------------------------------------- runs

def run(state):
    return {"attend": _run_attend, "tables": _run_tables, "copy": _run_copy}[state["case"]["kind"]](state)


def _run_attend(state):
    case = state["case"]
    step = (state["batch_idx"], state["pos"], state["ids"], state["lens"])
    if own:
        ops = _ops()
        plan = ops.shared_decode_plan(*step, q_heads=case["q_heads"], cached_heads=case["cached_heads"],
                                      head_dim=case["head_dim"], max_context=case["room"], plan=state["plan"])
        return [t for layer in range(case["layers"])
                for t in ops.paged_decode_shared(state["q"][layer], state["pool"][layer, 0], state["pool"][layer, 1],
                                                 state["table"], *step, case["page_size"], case["room"],
                                                 sinks=state["sinks"], plan=plan, workspace=state["workspace"])]
    return [t for layer in range(case["layers"])
            for t in _plain_attend(state["q"][layer], state["pool"][layer], state["table"], state["batch_idx"],
                                   state["pos"], case["page_size"], state["keys"], state["sinks"])]


def _plain_attend(q, pool, table, batch_idx, pos, page, keys, sinks):
    """Every sequence over the keys that its row of the page table names, a few sequences at a time."""
    B, Hq, S, D = q.shape
    Hc = pool.shape[1]
    t = torch.arange(keys, device=q.device)
    slots = table[batch_idx][:, t // page].clamp(min=0) * page + t % page  # [B, keys]
    out, lse = torch.empty_like(q), torch.empty((B, Hq, S), device=q.device)
    per = max(1, (1 << 26) // (keys * Hc * D))
    for b in range(0, B, per):
        rows = slots[b:b + per]
        n = rows.shape[0]
        k, v = (pool[i][:, rows].transpose(0, 1).float() for i in range(2))  # [n, Hc, keys, D]
        scores = q[b:b + per].float().reshape(n, Hc, Hq // Hc * S, D) @ k.transpose(2, 3) * D ** -0.5
        seen = t <= pos[b:b + per, :, None]  # [n, S, keys]
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


def _run_tables(state):
    case = state["case"]
    args = (state["slots"], state["old"], state["new"], state["free"], state["count"], state["table"])
    if own:
        made = _ops().step_tables(*args, case["page_size"], state["rows"], parents=state["parents"],
                                  row_multiple=case["row_multiple"])
        return [state["table"], made.batch_idx, made.input_pos, made.slot_map, made.row_starts, made.free_left,
                made.copy_src, made.copy_dst, made.copy_rows, made.status]
    return _plain_tables(*args, case["page_size"], state["rows"], state["parents"], case["row_multiple"])


def _plain_tables(slots, old, new, free, count, table, page, max_rows, parents, multiple):
    old, new = old.long(), new.long()
    columns = table.shape[1]
    fork = parents > 0
    blocks = (new + page - 1) // page
    have = torch.where(fork, old // page, (old + page - 1) // page)
    need = (blocks - have).clamp(min=0)
    behind = torch.cumsum(need, 0)
    padded = (new - old + multiple - 1) // multiple * multiple
    ends = torch.cumsum(padded, 0)
    named = torch.zeros(table.shape[0], dtype=torch.bool, device=table.device)
    named[slots.clamp(0, table.shape[0] - 1)] = True  # a parent is no request of the same call
    valid = (slots > 0) & (slots < table.shape[0]) & (old >= 0) & (new >= old) & (parents < table.shape[0])
    valid &= ~(fork & named[parents.clamp(0, table.shape[0] - 1)])
    order = torch.sort(slots).values
    twice = (order[1:] == order[:-1]).any()
    status = ((behind[-1] > count[0]).int() + 2 * (blocks > columns).any().int() + 4 * (ends[-1] > max_rows).int()
              + 8 * ((~valid).any() | twice).int())
    fine = status == 0

    # the requests' rows of the table
    c = torch.arange(columns, device=table.device)
    at = slots.clamp(0, table.shape[0] - 1)
    line = table[at]
    taken = free[(count[0] - behind[:, None] + c - have[:, None]).clamp(0, free.shape[0] - 1)]
    line = torch.where((c >= have[:, None]) & (c < blocks[:, None]), taken, line)
    line = torch.where(fork[:, None] & (c < have[:, None]), table[parents.clamp(0, table.shape[0] - 1)], line)
    table[at] = torch.where(fine, line, table[at])

    # the packed rows
    r = torch.arange(max_rows, device=table.device)
    b = torch.searchsorted(ends, r, right=True).clamp(max=slots.shape[0] - 1)
    pos = old[b] + r - (ends - padded)[b]
    real = fine & (r < ends[-1]) & (pos < new[b])
    pos = torch.where(real, pos, 0)
    slot = torch.where(real, slots[b], 0)
    where = torch.where(real, table[slot.clamp(0, table.shape[0] - 1), (pos // page).clamp(max=columns - 1)] * page
                        + pos % page, 0)

    # the page in which a forked prefix ends
    cut = fine & fork & (old % page != 0) & (blocks > have)
    last = have.clamp(max=columns - 1)
    src = torch.where(cut, table[parents.clamp(0, table.shape[0] - 1), last], -1)
    dst = torch.where(cut, table[at, last], -1)
    starts = torch.where(fine, torch.cat([torch.zeros_like(ends[:1]), ends]), 0)
    return [table, slot, pos.int(), where, starts.int(), count - torch.where(fine, behind[-1:], 0).int(), src, dst,
            torch.where(cut, old % page, 0).int(), status.int().view(1)]


def _run_copy(state):
    page = state["case"]["page_size"]
    if own:
        _ops().copy_pages(state["pool"], state["src"], state["dst"], state["rows"], page)
        return state["pool"]
    pool = state["pool"]
    flat = pool.view(-1, *pool.shape[-2:])
    t = torch.arange(page, device=pool.device)
    moved = (t < state["rows"][:, None])[..., None]
    src, dst = (s[:, None] * page + t for s in (state["src"], state["dst"]))
    flat[:, dst] = torch.where(moved, flat[:, src], flat[:, dst])
    return pool


# ------------------------------------------------------------------------------------------------------- 64-bit values

def exact(case, seed):
    """The copied pool; out and lse of every layer.  Tables are whole numbers."""
    if case["kind"] == "tables":
        return None
    state = prepare(case, seed)
    if case["kind"] == "copy":
        pages = state["pool"].double().unflatten(-2, (case["pool_pages"], case["page_size"]))
        for src, dst, n in zip(*(state[name].tolist() for name in ("src", "dst", "rows"))):
            pages[..., dst, :n, :] = pages[..., src, :n, :].clone()
        return pages.flatten(-3, -2)
    page, group = case["page_size"], case["q_heads"] // case["cached_heads"]
    lines = state["table"].cpu()
    where, positions = state["batch_idx"].tolist(), state["pos"].tolist()
    result = []
    for layer in range(case["layers"]):
        q = state["q"][layer]
        out = torch.zeros(q.shape, dtype=torch.float64, device=DEVICE)
        lse = torch.full(q.shape[:3], -math.inf, dtype=torch.float64, device=DEVICE)
        for b, slot in enumerate(where):
            length = max(positions[b]) + 1
            if length <= 0:
                continue
            ids = lines[slot, :-(-length // page)].tolist()
            k, v = (torch.cat([state["pool"][layer, i][:, p * page:(p + 1) * page] for p in ids], 1)[:, :length].double()
                    for i in range(2))
            k, v = (x.repeat_interleave(group, 0) for x in (k, v))  # one a query head
            scores = torch.bmm(q[b].double(), k.mT.contiguous()) / math.sqrt(case["head_dim"])
            for j, p in enumerate(positions[b]):
                if p < 0:
                    continue
                row = scores[:, j, :p + 1]
                lse[b, :, j] = torch.logsumexp(row, 1)
                out[b, :, j] = torch.bmm(torch.softmax(row, 1)[:, None], v[:, :p + 1])[:, 0]
        if state["sinks"] is not None:
            out *= torch.sigmoid(lse - state["sinks"].double()[:, None])[..., None]
        result += [out, lse]
    return result
