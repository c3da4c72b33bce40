"""Which sequences of a step share, how many keys, and that the work is cut evenly: the plan read back, and attention over such groups.

Reads the plan's memory as the kernels do (csrc/shared_decode.hip: Header, Sequence, tokens, place, Share, Tile)."""

import random

import numpy as np
import pytest
import torch

from falcon_perception_amd import ops
from tests.shared_cases import SharedBatch
from tests.test_gpu_prefix_sharing import Server

pytestmark = pytest.mark.gpu
UNIT, ROWS, TOKEN = 64, 64, 20


def plan_of(slots, ids, lens, pos, Hq, Hc, room):
    """(workgroups there are, units of each share, tiles as rows of 12, rows of each tile as {(sequence, token, head)})"""
    dev = lambda x, t: torch.tensor(x, dtype=t, device="cuda")
    B, S = len(pos), len(pos[0])
    plan = ops.shared_decode_plan(dev(slots, torch.int64), dev(pos, torch.int32), dev(ids, torch.int32), dev(lens, torch.int32), q_heads=Hq,
                                  cached_heads=Hc, head_dim=64, max_context=room).cpu().numpy().view(np.int32)
    most = max(1, 2 * torch.cuda.get_device_properties(0).multi_processor_count // Hc)
    lists = (B * S + 3) // 4 * 4
    at = [16, 16 + 16 * B, 16 + 16 * B + 2 * lists, 16 + 16 * B + 2 * lists + 16 * most]
    n_wg, n_tiles = int(plan[7]), int(plan[8])
    tokens, shares = plan[at[1]:at[1] + lists], plan[at[2]:at[3]].reshape(-1, 16)[:n_wg]
    tiles = plan[at[3]:at[3] + 12 * n_tiles].reshape(-1, 12)
    rows = []
    for t in tiles:
        at_row = [int(t[2]) + r for r in range(int(t[3]))]
        named = [int(tokens[int(t[1]) + x // (Hq // Hc)]) for x in at_row]
        rows.append({(n >> TOKEN, n & ((1 << TOKEN) - 1), x % (Hq // Hc)) for n, x in zip(named, at_row)})
    return most, [int(x) for x in shares[:, 2]], tiles, rows


def groups_of(slots, ids, lens, pos, max_batch, room):
    """{sequence: (leader, shared keys)} of the sequences that share, from the definition, with as many keys spared as there can be."""
    keys = [max([min(p + 1, room) for p in row if p >= 0], default=0) if 0 <= s < max_batch else 0 for s, row in zip(slots, pos)]
    out = {}
    for id_ in {ids[s] for s, k in zip(slots, keys) if k > 0 and ids[s] > 0}:
        members = [b for b, (s, k) in enumerate(zip(slots, keys)) if k > 0 and ids[s] == id_ and lens[s] >= UNIT]
        if len(members) < 2:
            continue
        longest = max(keys[b] for b in members)
        usable = {b: min(max(lens[slots[b]], 0), longest) // UNIT for b in members}
        spared = lambda u: u * (sum(x >= u for x in usable.values()) - 1)
        best = max(spared(u) for u in usable.values())
        cut = min(u for u in usable.values() if spared(u) == best)
        if len(members) > 2:
            members = [b for b in members if usable[b] >= cut]
        shared = min(min(max(lens[slots[b]], 0) for b in members), max(keys[b] for b in members)) // UNIT * UNIT
        if len(members) > 1 and shared > 0:
            out |= {b: (members[0], shared) for b in members}
    return out, keys


def check(slots, ids, lens, pos, Hq, Hc, room):
    G, max_batch = Hq // Hc, len(ids)
    most, units, tiles, rows = plan_of(slots, ids, lens, pos, Hq, Hc, room)
    groups, keys = groups_of(slots, ids, lens, pos, max_batch, room)
    got = {}
    for t, named in zip(tiles, rows):
        if t[8]:
            for b, _, _ in named:
                got[b] = (int(t[0]), int(t[4]), int(t[5]))
    assert got == {b: (slots[lead], 0, shared) for b, (lead, shared) in groups.items()}
    # All keys of all tiles, and what a tile costs beside them, are cut into shares of one length, but for the last of every axis: the
    # prefixes of several tiles have one for each number of tiles, everything else has one.
    cost = lambda t: int(t[9]) + -(-int(t[5] - t[4]) // UNIT)
    all_units = sum(cost(t) for t in tiles)
    shortest = max(3, -(-all_units // most))
    assert sum(units) == all_units and len(units) <= most
    members = {}
    for b, (lead, _) in groups.items():
        members.setdefault(lead, []).append(b)
    n_tiles = lambda group: -(-sum(p >= 0 for b in group for p in pos[b]) * G // ROWS)
    kinds = {n for n in map(n_tiles, members.values()) if n > 1}
    if not kinds:
        assert all(u == shortest for u in units[:-1]) and len(units) == -(-all_units // shortest)
    elif units:
        length = max(units)
        assert length <= max(3 * shortest + 1, shortest)
        assert sum(u < length for u in units) <= sum(kinds) + 1
    return groups


def test_one_short_member_does_not_keep_the_others_from_sharing():
    slots, B = list(range(1, 9)), 8
    ids, lens = [0] + [5] * 8, [0] + [4000] * 4 + [63] + [4000] * 3
    pos = [[4000 + 9 * b] for b in range(B)]
    groups = check(slots, ids, lens, pos, 16, 8, 8192)
    assert set(groups) == {0, 1, 2, 3, 5, 6, 7} and set(groups.values()) == {(0, 3968)}
    # the short one first, which would have led; two lengths that spare the same: the more members
    lens = [0, 63] + [4000] * 3 + [640] * 4
    groups = check(slots, ids, lens, pos, 16, 8, 8192)
    assert set(groups) == {1, 2, 3} and set(groups.values()) == {(1, 3968)}
    lens = [0] + [128] * 3 + [640] + [256] * 4  # 2 * 7 = 14, 4 * 4 = 16, 10 * 0
    assert set(check(slots, ids, lens, pos, 16, 8, 8192).values()) == {(3, 256)}
    lens = [0] + [64] * 5 + [192] * 3  # 1 * 7, 3 * 2
    assert set(check(slots, ids, lens, pos, 16, 8, 8192).values()) == {(0, 64)}
    lens = [0] + [64] * 3 + [128] * 5  # 1 * 7, 2 * 4
    assert set(check(slots, ids, lens, pos, 16, 8, 8192).values()) == {(3, 128)}
    lens = [0, 4000, 100, 0, 0, 0, 0, 0, 0]  # two share what the shorter has
    assert check(slots, ids, lens, pos, 16, 8, 8192) == {0: (0, 64), 1: (0, 64)}


def test_lengths_beyond_the_keys_count_as_far_as_the_keys():
    ids, lens = [0] + [5] * 6, [0, 2 ** 31 - 1, 700, 700, 2 ** 31 - 1, 650, -5]
    pos = [[640 + b] for b in range(6)]
    groups = check(list(range(1, 7)), ids, lens, pos, 8, 8, 4096)
    assert set(groups) == {0, 1, 2, 3, 4} and set(groups.values()) == {(0, 640)}


@pytest.mark.parametrize("B,S,Hq,Hc,room", [(2, 1, 8, 8, 300), (3, 1, 8, 4, 5000), (16, 1, 16, 8, 1300), (30, 1, 16, 8, 9000), (64, 1, 16, 8, 4000),
                                            (200, 1, 32, 4, 9000), (520, 1, 64, 8, 2500), (1100, 1, 2, 2, 1500), (1536, 1, 8, 1, 900),
                                            (40, 24, 16, 8, 3000), (9, 100, 8, 1, 2000), (700, 2, 5, 5, 900)])
@pytest.mark.parametrize("seed", range(4))
def test_groups_and_their_cut(seed, B, S, Hq, Hc, room):
    """Lengths of one group: all alike, two of them, any."""
    r = random.Random(1000 * seed + B)
    max_batch = B + 40
    slots = r.sample(range(1, max_batch), B) if seed % 2 else [r.randrange(1, max_batch) for _ in range(B)]
    n_groups = r.choice([1, 3, 12])
    ids = [r.randrange(0, n_groups + 1) for _ in range(max_batch)]
    own = [r.randrange(64, room) for _ in range(n_groups + 1)]
    lens = [own[i] if seed < 2 else r.choice([own[i], own[i] // 3]) if seed == 2 else r.randrange(0, room) for i in ids]
    pos = [[r.randrange(0, room) if r.random() < 0.2 else r.randrange(max(0, lens[s] - 1), room) for _ in range(S)] for s in slots]
    if seed:
        pos = [[p if r.random() < 0.9 else -1 for p in row] for row in pos]
    check(slots, ids, lens, pos, Hq, Hc, room)


@pytest.mark.parametrize("dtype,D,Hq,Hc,P", [(torch.bfloat16, 128, 8, 4, 32), (torch.float16, 64, 8, 1, 48), (torch.float32, 64, 4, 4, 16)])
@pytest.mark.parametrize("tokens", [1, 5])
def test_attention_over_groups_of_several_lengths(dtype, D, Hq, Hc, P, tokens):
    """What slots are said to share is less than what they do, and different for each."""
    sequences = [(0, 30 + 3 * b, tokens) for b in range(7)] + [(1, 9 + b, tokens) for b in range(4)] + [(-1, 70, 1)]
    case = SharedBatch(61, [700, 333], sequences, Hq=Hq, Hc=Hc, D=D, P=P, dtype=dtype, S=tokens).on()
    slots = case.batch_idx.tolist()
    for lens in ([700] * 6 + [20] + [333] * 4, [20] + [700] * 6 + [333, 70, 333, 0], [64, 128, 192, 256, 320, 640, 700, 333, 333, 64, 64],
                 [64] * 6 + [700, 1, 2, 3, 4], [700, 640, 700, 640, 0, -7, 700, 333, 128, 128, 128]):
        for s, n in zip(slots, lens):
            case.lens_d[s] = n
        got = case.call(ops)
        case.check(got)
        again = case.call(ops)
        assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


def test_questions_about_pictures_behind_one_prompt_decode():
    """Forks of forks that have a line of their own, beside the lines they came from."""
    s = Server(n_pages=400, slots=40)
    system = s.picture(70)
    pictures = s.fork(system, 70, 3)
    s.extend(pictures, [200, 130, 150])
    asked = [s.fork(p, s.length(p), 3) for p in pictures[:2]] + [s.fork(pictures[2], 71, 2)]
    ids = s.cache.prefix_ids.tolist()
    assert len({ids[x] for x in (system, *pictures)}) == 3 and ids[system] == ids[pictures[2]] == ids[asked[2][0]]
    everyone = [x for forks in asked for x in forks]
    s.extend(everyone, [1 + 2 * i for i in range(len(everyone))])
    for batch in (everyone, [system, *everyone, *pictures], [asked[0][1], asked[1][0], system]):
        s.decode(batch)
    s.forget(pictures[0])
    s.forget(system)
    s.decode(everyone)
    s.check_pool()


@pytest.mark.parametrize("seed", range(6))
def test_a_server_with_forks_of_forks(seed):
    """Any order of pictures, forks, prompts, decode steps and releases; every step against float64, the pool at the end."""
    r = random.Random(seed)
    s = Server(n_pages=300, slots=26, P=r.choice([16, 32, 48]), layers=2, dtype=r.choice([torch.bfloat16, torch.float16, torch.float32]), seed=seed)
    room = 16 * s.P - 8
    for _ in range(40):
        live, what = list(s.keys), r.random()
        pages = s.cache.num_free_pages
        if not live or (what < 0.12 and len(live) < 20 and pages > 40):
            s.picture(r.randrange(1, 2 * room // 3))
        elif what < 0.45 and len(live) < 20 and pages > 40:
            parent = r.choice(live)
            n = s.length(parent) - (r.randrange(s.length(parent)) if r.random() < 0.4 else 0)
            s.fork(parent, n, r.randrange(1, min(5, 25 - len(live))))
        elif what < 0.6 and pages > 60:
            some = [x for x in r.sample(live, min(len(live), 4)) if s.length(x) < room - 30]
            if some:
                s.extend(some, [r.randrange(0, 30) for _ in some], row_multiple=r.choice([1, 8]))
        elif what < 0.85:
            batch = [x for x in live if s.length(x) < room]
            r.shuffle(batch)
            if batch and pages >= len(batch):
                s.decode(batch[:r.randrange(1, len(batch) + 1)])
        else:
            s.forget(r.choice(live))
    s.check_pool()
    for x in list(s.keys):
        s.forget(x)
    assert not s.cache._page_slots and not s.cache._prefixes and not s.cache.prefix_ids.any()
    assert sorted(s.cache.free_pages) == list(range(1, 300))
