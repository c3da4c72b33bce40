"""The plan of an attention over shared prefixes: every key of every row once, partial results in rows of their own.

Reads the plan's memory as the kernels do (csrc/shared_decode.hip: Header, Sequence, tokens, place, Share, Tile)."""

import random

import numpy as np
import pytest
import torch

from falcon_perception_amd import ops

pytestmark = pytest.mark.gpu
UNIT, ROWS, TOKEN = 64, 64, 20


def make(seed, B, S, max_batch, room):
    r = random.Random(seed)
    slots = [r.randrange(1, max_batch) if r.random() < 0.95 else r.choice([-1, max_batch]) for _ in range(B)]
    groups = r.choice([1, 2, 5, 20])
    ids = [r.choice([0, *range(1, groups + 1)]) for _ in range(max_batch)]
    lens = [r.randrange(0, room) if r.random() < 0.3 else 64 * (ids[i] + 1) * r.choice([1, 8]) for i in range(max_batch)]
    pos = [[r.randrange(-1, room) if r.random() < 0.9 else -1 for _ in range(S)] for _ in range(B)]
    return slots, ids, lens, pos


@pytest.mark.parametrize("B,S,Hq,Hc,room", [(1, 1, 8, 8, 300), (3, 1, 8, 4, 5000), (64, 1, 16, 8, 4000), (200, 1, 32, 4, 9000), (300, 1, 64, 8, 700),
                                            (1536, 1, 2, 2, 400), (40, 24, 16, 8, 3000), (9, 100, 8, 1, 2000), (2, 1000, 6, 3, 1500),
                                            (700, 2, 5, 5, 900), (130, 1, 16, 2, 20000)])
@pytest.mark.parametrize("seed", [1, 2, 3])
def test_every_key_once(seed, B, S, Hq, Hc, room):
    G, max_batch = Hq // Hc, 50 if seed == 1 else 2000
    slots, ids, lens, pos = make(seed, B, S, max_batch, room)
    dev = lambda x, t: torch.tensor(x, dtype=t, device="cuda")
    shape = dict(q_heads=Hq, cached_heads=Hc, head_dim=64)
    plan = ops.shared_decode_plan(dev(slots, torch.int64), dev(pos, torch.int32), dev(ids, torch.int32), dev(lens, torch.int32),
                                  max_context=room, **shape).cpu().numpy().view(np.int32)
    part_rows = ops.shared_decode_workspace_bytes(B, S, **shape) // (Hc * 66 * 4)
    n_most = max(1, 2 * torch.cuda.get_device_properties(0).multi_processor_count // Hc)
    lists = (B * S + 3) // 4 * 4
    at = [16, 16 + 16 * B, 16 + 16 * B + lists, 16 + 16 * B + 2 * lists, 16 + 16 * B + 2 * lists + 16 * n_most]
    head, seqs, tokens = plan[:16], plan[16:at[1]].reshape(B, 16), plan[at[1]:at[2]]
    n_wg, n_tiles = int(head[7]), int(head[8])
    assert 0 <= n_wg <= n_most and at[4] + 12 * n_tiles <= plan.size
    shares = plan[at[3]:at[4]].reshape(-1, 16)[:n_wg]
    tiles = plan[at[4]:at[4] + 12 * n_tiles].reshape(-1, 12)

    # what the workgroups do, as the kernel walks it
    done = {}  # tile -> [(piece, first unit, end)]
    for w in range(n_wg):
        tile, offset, left, piece = (int(x) for x in shares[w][:4])
        assert left > 0
        first = shares[w][4:]
        assert (first == tiles[tile]).all()
        while True:
            t = tiles[tile]
            units = -(-int(t[5] - t[4]) // UNIT)
            lo, hi = max(0, offset - int(t[9])), min(units, offset + left - int(t[9]))
            left -= int(t[9]) + units - offset
            offset = 0
            if hi > lo:
                done.setdefault(tile, []).append((piece, lo, hi))
            piece, tile = 0, int(t[11])
            if left <= 0 or tile >= n_tiles:
                break
    used = []
    for i, t in enumerate(tiles):
        pieces = sorted(done[i])
        units = -(-int(t[5] - t[4]) // UNIT)
        assert [p for p, _, _ in pieces] == list(range(int(t[6])))
        assert pieces[0][1] == 0 and pieces[-1][2] == units and all(a[2] == b[1] for a, b in zip(pieces, pieces[1:]))
        assert 0 < t[3] <= ROWS
        used.append((int(t[7]), int(t[7] + t[6] * t[3])))
    used.sort()
    assert all(a[1] <= b[0] for a, b in zip(used, used[1:]))
    assert not used or (used[0][0] >= 0 and used[-1][1] <= part_rows)

    # every row has the keys it sees: those of its group's tile and its own
    rows = {}
    for i, t in enumerate(tiles):
        for r in range(int(t[3])):
            x = int(t[2]) + r
            token = int(tokens[int(t[1]) + x // G])
            rows.setdefault((token >> TOKEN, token & ((1 << TOKEN) - 1), x % G), []).append((int(t[4]), int(t[5]), int(t[0]), int(t[8])))
    for b in range(B):
        valid = 0 <= slots[b] < max_batch
        keys = max(min(p + 1, room) for p in pos[b]) if valid else 0
        assert seqs[b][0] == (slots[b] if valid else -1) and seqs[b][1] == max(keys, 0)
        for j in range(S):
            if not valid or pos[b][j] < 0:
                assert (b, j, 0) not in rows
                continue
            for g in range(G):
                got = sorted(rows[b, j, g])
                assert got[0][0] == 0 and got[-1][1] >= min(pos[b][j] + 1, room)
                assert len(got) == 1 or (len(got) == 2 and got[0][1] == got[1][0] and got[0][3] and not got[1][3])
                for lo, hi, slot, shared in got:
                    if shared:  # through the row of a sequence with the same id, within what both say they share
                        assert ids[slot] == ids[slots[b]] > 0 and hi <= lens[slots[b]] and hi % UNIT == 0
                    else:
                        assert slot == slots[b]
