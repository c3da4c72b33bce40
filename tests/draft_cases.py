"""Steps of drafted tokens: trees, decisions and moved rows by plain Python, and a batch of trees over a paged pool."""

from __future__ import annotations

import math

import numpy as np
import torch

from tests.shared_cases import HALF_STEP, SharedBatch


def ancestors(parents):
    """Per token the set of tokens it sees, None where there is no token."""
    seen = []
    for j, p in enumerate(parents):
        if p == -1:
            seen.append({j})
        elif 0 <= p < j and seen[p] is not None:
            seen.append(seen[p] | {j})
        else:
            seen.append(None)
    return seen


def random_tree(gen, n, reach):
    """Parents of n tokens, each within `reach` rows of its token."""
    draw = torch.randint(0, 1 << 30, (max(n, 1),), generator=gen).tolist()
    return [-1 if j == 0 else max(0, j - 1 - draw[j] % reach) for j in range(n)]


def tree_tensors(trees, S, cached):
    """What `draft_tree` has to return, for lists of parents."""
    B = len(trees)
    masks = torch.zeros((B, S), dtype=torch.int64)
    input_pos, rope_pos = torch.full((B, S), -1, dtype=torch.int32), torch.zeros((B, S), dtype=torch.int32)
    for b, tree in enumerate(trees):
        if cached[b] < 0 or cached[b] > 2 ** 31 - 65:
            continue
        for j, seen in enumerate(ancestors(tree)):
            if seen is not None:
                bits = sum(1 << i for i in seen)
                masks[b, j] = bits - (1 << 64) if bits >> 63 else bits
                input_pos[b, j] = cached[b] + j
                rope_pos[b, j] = cached[b] + len(seen) - 1
    return masks, input_pos, rope_pos


class DraftBatch(SharedBatch):
    """`sequences`: per sequence (group or -1, cached keys behind the prefix, parents of its tokens)."""

    def __init__(self, seed, prefixes, sequences, **kw):
        self.trees = [list(t) for _, _, t in sequences]
        super().__init__(seed, prefixes, [(g, n + len(t), len(t)) for g, n, t in sequences], **kw)
        self.cached = torch.tensor([L - len(t) for L, t in zip(self.lengths, self.trees)], dtype=torch.int32)
        self.parents = torch.full((self.B, self.S), -2, dtype=torch.int32)
        for b, t in enumerate(self.trees):
            self.parents[b, :len(t)] = torch.tensor(t, dtype=torch.int32)
        self.masks, self.pos, self.rope = tree_tensors(self.trees, self.S, self.cached.tolist())

    def on(self, device="cuda"):
        super().on(device)
        for name in ("parents", "cached", "masks"):
            setattr(self, name + "_d", getattr(self, name).to(device))
        return self

    def call(self, ops, share=True, **kw):
        tree = kw.pop("tree", None) or ops.DraftTree(self.masks_d, self.pos_d, self.pos_d)
        if share:
            kw.update(prefix_ids=self.ids_d, prefix_lens=self.lens_d)
        return ops.paged_decode_tree(kw.pop("q", self.q_d), self.pool_d[0], self.pool_d[1], self.table_d, self.batch_idx_d, tree, self.P,
                                     kw.pop("max_context", self.columns * self.P), **kw)

    def seen(self, b, j, max_context=None):
        """Positions that token j of sequence b sees."""
        pos, mask = int(self.pos[b, j]), int(self.masks[b, j])
        if pos < 0:
            return []
        base = pos - j
        keys = list(range(base)) + [base + i for i in range(j + 1) if mask >> i & 1]
        return [t for t in keys if max_context is None or t < max_context]

    def expect(self, sinks=None, scale=None, pos=None, max_context=None):
        """(out, lse) in float64 and how far a result in the type may be off (the terms are those of SharedBatch.expect)."""
        assert pos is None
        u, scale = HALF_STEP[self.dtype], self.D ** -0.5 if scale is None else scale
        G = self.Hq // self.Hc
        out = np.zeros((self.B, self.Hq, self.S, self.D))
        lse = np.full((self.B, self.Hq, self.S), -np.inf)
        o_tol, l_tol = np.zeros_like(out), np.zeros_like(lse)
        q = self.q.double().numpy()
        for b in range(self.B):
            k, v = (x.double().numpy() for x in self.keys[b])
            for j in range(self.S):
                keys = self.seen(b, j, max_context)
                n = len(keys)
                if n == 0:
                    continue
                for hc in range(self.Hc):
                    kk, vv = k[hc, keys], v[hc, keys]
                    hs = slice(hc * G, hc * G + G)
                    x = q[b, hs, j] @ kk.T * scale
                    c = (np.abs(q[b, hs, j]) @ np.abs(kk).T * abs(scale)).max(1)
                    top = x.max(1)
                    w = np.exp(x - top[:, None])
                    den = w.sum(1)
                    out[b, hs, j] = w @ vv / den[:, None]
                    lse[b, hs, j] = top + np.log(den)
                    d = (self.D + 2) * 2.0 ** -24 * c + 2 * c * 2.0 ** -22 + 2.0 ** -21
                    sums = (n + 64) * 2.0 ** -24
                    mag = w @ np.abs(vv) / den[:, None]
                    rounding = 0.0 if self.dtype == torch.float32 else 2 * u * u + (n * 2.0 ** -31 / den if self.dtype == torch.float16 else 0.0)
                    o_tol[b, hs, j] = mag * (2 * d + 2 * sums + rounding)[:, None] * 1.01 + u * np.abs(out[b, hs, j]) + 1e-30
                    l_tol[b, hs, j] = d + sums + 2.0 ** -22 * (1 + np.abs(lse[b, hs, j]))
        if sinks is not None:
            gate = 1.0 / (1.0 + np.exp(sinks.double().numpy()[None, :, None] - lse))
            o_tol = (o_tol - u * np.abs(out)) * gate[..., None] + u * np.abs(out) * gate[..., None] + np.abs(out) * gate[..., None] * (l_tol[..., None] + 2.0 ** -21)
            out = out * gate[..., None]
        if self.dtype == torch.float16:
            o_tol = o_tol + 2.0 ** -24  # results below the normal numbers
        return out, lse, o_tol, l_tol

    def check(self, got, sinks=None, scale=None, max_context=None):
        want = self.expect(sinks, scale, max_context=max_context)
        out, lse, o_tol, l_tol = want
        o, l = got[0].double().cpu().numpy(), got[1].double().cpu().numpy()
        empty = np.isneginf(lse)
        assert np.array_equal(np.isneginf(l), empty)
        assert (o[empty] == 0).all()
        assert np.isfinite(o).all()
        off = np.abs(o - out) - o_tol
        assert off.max() <= 0, f"out is off by {off.max():.3g} more than it may at {np.unravel_index(off.argmax(), off.shape)}"
        off = np.where(empty, -1.0, np.abs(np.where(empty, 0, l) - np.where(empty, 0, lse)) - l_tol)
        assert off.max() <= 0, f"lse is off by {off.max():.3g} more than it may at {np.unravel_index(off.argmax(), off.shape)}"


def verify(logits, tokens, parents, uniforms, temperatures=None, probs=None):
    """One sequence's decision in float64: (accepted rows, answer, (log p, weight of the row's other tokens than its largest) of each) and
    how near the nearest border lay, relative to the whole.

    logits [S, V] as float64, probs likewise or None."""
    S, V = logits.shape
    near = math.inf
    heat = 1.0 if temperatures is None else float(temperatures)
    greedy = not heat > 0
    heat = 1.0 if greedy else heat
    if parents[0] != -1:
        return None, [], [], near
    node, rows, answer, says = 0, [], [], []
    while True:
        x = np.where(np.isnan(logits[node]), -np.inf, logits[node])
        top = x.max()
        if top == -np.inf:
            w = np.zeros(V)
        elif top == np.inf:
            w = (x == np.inf).astype(float)
        else:
            with np.errstate(invalid="ignore", over="ignore"):
                w = np.exp((x - top) / heat)
            w[x == -np.inf] = 0.0
        z = w.sum()
        best = int(np.argmax(x == top)) if top > -np.inf else -1
        with np.errstate(divide="ignore", invalid="ignore"):
            log_p = np.log(w / z) if z > 0 else np.full(V, -np.inf)
            if top < np.inf and z > 0:
                log_p = (x - top) / heat - np.log(z)
        others = (z - (w == 1).sum()) / z if z > 0 else 0.0
        left, stands, tested = w.copy(), None, False
        for j in [j for j in range(1, S) if parents[j] == node]:
            name, known = int(tokens[j]), 0 <= tokens[j] < V
            if greedy:
                takes = known and name == best
            elif probs is None:
                takes = known and uniforms[j] * left.sum() < left[name]
                if known and z > 0:
                    near = min(near, abs(uniforms[j] * left.sum() - left[name]) / z)
            else:
                takes = known and uniforms[j] * probs[node, name] * z < w[name]
                if known and z > 0:
                    near = min(near, abs(uniforms[j] * probs[node, name] * z - w[name]) / z)
            if takes:
                stands = j
                break
            tested = True
            if probs is None and known:
                left[name] = 0.0
            if probs is not None:
                break
        if stands is not None:
            rows.append(stands)
            answer.append(int(tokens[stands]))
            says.append((log_p[int(tokens[stands])], others))
            node = stands
            continue
        if greedy:
            name = best
        else:
            if probs is not None and tested and z > 0:
                rest = np.maximum(w / z - probs[node], 0.0)
                left = rest if rest.sum() > 0 else w
            sums = np.cumsum(left)
            name = -1
            if sums[-1] > 0:
                goal = max(float(uniforms[0]), 0.0) * sums[-1]
                name = min(int(np.searchsorted(sums, goal, side="right")), int(np.nonzero(left)[0][-1]))
                near = min(near, np.abs(sums[:-1][left[:-1] > 0] - goal).min(initial=np.inf) / sums[-1])
        answer.append(name)
        says.append((log_p[name] if name >= 0 else 0.0, others))
        return rows, answer, says, near


def sum_bounds(V):
    """How far the logarithm of a row's sum may be off, in parts of what its smaller logits weigh, and in all.

    The sum's weights are in 32 bits.  A weight 2^-p is off by 2.5 p 2^-24 ln 2 (difference, product and rate rounded) and 2^-23 (the
    exponential); weights of 2^-p are V 2^-p of the whole at most, so that p is log2 V where it matters, 16 of 65536 tokens.  Sums of 8 are off by
    3 * 2^-24, the largest weight and all, and that by 2^-22 where a thread weighs by a logit with up to 2^20 to spare."""
    return 2.0 ** -23 + 2.5 * math.log2(max(V, 2)) * math.log(2) * 2.0 ** -24, 3 * 2.0 ** -24 + 2.0 ** -22


def same_answers(one, other, V):
    """Whether two calls on the same logits, cut differently, decide alike; logprobs are within what each may be off by."""
    for x, y in zip(one[:3], other[:3]):
        assert torch.equal(x, y)
    assert torch.allclose(one[3], other[3], rtol=2.0 ** -23, atol=2 * sum(sum_bounds(V)))


def check_verified(got, logits, tokens, parents, uniforms, temperatures=None, probs=None):
    """A `VerifiedDrafts` against `verify`, decision by decision.  The decisions of two float64 computations can differ where a border
    is nearer than their sums are exact (weights to 2^-50, sums over V terms): such inputs are not compared, and there are hardly any."""
    accepted, path, answer, logprobs = (t.cpu() for t in got)
    B, S, V = logits.shape
    skipped = 0
    for b in range(B):
        x = logits[b].double().cpu().numpy()
        q = None if probs is None else probs[b].double().cpu().numpy()
        rows, words, says, near = verify(x, tokens[b].tolist(), parents[b].tolist(), uniforms[b].double().tolist(),
                                         None if temperatures is None else temperatures[b].item(), q)
        if near < V * 2.0 ** -50:
            skipped += 1
            continue
        if rows is None:
            assert accepted[b] == 0 and (path[b] == -1).all() and (answer[b] == -1).all() and (logprobs[b] == 0).all()
            continue
        pad = lambda line, empty: line + [empty] * (S - len(line))
        assert accepted[b] == len(rows), (b, accepted[b], rows)
        assert path[b].tolist() == pad([0] + rows, -1), (b, path[b], rows)
        assert answer[b].tolist() == pad(words, -1), (b, answer[b], words)
        want, others = np.array(pad(says, (0.0, 0.0))).T
        off = np.abs(logprobs[b].double().numpy() - want)
        relative, whole = sum_bounds(V)
        assert (off <= np.abs(want) * 2.0 ** -24 + others * relative + whole + V * 2.0 ** -49).all(), (b, off.max())
    assert skipped <= B // 16
