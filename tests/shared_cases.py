"""Batches whose sequences share a prefix: a pool, its tables and the float64 values of the attention over them.

The pool is NaN wherever no sequence has a key: whatever a kernel reads there must not reach a result.
"""

from __future__ import annotations

import numpy as np
import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


class SharedBatch:
    """`sequences`: per sequence (group or -1, keys behind the prefix, query tokens).  `prefixes`: keys of each group's prefix."""

    def __init__(self, seed, prefixes, sequences, *, Hq, Hc, D, P, dtype, S=None, spread=1.0, idle_slots=2, columns=None):
        gen = torch.Generator().manual_seed(seed)
        self.Hq, self.Hc, self.D, self.P, self.dtype = Hq, Hc, D, P, dtype
        B = len(sequences)
        self.B, self.S = B, S or max([1] + [n for _, _, n in sequences])
        blocks = lambda n: -(-n // P)
        whole = [n // P for n in prefixes]
        lengths = [(prefixes[g] if g >= 0 else 0) + behind for g, behind, _ in sequences]
        wanted = [blocks(L) - (whole[g] if g >= 0 else 0) for L, (g, _, _) in zip(lengths, sequences)]
        n_pages = 1 + sum(whole) + sum(wanted) + 2
        free = (torch.randperm(n_pages - 1, generator=gen) + 1).tolist()
        take = lambda n: [free.pop() for _ in range(n)]
        lines = [take(n) for n in whole]
        self.columns = columns or max([1] + [blocks(L) for L in lengths]) + 1
        self.max_batch = B + 1 + idle_slots
        slots = (torch.randperm(self.max_batch - 1, generator=gen) + 1).tolist()[:B]
        table = torch.full((self.max_batch, self.columns), -1, dtype=torch.int64)
        table[0] = 0
        self.ids = torch.zeros(self.max_batch, dtype=torch.int32)
        self.lens = torch.zeros(self.max_batch, dtype=torch.int32)
        self.pos = torch.full((B, self.S), -1, dtype=torch.int32)
        self.pool = torch.full((2, Hc, n_pages * P, D), float("nan"), dtype=dtype)
        self.n_pages = n_pages
        rnd = lambda *shape: (torch.randn(shape, generator=gen) * spread).to(dtype)
        shared = [(rnd(Hc, n, D), rnd(Hc, n, D)) for n in prefixes]
        self.keys = []  # per sequence: k, v [Hc, L, D]
        for b, (g, behind, n) in enumerate(sequences):
            s, L = slots[b], lengths[b]
            line = (lines[g] if g >= 0 else []) + take(wanted[b])
            table[s, :len(line)] = torch.tensor(line, dtype=torch.int64)
            k, v = rnd(Hc, behind, D), rnd(Hc, behind, D)
            if g >= 0:
                k, v = torch.cat([shared[g][0], k], 1), torch.cat([shared[g][1], v], 1)
                self.ids[s], self.lens[s] = 7 * g + 3, prefixes[g]
            at = torch.tensor([line[t // P] * P + t % P for t in range(L)], dtype=torch.int64)
            self.pool[0][:, at], self.pool[1][:, at] = k, v
            self.pos[b, :n] = torch.arange(L - n, L)
            self.keys.append((k, v))
        self.table = table
        self.batch_idx = torch.tensor(slots, dtype=torch.int64)
        self.q = rnd(B, Hq, self.S, D)
        self.lengths = lengths
        self.gen = gen

    def on(self, device="cuda"):
        for name in ("pool", "table", "ids", "lens", "pos", "batch_idx", "q"):
            setattr(self, name + "_d", getattr(self, name).to(device))
        return self

    def call(self, ops, **kw):
        kw.setdefault("max_context", self.columns * self.P)
        mc = kw.pop("max_context")
        return ops.paged_decode_shared(kw.pop("q", self.q_d), self.pool_d[0], self.pool_d[1], self.table_d, self.batch_idx_d,
                                       kw.pop("pos", self.pos_d), self.ids_d, self.lens_d, self.P, mc, **kw)

    def expect(self, sinks=None, scale=None, pos=None):
        """(out, lse) in float64 and how far a result in the type may be off, element by element.

        With u half a step of the type, n keys and c = scale * sum |q k| (natural units):
        a score is off by at most d = (D + 2) 2^-24 c (sums and the scale in fp32), its exponential by that, by the rounding of
        its argument (2^-23 of it, at most c * 2^-22) and 2^-22 of its own; the probabilities of the 16-bit types are sums of two
        numbers of the type, the second below 2u of the first and rounded by u of itself, so off by 2 u^2 (and in f16 by at
        most 2^-31 of the largest, where a part would vanish); sums over n keys, in parts that are joined, are off by
        (n + 64) 2^-24 of the sum of magnitudes.  The result is rounded once, also behind a sink gate."""
        u, scale = HALF_STEP[self.dtype], self.D ** -0.5 if scale is None else scale
        G = self.Hq // self.Hc
        pos = self.pos if pos is None else pos
        out = np.zeros((self.B, self.Hq, self.S, self.D))
        lse = np.full((self.B, self.Hq, self.S), -np.inf)
        o_tol, l_tol = np.zeros_like(out), np.zeros_like(lse)
        q = self.q.double().numpy()
        for b in range(self.B):
            k, v = (x.double().numpy() for x in self.keys[b])
            for j in range(self.S):
                n = int(pos[b, j]) + 1
                if n <= 0:
                    continue
                for h in range(self.Hq):
                    kk, vv = k[h // G, :n], v[h // G, :n]
                    x = kk @ q[b, h, j] * scale
                    c = (np.abs(kk) @ np.abs(q[b, h, j]) * abs(scale)).max()
                    top = x.max()
                    w = np.exp(x - top)
                    den = w.sum()
                    out[b, h, j] = w @ vv / den
                    lse[b, h, j] = top + np.log(den)
                    d = (self.D + 2) * 2.0 ** -24 * c + 2 * c * 2.0 ** -22 + 2.0 ** -21
                    sums = (n + 64) * 2.0 ** -24
                    mag = w @ np.abs(vv) / den
                    rounding = 0.0 if self.dtype == torch.float32 else 2 * u * u + (n * 2.0 ** -31 / den if self.dtype == torch.float16 else 0.0)
                    o_tol[b, h, j] = mag * (2 * d + 2 * sums + rounding) * 1.01 + u * np.abs(out[b, h, j]) + 1e-30
                    l_tol[b, h, j] = d + sums + 2.0 ** -22 * (1 + abs(lse[b, h, j]))
        if sinks is not None:
            gate = 1.0 / (1.0 + np.exp(sinks.double().numpy()[None, :, None] - lse))
            o_tol = (o_tol - u * np.abs(out)) * gate[..., None] + u * np.abs(out) * gate[..., None] + np.abs(out) * gate[..., None] * (l_tol[..., None] + 2.0 ** -21)
            out = out * gate[..., None]
        if self.dtype == torch.float16:
            o_tol = o_tol + 2.0 ** -24  # results below the normal numbers
        return out, lse, o_tol, l_tol

    def check(self, got, sinks=None, scale=None, pos=None):
        out, lse, o_tol, l_tol = self.expect(sinks, scale, pos)
        o, l = got[0].double().cpu().numpy(), got[1].double().cpu().numpy()
        empty = np.isneginf(lse)
        assert np.array_equal(np.isneginf(l), empty)
        assert (o[empty] == 0).all()
        assert np.isfinite(o).all()
        off = np.abs(o - out) - o_tol
        assert off.max() <= 0, f"out is off by {off.max():.3g} more than it may at {np.unravel_index(off.argmax(), off.shape)}"
        off = np.where(empty, -1.0, np.abs(np.where(empty, 0, l) - np.where(empty, 0, lse)) - l_tol)
        assert off.max() <= 0, f"lse is off by {off.max():.3g} more than it may at {np.unravel_index(off.argmax(), off.shape)}"
