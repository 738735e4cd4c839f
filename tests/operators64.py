"""64-bit references of the operators beside plain causal attention: attention with capped,
biased and range-masked scores, accumulated attention weights, eviction. Elementary float64
operations on the CPU; a key that a query does not see is left out by indexing, so nothing that
it holds can reach the result.
"""

from __future__ import annotations

import math

import torch

LOG2E = 1 / math.log(2)
HALF_STEP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}


def slots_of(table, n: int, bs: int) -> list[int]:
    return [int(table[p // bs]) * bs + p % bs for p in range(n)]


class Step:
    """A step's inputs, on the CPU: K/V pools, tables, contexts and query rows. Blocks are
    scattered; ``new`` queries per sequence, the last tokens of its context."""

    def __init__(self, dtype, nh, nkv, hd, bs, ctx, new, seed=0, spare=2, width=None):
        g = torch.Generator().manual_seed(seed)
        self.dtype, self.bs, self.nh, self.nkv, self.hd = dtype, bs, nh, nkv, hd
        self.ctx, self.new = list(ctx), list(new)
        need = [-(-n // bs) for n in ctx]
        blocks = sum(need) + spare
        order = torch.randperm(blocks, generator=g).tolist()
        width = width or max(1, max(need))
        self.tables = torch.zeros(len(ctx), width, dtype=torch.int32)
        for i, n in enumerate(need):
            self.tables[i, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
        shape = (blocks * bs, nkv, hd)
        self.k = torch.randn(shape, generator=g).to(dtype)
        self.v = torch.randn(shape, generator=g).to(dtype)
        self.q = torch.randn(sum(new), nh, hd, generator=g).to(dtype)
        self.cu = torch.tensor([0] + self.new).cumsum(0).to(torch.int32)
        self.context_lens = torch.tensor(self.ctx, dtype=torch.int32)

    def slots(self, i: int) -> list[int]:
        return slots_of(self.tables[i].tolist(), self.ctx[i], self.bs)

    def positions(self):
        """(sequence, position) of every query row."""
        return [(i, c - n + j) for i, (c, n) in enumerate(zip(self.ctx, self.new, strict=True))
                for j in range(n)]  # fmt: skip

    def causal(self) -> torch.Tensor:
        return torch.tensor([[0, p + 1] for _, p in self.positions()], dtype=torch.int32).view(-1, 2)


def scores64(s: Step, row: int, i: int, pos: int, lo: int, hi: int, softcap=None, slopes=None):
    """Scores [nh, hi - lo] of query row ``row`` (sequence i, position pos), natural units."""
    slots = s.slots(i)[lo:hi]
    g = s.nh // s.nkv
    k = s.k[slots].double().repeat_interleave(g, dim=1)  # [n, nh, hd]
    x = (k * s.q[row].double()).sum(-1).T / math.sqrt(s.hd)
    if softcap:
        x = softcap * torch.tanh(x / softcap)
    if slopes is not None:
        far = (pos - torch.arange(lo, hi)).abs().double()
        x = x - slopes.double()[:, None] * far
    return x


def bounds(s: Step, ranges):
    """Every query row's keys [lo, hi), cut to its context."""
    ranges = s.causal() if ranges is None else ranges
    out = []
    for (i, _), (lo, hi) in zip(s.positions(), ranges.tolist(), strict=True):
        lo, hi = max(lo, 0), min(hi, s.ctx[i])
        out.append((lo, hi) if lo < hi else (0, 0))
    return out


def attention64(s: Step, softcap=None, slopes=None, ranges=None):
    """(out [T, nh, hd], log2 normalisers [T, nh]) in float64."""
    out = torch.zeros(s.q.shape, dtype=torch.float64)
    lse = torch.full(s.q.shape[:2], -math.inf, dtype=torch.float64)
    g = s.nh // s.nkv
    spans = bounds(s, ranges)
    for row, (i, pos) in enumerate(s.positions()):
        lo, hi = spans[row]
        if lo >= hi:
            continue
        x = scores64(s, row, i, pos, lo, hi, softcap, slopes)
        lse[row] = torch.logsumexp(x, -1) * LOG2E
        p = torch.softmax(x, -1)
        v = s.v[s.slots(i)[lo:hi]].double().repeat_interleave(g, dim=1)  # [n, nh, hd]
        out[row] = (p.T[:, :, None] * v).sum(0)
    return out, lse


def weights64(s: Step, old, decay, lse, softcap=None, slopes=None, ranges=None, rows=None):
    """The accumulated weights after the step, in float64; lse [T, nh] as the call was given."""
    w = old.double().clone()
    spans = bounds(s, ranges)
    places = list(enumerate(s.positions()))
    for i, n in enumerate(s.ctx):
        r = i if rows is None else int(rows[i])
        if not 0 <= r < w.shape[0]:
            continue
        new = torch.zeros(n, dtype=torch.float64)
        for row, (j, pos) in places:
            lo, hi = spans[row]
            if j != i or lo >= hi:
                continue
            x = scores64(s, row, i, pos, lo, hi, softcap, slopes) * LOG2E
            y = lse[row].double()[:, None]
            new[lo:hi] += torch.where(y > -math.inf, torch.exp2(x - y), torch.zeros_like(x)).sum(0)
        w[r, :n] = (w[r, :n] * decay if decay else 0) + new
    return w


def score_error(s: Step, softcap=None, slopes=None) -> float:
    """A bound on a score's error in fp32: a dot product of hd terms and its scaling ((hd + 2)
    half steps of the terms' absolute sum), the cap (the 16-bit kernels' c2 - 2 c2 / (1 + e): e's
    and the reciprocal's step and the subtraction, 4 steps of c2; in fp32 its value's own, smaller),
    the bias and its addition (3 half steps of the largest distance's)."""
    u = 2.0**-24
    top = float(s.q.float().norm(dim=-1).max() * _finite(s.k).norm(dim=-1).max()) / math.sqrt(s.hd)
    e = (s.hd + 2) * u * top
    if softcap:
        e += 8 * u * softcap
    if slopes is not None:
        e += 3 * u * float(slopes.abs().max()) * max(s.ctx)
    return e


def _finite(x: torch.Tensor) -> torch.Tensor:
    return torch.nan_to_num(x.float(), nan=0.0, posinf=0.0, neginf=0.0)


def tolerance(s: Step, want: torch.Tensor, out_dtype, softcap=None, slopes=None, p16=False):
    """How far an output may be from ``want``: its rounding, weights off by the scores' error
    twice (in the numerator and the normaliser), fp32 sums over the context likewise, and with p16
    (the 16-bit prefill) weights rounded to fp16, 2^-11 of each in both; all against the largest
    |V|."""
    vmax = float(_finite(s.v).abs().max())
    n = max(max(s.ctx), 1)
    rel = 2 * (score_error(s, softcap, slopes) + (n + 4) * 2.0**-24) + (2 * 2.0**-11 if p16 else 0)
    return HALF_STEP[out_dtype] * want.abs() + rel * vmax


def evict64(k, v, w, tables, ctx, bs, keep, recent, rows=None):
    """(new lengths, k, v, w) after an eviction, pools [L, slots, nkv, hd], w [L, R, P]; a NaN
    weight counts as the smallest, ties go to the lowest position."""
    k, v, w = k.clone(), v.clone(), w.clone()
    lens = []
    blocks = k.shape[1] // bs
    for b, n in enumerate(ctx):
        n = min(max(n, 0), tables.shape[1] * bs)
        r = b if rows is None else int(rows[b])
        if not 0 <= r < w.shape[1]:
            lens.append(ctx[b])
            continue
        lens.append(min(n, keep))
        if n <= keep:
            continue
        row = tables[b].tolist()
        for layer in range(k.shape[0]):
            x = w[layer, r, :n].tolist()
            order = sorted(range(n - recent), key=lambda p: (math.isnan(x[p]), 0.0 if math.isnan(x[p]) else -x[p], p))
            kept = sorted(order[: keep - recent]) + list(range(n - recent, n))
            for pool in (k, v):
                old = pool[layer].clone()
                for i, p in enumerate(kept):
                    src, dst = row[p // bs], row[i // bs]
                    if 0 <= src < blocks and 0 <= dst < blocks:
                        pool[layer, dst * bs + i % bs] = old[src * bs + p % bs]
            w[layer, r, : len(kept)] = torch.tensor([x[p] for p in kept])
            w[layer, r, len(kept) : n] = 0.0
    return lens, k, v, w
