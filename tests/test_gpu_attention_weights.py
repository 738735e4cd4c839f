"""Accumulated attention weights against 64 bits, with the normalisers of the attention call."""

from __future__ import annotations

import math

import pytest
import torch
from operators64 import Step, attention64, score_error, weights64
from test_gpu_score_mods import BF16, FP16, FP32, cuda, how_of, slopes_of

from engine.kernels import paged_attention as pa

pytestmark = pytest.mark.gpu

SHAPES = [
    # dtype, heads, KV heads, head_dim, block size, (queries, context)
    (BF16, 32, 8, 128, 16, [(1, 300), (1, 1), (1, 64), (1, 129)]),
    (FP16, 8, 2, 64, 16, [(1, 500), (1, 17)]),
    (FP32, 8, 2, 64, 16, [(1, 90), (3, 40)]),
    (BF16, 8, 2, 128, 16, [(20, 150), (64, 70), (1, 5)]),
    (FP16, 6, 3, 128, 12, [(5, 100), (2, 11)]),  # 3 KV heads over 2 waves
    (BF16, 16, 16, 64, 16, [(4, 130)]),  # more KV heads than waves
    (BF16, 8, 1, 256, 16, [(9, 77)]),
    (FP32, 4, 4, 128, 5, [(7, 33)]),
    (FP32, 2, 1, 256, 16, [(3, 50)]),
    (FP32, 4, 2, 16, 16, [(3, 50)]),
    (BF16, 4, 2, 16, 16, [(17, 60)]),
    (FP16, 4, 2, 32, 16, [(6, 200)]),
    (BF16, 12, 1, 64, 16, [(1, 40), (2, 41)]),
]


def run(s: Step, w, how, lse, decay=1.0, rows=None, decode=False):
    cap, slopes, ranges = how
    return pa.paged_attention_weights(
        w, s.q.cuda(), s.k.cuda(), s.tables.cuda(), s.context_lens.cuda(), s.bs, lse.cuda(),
        None if decode else s.cu.cuda(), max(s.new), decay=decay, weight_rows=cuda(rows),
        softcap=cap, alibi_slopes=cuda(slopes), key_ranges=cuda(ranges))  # fmt: skip


def bound(s: Step, want, old, decay, how):
    """A weight's relative error is its score's (and exp2's argument's rounding, 2^-23 of some
    64), fp32 sums over queries and heads add half a step each."""
    each = score_error(s, how[0], how[1]) + 2.0**-17 + s.q.shape[0] * s.nh * 2.0**-24
    return (want - (old.double() * decay if decay else 0)).abs() * each + want.abs() * 2.0**-22 + 1e-30


@pytest.mark.parametrize("mods", ["", "c", "d", "r", "cdr"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_weights(shape, mods):
    dtype, nh, nkv, hd, bs, chunks = shape
    s = Step(dtype, nh, nkv, hd, bs, [c for _, c in chunks], [n for n, _ in chunks], seed=2)
    how = how_of(s, mods)
    lse = attention64(s, *how)[1].float()
    old = torch.rand(len(chunks) + 1, s.tables.shape[1] * bs + 3, generator=torch.Generator().manual_seed(1))
    for decay in (1.0, 0.0, 0.75):
        w = old.cuda()
        if decay == 0.0:
            for i, n in enumerate(s.ctx):
                w[i, :n] = float("nan")  # not read
        got = run(s, w, how, lse, decay).cpu()
        assert got.data_ptr() != 0
        want = weights64(s, old, decay, lse, *how)
        err = (got.double() - want).abs()
        assert bool((err <= bound(s, want, old, decay, how)).all()), float(err.max())
        for i, n in enumerate(s.ctx):  # behind the context, and rows of nobody
            assert torch.equal(got[i, n:], old[i, n:])
        assert torch.equal(got[-1], old[-1])


def test_weights_single_queries_and_rows():
    """One query per sequence without cu_seqlens_q; rows by index, some outside; twice the same
    bits."""
    s = Step(BF16, 8, 2, 128, 16, [70, 200, 33, 90], [1] * 4, seed=4)
    how = (None, None, None)
    lse = attention64(s)[1].float()
    rows = torch.tensor([3, -1, 0, 9])
    old = torch.rand(5, s.tables.shape[1] * 16)
    w = old.cuda()
    got = run(s, w, how, lse, 0.5, rows, decode=True).cpu()
    want = weights64(s, old, 0.5, lse, rows=rows)
    assert bool(((got.double() - want).abs() <= bound(s, want, old, 0.5, how)).all())
    assert torch.equal(got[[1, 2, 4]], old[[1, 2, 4]])
    again = run(s, old.cuda(), how, lse, 0.5, rows, decode=True).cpu()
    assert torch.equal(got, again)


def test_weights_many_key_groups():
    """Contexts long enough that a workgroup takes several groups of keys one after the other, and
    a sum that must come to heads x queries."""
    b = 70
    g = torch.Generator().manual_seed(3)
    ctx = torch.randint(0, 5000, (b,), generator=g).tolist()
    s = Step(BF16, 4, 2, 64, 16, ctx, [1] * b, seed=5, width=320)
    lse = torch.empty(b, 4, device="cuda")
    pa.paged_decode_attention(s.q.cuda(), s.k.cuda(), s.v.cuda(), s.tables.cuda(),
                              s.context_lens.cuda(), 16, lse=lse)  # fmt: skip
    w = torch.zeros(b, 320 * 16, device="cuda")
    run(s, w, (None, None, None), lse, decode=True)
    live = torch.tensor([n > 0 for n in ctx])
    # every weight off by at most the error of a score and of the normaliser, and their sum
    total = w.double().sum(1).cpu()
    assert bool(((total[live] - 4).abs() <= 4 * (2 * score_error(s) + 5000 * 2.0**-24 + 2.0**-16)).all())
    assert bool((total[~live] == 0).all())
    for i in (0, 17, 69):
        one = Step(BF16, 4, 2, 64, 16, [ctx[i]], [1], seed=5)
        one.k, one.v, one.tables, one.q = s.k, s.v, s.tables[i : i + 1], s.q[i : i + 1]
        want = weights64(one, torch.zeros(1, 5120), 1.0, lse[i : i + 1].cpu())
        err = (w[i].cpu().double() - want[0]).abs()
        assert bool((err <= bound(one, want, torch.zeros(1, 5120), 1.0, (None, None, None))[0]).all())


def test_weights_masked_garbage():
    """Keys that no query sees hold NaN: their weights stay what the decay makes of them."""
    s = Step(FP16, 8, 2, 64, 16, [100, 40], [3, 1], seed=6)
    ranges = torch.tensor([[20, 60], [30, 70], [33, 34], [5, 5]], dtype=torch.int32)
    s.k[s.slots(0)[:20] + s.slots(0)[70:] + s.slots(1)] = float("nan")
    how = (7.0, slopes_of(8), ranges)
    lse = attention64(s, *how)[1].float()
    assert bool((lse[3] == -math.inf).all())
    old = torch.rand(2, s.tables.shape[1] * 16)
    got = run(s, old.cuda(), how, lse, 1.0).cpu()
    want = weights64(s, old, 1.0, lse, *how)
    assert bool(((got.double() - want).abs() <= bound(s, want, old, 1.0, how)).all())
    assert torch.equal(got[1], old[1])


def test_weights_bad_blocks():
    """A block id outside the pool holds no key: nothing is read there."""
    s = Step(FP32, 4, 2, 64, 16, [60], [2], seed=7)
    lse = attention64(s)[1].float()
    old = torch.rand(1, 64)
    want = weights64(s, old, 1.0, lse)
    want[0, 16:48] = old[0, 16:48]
    s.tables[0, 1], s.tables[0, 2] = -3, 1 << 30
    got = run(s, old.cuda(), (None, None, None), lse, 1.0).cpu()
    assert bool(((got.double() - want).abs() <= bound(s, want, old, 1.0, (None, None, None))).all())
