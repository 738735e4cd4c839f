"""The 16-bit prefill's kernels for ranges, a cap, a bias and all of them: each combination, the
cap's two forms in one call, biases of keys that are all far away, masked infinities."""

from __future__ import annotations

import pytest
import torch
from operators64 import Step, attention64, tolerance
from test_gpu_score_mods import BF16, FP16, check, how_of, prefill, slopes_of

pytestmark = pytest.mark.gpu

SHAPES = [
    (BF16, 8, 2, 128, 16, [(70, 70), (5, 133), (33, 40)]),
    (FP16, 6, 2, 64, 16, [(17, 150), (64, 64), (2, 3)]),
    (BF16, 4, 4, 64, 16, [(130, 200)]),
    (BF16, 8, 1, 32, 32, [(40, 77)]),
    (FP16, 4, 2, 256, 16, [(33, 90), (1, 40)]),
    (FP16, 4, 2, 128, 24, [(33, 90), (1, 40)]),
]


def step_of(shape, seed=21):
    dtype, nh, nkv, hd, bs, chunks = shape
    return Step(dtype, nh, nkv, hd, bs, [c for _, c in chunks], [n for n, _ in chunks], seed=seed)


@pytest.mark.parametrize("mods", ["cr", "cw", "dr", "dw", "cd", "cdw"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_combinations(shape, mods):
    s = step_of(shape)
    how = how_of(s, mods, 9)
    lse = torch.empty(s.q.shape[:2], device="cuda")
    check(s, prefill(s, how, lse=lse), lse, how, True)


@pytest.mark.parametrize("distance", [False, True])
@pytest.mark.parametrize("cap", [0.5, 6.0, 30.0, 1000.0, 1e-20])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_cap_of_small_and_large_scores(shape, cap, distance):
    """Every fifth query row is eight times as long and key 20 of each sequence too: the scores of
    some tiles reach the cap, others stay far below it."""
    s = step_of(shape, 22)
    s.q[::5] *= 8
    for i, n in enumerate(s.ctx):
        if n > 20:
            s.k[s.slots(i)[20]] *= 8
    how = (cap, slopes_of(s.nh) if distance else None, None)
    lse = torch.empty(s.q.shape[:2], device="cuda")
    check(s, prefill(s, how, lse=lse), lse, how, True)


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("shape", [SHAPES[0], SHAPES[1], SHAPES[5]], ids=str)
def test_bias_of_far_keys(shape, sign):
    """Rows that see only keys far behind them, or ahead of them, or one key: the bias common to a
    row's keys does not cost the others their bits, and the normaliser holds it. A negative slope
    favours the far ones."""
    dtype, nh, nkv, hd, bs, _ = shape
    ctx, new = [1500, 700], [30, 40]
    s = Step(dtype, nh, nkv, hd, bs, ctx, new, seed=23)
    rows = []
    for j, (i, p) in enumerate(s.positions()):
        rows.append([[0, 90], [p - 3, p - 2], [p + 1, p + 9], [max(0, p - 700), p + 1], [40, 41]][(j + i) % 5])
    ranges = torch.tensor(rows, dtype=torch.int32)
    how = (None, sign * slopes_of(nh), ranges)
    lse = torch.empty(s.q.shape[:2], device="cuda")
    check(s, prefill(s, how, lse=lse), lse, how, True)


@pytest.mark.parametrize("shape", [SHAPES[0], SHAPES[1], SHAPES[3], SHAPES[5]], ids=str)
@pytest.mark.parametrize("mods", ["c", "d", "cd", ""])
def test_masked_infinities(shape, mods):
    """Keys of other documents with infinities and NaN in K, and in V: nothing of them reaches the
    rows that do not see them."""
    dtype, nh, nkv, hd, bs, _ = shape
    s = Step(dtype, nh, nkv, hd, bs, [150], [110], seed=24)
    bad = s.slots(0)[48:60]
    s.k[bad[:4]], s.k[bad[4:8]], s.k[bad[8:]] = float("inf"), float("-inf"), float("nan")
    s.v[bad[::2]], s.v[bad[1::2]] = float("nan"), float("inf")
    ranges = torch.tensor([[60, p + 1] if p >= 60 else [0, min(p + 1, 48)] for _, p in s.positions()],
                          dtype=torch.int32)  # fmt: skip
    cap = 15.0 if "c" in mods else None
    slopes = slopes_of(nh) if "d" in mods else None
    got = prefill(s, (cap, slopes, ranges)).cpu()
    want, _ = attention64(s, cap, slopes, ranges)
    assert bool(((got.double() - want).abs() <= tolerance(s, want, dtype, cap, slopes, True)).all())
