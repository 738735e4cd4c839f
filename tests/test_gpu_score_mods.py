"""Attention with capped, biased and range-masked scores against 64 bits (tests/operators64.py),
decode and prefill, at the sizes and masks where they can go wrong."""

from __future__ import annotations

import math

import pytest
import torch
from operators64 import Step, _finite, attention64, tolerance

from engine.kernels import paged_attention as pa
from engine.model import layers
from engine.runtime.paged_cache import KVShape, PagedBatch, PagedKVCache, step_key_ranges

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def slopes_of(nh: int) -> torch.Tensor:
    return torch.exp2(-8.0 * torch.arange(1, nh + 1) / nh).float()


def random_ranges(s: Step, seed: int, empty: float = 0.15) -> torch.Tensor:
    """Any [lo, hi) per query row: cut ones, empty ones, ones past the context or before 0."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for i, _ in s.positions():
        n = max(s.ctx[i], 1)
        lo, hi = sorted(torch.randint(-2, n + 3, (2,), generator=g).tolist())
        if torch.rand((), generator=g) < empty:
            lo, hi = hi + 1, lo
        out.append([lo, hi])
    return torch.tensor(out, dtype=torch.int32).view(-1, 2)


def how_of(s: Step, mods: str, seed: int = 5):
    """(softcap, slopes, ranges) of a string of c(ap), d(istance), r(anges), w(indow)."""
    ranges = None
    if "r" in mods:
        ranges = random_ranges(s, seed)
    elif "w" in mods:
        ranges = torch.tensor([[max(0, p - 36), p + 1] for _, p in s.positions()], dtype=torch.int32)
    return 11.0 if "c" in mods else None, slopes_of(s.nh) if "d" in mods else None, ranges


def cuda(x):
    return None if x is None else x.cuda()


def decode(s: Step, mods, out=None, lse=None, **more):
    cap, slopes, ranges = mods
    return pa.paged_decode_attention(s.q.cuda(), s.k.cuda(), s.v.cuda(), s.tables.cuda(),
                                     s.context_lens.cuda(), s.bs, softcap=cap,
                                     alibi_slopes=cuda(slopes), key_ranges=cuda(ranges), out=out,
                                     lse=lse, **more)  # fmt: skip


def prefill(s: Step, mods, out=None, lse=None, **more):
    cap, slopes, ranges = mods
    return pa.paged_prefill_attention(s.q.cuda(), s.k.cuda(), s.v.cuda(), s.tables.cuda(),
                                      s.context_lens.cuda(), s.bs, s.cu.cuda(), max(s.new),
                                      softcap=cap, alibi_slopes=cuda(slopes),
                                      key_ranges=cuda(ranges), out=out, lse=lse, **more)  # fmt: skip


def check(s: Step, got, lse, mods, p16=False):
    cap, slopes, _ = mods
    want, want_lse = attention64(s, *mods)
    got = got.cpu()
    err = (got.double() - want).abs()
    tol = tolerance(s, want, got.dtype, cap, slopes, p16)
    assert bool((err <= tol).all()), f"max error {err.max()}, {(err > tol).sum()} past the bound"
    if lse is not None:
        lse = lse.cpu().double()
        empty = want_lse == -math.inf
        assert torch.equal(lse == -math.inf, empty)
        # log2 units: the scores' error, fp32 sums of weights, and log2 itself near the value
        rel = tolerance(s, torch.zeros(()), FP32, cap, slopes, p16) / float(_finite(s.v).abs().max())
        bound = rel * 1.4427 + 2.0**-21 * (1 + want_lse.abs())
        assert bool(((lse - want_lse).abs() <= bound)[~empty].all())


# --- decode ---------------------------------------------------------------------------------

DECODE = [
    # dtype, heads, KV heads, head_dim, block size, contexts
    (BF16, 8, 2, 128, 16, [1, 16, 17, 300, 0, 129]),  # split pass, one launch
    (FP16, 8, 2, 64, 16, [5, 33, 200, 1]),
    (BF16, 4, 4, 64, 16, [31, 64, 100]),
    (BF16, 16, 2, 128, 16, [40, 77, 160, 2]),  # wide form: groups of 8
    (FP16, 12, 2, 128, 16, [90, 1, 140]),  # groups of 6
    (BF16, 8, 2, 128, 12, [50, 13, 24]),  # blocks that are no multiple of 16
    (FP16, 6, 2, 64, 5, [11, 64, 7]),
    (FP32, 8, 2, 64, 16, [40, 1, 131, 0]),
    (FP32, 4, 1, 256, 16, [77, 20]),
    (BF16, 4, 2, 16, 16, [70, 3]),
    (FP16, 8, 4, 32, 16, [65, 100]),
    (BF16, 10, 2, 256, 16, [33, 80]),  # groups of 5 on the VALU form
]


@pytest.mark.parametrize("mods", ["c", "d", "r", "w", "cdr", ""])
@pytest.mark.parametrize("shape", DECODE, ids=str)
def test_decode(shape, mods):
    dtype, nh, nkv, hd, bs, ctx = shape
    s = Step(dtype, nh, nkv, hd, bs, ctx, [1] * len(ctx), seed=3)
    how = how_of(s, mods)
    lse = torch.empty(len(ctx), nh, device="cuda")
    check_step(s, how, lse)


def check_step(s, how, lse, **more):
    check(s, decode(s, how, lse=lse, **more), lse, how)


@pytest.mark.parametrize("ranges", [1, 3, 40, 200])
@pytest.mark.parametrize("shape", [DECODE[0], DECODE[3], DECODE[5], DECODE[7], DECODE[1]], ids=str)
def test_decode_split_counts(shape, ranges):
    """Any number of ranges, fewer and more than there are units of work (the combine)."""
    dtype, nh, nkv, hd, bs, ctx = shape
    s = Step(dtype, nh, nkv, hd, bs, ctx, [1] * len(ctx), seed=4)
    check_step(s, how_of(s, "cdr", 9), torch.empty(len(ctx), nh, device="cuda"), num_workgroups=ranges)


@pytest.mark.parametrize("batch", [65, 130, 1030])
@pytest.mark.parametrize("hd,dtype", [(64, BF16), (128, FP16), (32, BF16)])
def test_decode_large_batches(batch, hd, dtype):
    """Lengths staged in LDS (65 to 1,024 sequences) and walked (more)."""
    g = torch.Generator().manual_seed(batch)
    ctx = torch.randint(0, 70, (batch,), generator=g).tolist()
    s = Step(dtype, 4, 2, hd, 16, ctx, [1] * batch, seed=1)
    check_step(s, how_of(s, "cr"), torch.empty(batch, 4, device="cuda"), num_workgroups=96)
    check_step(s, how_of(s, "d"), None)


def test_decode_long_window():
    """Ranges that start far into a long context and end before it, across table windows."""
    ctx = [9000, 2500, 4097]
    s = Step(BF16, 8, 2, 128, 16, ctx, [1] * 3, seed=2)
    ranges = torch.tensor([[7003, 8999], [100, 2101], [4090, 4097]], dtype=torch.int32)
    check_step(s, (30.0, slopes_of(8), ranges), torch.empty(3, 8, device="cuda"))
    check_step(s, (None, None, ranges), None)


def test_decode_rows_out_and_streams():
    """Rows of a larger step (negative, outside), an fp32 result, padded strides, another stream."""
    ctx = [40, 77, 20, 66]
    s = Step(BF16, 8, 2, 128, 16, ctx, [1] * 4, seed=6)
    rows = torch.tensor([5, -1, 9, 2])  # of 8: row 9 does not exist
    big = torch.zeros(8, 8, 128, dtype=BF16)
    big[[5, 7, 2]] = s.q[[0, 1, 3]]
    ranges = torch.full((8, 2), 3, dtype=torch.int32)
    ranges[5], ranges[7], ranges[2] = (torch.tensor(x) for x in ((2, 40), (60, 77), (0, 66)))
    q = big.cuda()
    out = torch.full_like(q, 7.0)
    k = torch.full((s.k.shape[0], 3, 128), float("nan"), dtype=BF16, device="cuda")
    v = torch.full_like(k, float("nan"))
    k[:, :2], v[:, :2] = s.k.cuda(), s.v.cuda()
    lse = torch.full((4, 8), 5.0, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        pa.paged_decode_attention(q, k[:, :2], v[:, :2], s.tables.cuda(), s.context_lens.cuda(),
                                  16, out=out, rows=rows.cuda(), softcap=9.0,
                                  key_ranges=ranges.cuda(), lse=lse)  # fmt: skip
    torch.cuda.current_stream().wait_stream(stream)
    seq = torch.tensor([[2, 40], [60, 77], [0, 0], [0, 66]], dtype=torch.int32)
    want, _ = attention64(s, 9.0, None, seq)
    got = out.cpu()
    for row, i in ((5, 0), (7, 1), (2, 3)):
        assert bool(((got[row].double() - want[i]).abs() <= tolerance(s, want[i], BF16, 9.0)).all())
    left = [r for r in range(8) if r not in (5, 7, 2)]
    assert bool((got[left] == 7.0).all())  # rows that no sequence names
    # an fp32 result of the same call
    s.tables[2, :] = s.tables[0, 0]
    out32 = torch.empty(4, 8, 128, device="cuda")
    check(s, decode(s, (9.0, None, seq), out=out32), None, (9.0, None, seq))


@pytest.mark.parametrize("hd,dtype,nh", [(128, BF16, 8), (64, FP16, 8), (128, FP16, 16), (64, FP32, 8)])
def test_decode_poison_outside_ranges(hd, dtype, nh):
    """Keys outside a sequence's range hold NaN and infinities in K and V: none reaches its row."""
    ctx = [100, 61, 16, 48]
    s = Step(dtype, nh, 2, hd, 16, ctx, [1] * 4, seed=8)
    ranges = torch.tensor([[37, 90], [5, 7], [15, 16], [9, 9]], dtype=torch.int32)
    for i, (lo, hi) in enumerate(ranges.tolist()):
        out = s.slots(i)[:lo] + s.slots(i)[hi:]
        s.k[out], s.v[out] = float("nan"), float("inf")
    for wgs in (None, 1, 7):
        lse = torch.empty(4, nh, device="cuda")
        check(s, decode(s, (20.0, None, ranges), lse=lse, num_workgroups=wgs), lse, (20.0, None, ranges))


# --- prefill --------------------------------------------------------------------------------

PREFILL = [
    (BF16, 8, 2, 128, 16, [(70, 70), (5, 133), (33, 40)]),
    (FP16, 8, 2, 64, 16, [(17, 150), (64, 64), (2, 3)]),
    (BF16, 4, 4, 64, 16, [(130, 200)]),
    (FP16, 6, 2, 128, 16, [(50, 51)]),
    (BF16, 8, 1, 32, 16, [(40, 77)]),
    (BF16, 4, 2, 256, 16, [(33, 90), (1, 40)]),
    (FP16, 4, 2, 256, 16, [(20, 64)]),
    (BF16, 4, 2, 128, 12, [(30, 61)]),
    (FP16, 4, 2, 64, 5, [(21, 33)]),
    (FP32, 8, 2, 64, 16, [(40, 100), (3, 3)]),
    (FP32, 4, 2, 128, 16, [(20, 70)]),
    (FP32, 2, 1, 256, 16, [(18, 33)]),
    (FP32, 4, 2, 32, 16, [(9, 50)]),
    (BF16, 4, 2, 16, 16, [(30, 64)]),
    (FP16, 4, 4, 16, 16, [(16, 16)]),
]


def step_of(shape, seed=1):
    dtype, nh, nkv, hd, bs, chunks = shape
    return Step(dtype, nh, nkv, hd, bs, [c for _, c in chunks], [n for n, _ in chunks], seed=seed)


def p16(s: Step) -> bool:
    return s.dtype != FP32 and s.hd > 16


@pytest.mark.parametrize("mods", ["c", "d", "r", "w", "cdr", ""])
@pytest.mark.parametrize("shape", PREFILL, ids=str)
def test_prefill(shape, mods):
    s = step_of(shape)
    how = how_of(s, mods)
    lse = torch.empty(s.q.shape[:2], device="cuda")
    check(s, prefill(s, how, lse=lse), lse, how, p16(s))


@pytest.mark.parametrize("shape", [PREFILL[0], PREFILL[2], PREFILL[5]], ids=str)
def test_prefill_without_workspace(shape):
    """bf16 without the fp16 copy of V (P as a hi + lo pair)."""
    s = step_of(shape, 2)
    how = how_of(s, "cdr", 4)
    none = torch.empty(0, dtype=torch.uint8, device="cuda")
    check(s, prefill(s, how, workspace=none), None, how, True)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_prefill_documents_and_prefixes(dtype):
    """Documents that do not see each other, and a prefix that sees itself both ways."""
    s = Step(dtype, 4, 2, 64, 16, [300, 150], [260, 150], seed=3)
    docs = step_key_ranges(s.ctx, s.new, "cpu", doc_starts=[[0, 100, 101, 250], [0, 64]])
    check(s, prefill(s, (None, None, docs)), None, (None, None, docs), p16(s))
    both = step_key_ranges(s.ctx, s.new, "cpu", prefix_lens=[120, 500])
    check(s, prefill(s, (None, slopes_of(4), both)), None, (None, slopes_of(4), both), p16(s))


@pytest.mark.parametrize("dtype,hd", [(BF16, 128), (FP16, 128), (BF16, 64), (FP32, 64), (BF16, 256)])
def test_prefill_poison_in_masked_places(dtype, hd):
    """V of one document holds infinities and NaN: the other documents' rows, in the same tiles,
    are as without them, and rows without keys are 0; K's garbage likewise."""
    s = Step(dtype, 4, 2, hd, 16, [150], [150], seed=5)
    ranges = step_key_ranges(s.ctx, s.new, "cpu", doc_starts=[[0, 40, 55, 130]])
    ranges[60:64] = 0
    bad = s.slots(0)[40:55]
    s.v[bad[:5]], s.v[bad[5:]] = float("inf"), float("nan")
    s.k[bad[3:]] = float("nan")
    for softcap in (None, 15.0):
        lse = torch.empty(s.q.shape[:2], device="cuda")
        got = prefill(s, (softcap, None, ranges), lse=lse).cpu()
        want, _ = attention64(s, softcap, None, ranges)
        clean = torch.tensor([not 40 <= p < 55 for p in range(150)])
        tol = tolerance(s, want[clean], dtype, softcap, None, p16(s))
        assert bool(((got[clean].double() - want[clean]).abs() <= tol).all())
        assert bool((got[60:64] == 0).all())
        assert not bool(torch.isfinite(got[40:55].float()).any(-1).all())


def test_prefill_rows_in_place_and_layers():
    """A mixed step through layers.paged_attention: decode rows and chunks with one range per
    token, in place and through gathered copies (a layout the kernels cannot address)."""
    nh, nkv, hd, bs = 8, 2, 64, 16
    ctx, new = [90, 33, 50, 1, 70], [40, 1, 1, 1, 20]
    cache = PagedKVCache(KVShape(1, nkv, hd), 40, bs, "cuda", BF16)
    s = Step(BF16, nh, nkv, hd, bs, ctx, new, seed=7, spare=3)
    cache.k[0, : s.k.shape[0]].copy_(s.k)
    cache.v[0, : s.v.shape[0]].copy_(s.v)
    tables = [s.tables[i, : -(-n // bs)].tolist() for i, n in enumerate(ctx)]
    batch = PagedBatch.build(cache, tables, ctx, new, "cuda", use_kernel=True)
    assert batch.mixed
    k = torch.cat([s.k[s.slots(i)[n - m :]] for i, (n, m) in enumerate(zip(ctx, new, strict=True))])
    v = torch.cat([s.v[s.slots(i)[n - m :]] for i, (n, m) in enumerate(zip(ctx, new, strict=True))])
    ranges = step_key_ranges(ctx, new, "cuda", window=29)
    how = {"softcap": 12.0, "alibi_slopes": slopes_of(nh).cuda(), "key_ranges": ranges}
    want, _ = attention64(s, 12.0, slopes_of(nh), ranges.cpu())
    tol = tolerance(s, want, BF16, 12.0, slopes_of(nh), True)
    got = layers.paged_attention(0, s.q.cuda(), k.cuda(), v.cuda(), batch, **how)
    assert bool(((got.view(want.shape).cpu().double() - want).abs() <= tol).all())
    odd = torch.empty(s.q.shape[0], nh, hd + 4, dtype=BF16, device="cuda")[..., :hd]
    odd.copy_(s.q)
    got = layers.paged_attention(0, odd, k.cuda(), v.cuda(), batch, **how)
    assert bool(((got.view(want.shape).cpu().double() - want).abs() <= tol).all())
    # a decode batch
    batch = PagedBatch.build(cache, tables, ctx, [1] * 5, "cuda", use_kernel=True)
    d = Step(BF16, nh, nkv, hd, bs, ctx, [1] * 5, seed=7, spare=3)
    d.tables, d.k, d.v = s.tables, s.k, s.v
    last = [s.slots(i)[-1] for i in range(5)]
    how["key_ranges"] = step_key_ranges(ctx, [1] * 5, "cuda", window=29)
    got = layers.paged_attention(0, d.q.cuda(), s.k[last].cuda(), s.v[last].cuda(), batch, **how)
    want, _ = attention64(d, 12.0, slopes_of(nh), how["key_ranges"].cpu())
    tol = tolerance(d, want, BF16, 12.0, slopes_of(nh))
    assert bool(((got.view(want.shape).cpu().double() - want).abs() <= tol).all())


def test_modified_matches_plain_without_modifiers():
    """With ranges that are the causal limits and no cap, both forms give the same attention."""
    s = step_of(PREFILL[0], 11)
    plain = pa.paged_prefill_attention(s.q.cuda(), s.k.cuda(), s.v.cuda(), s.tables.cuda(),
                                       s.context_lens.cuda(), 16, s.cu.cuda(), max(s.new))  # fmt: skip
    check(s, plain, None, (None, None, None), True)
    check(s, prefill(s, (None, None, s.causal())), None, (None, None, None), True)


def test_captured_calls():
    """A graph of a decode and a prefill call serves new lengths, ranges and queries."""
    s = Step(BF16, 8, 2, 64, 16, [60, 100, 9], [1, 1, 1], seed=12)
    c = Step(BF16, 8, 2, 64, 16, [60, 100], [30, 7], seed=13)
    x = {n: getattr(s, n).cuda() for n in ("q", "k", "v", "tables", "context_lens")}
    y = {n: getattr(c, n).cuda() for n in ("q", "k", "v", "tables", "context_lens", "cu")}
    rs, rc = random_ranges(s, 1).cuda(), random_ranges(c, 2).cuda()
    lse = torch.empty(3, 8, device="cuda")

    def both():
        a = pa.paged_decode_attention(x["q"], x["k"], x["v"], x["tables"], x["context_lens"], 16,
                                      softcap=8.0, key_ranges=rs, lse=lse)  # fmt: skip
        b = pa.paged_prefill_attention(y["q"], y["k"], y["v"], y["tables"], y["context_lens"], 16,
                                       y["cu"], 30, softcap=8.0, key_ranges=rc)  # fmt: skip
        return a, b

    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a, b = both()
    for k in range(3):
        rs.copy_(random_ranges(s, 20 + k))
        rc.copy_(random_ranges(c, 30 + k))
        x["q"].normal_(generator=torch.Generator("cuda").manual_seed(k))
        s.q = x["q"].cpu()
        s.ctx = [60 - k, 100, 9 + k]
        s.ctx[2] = min(s.ctx[2], 16)
        x["context_lens"].copy_(torch.tensor(s.ctx))
        graph.replay()
        check(s, a, lse, (8.0, None, rs.cpu()))
        check(c, b, None, (8.0, None, rc.cpu()), True)
        ea, eb = both()
        assert torch.equal(ea, a) and torch.equal(eb, b)
