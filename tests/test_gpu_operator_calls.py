"""The operators beside plain attention as a serving program calls them: captured and replayed,
two streams at once, chunks without queries and contexts without tokens, long lists of queries."""

from __future__ import annotations

import pytest
import torch
from operators64 import Step, attention64, evict64, tolerance, weights64
from test_gpu_attention_weights import bound, run
from test_gpu_score_mods import BF16, FP16, FP32, check, decode, how_of, prefill, slopes_of

from engine.kernels import _native
from engine.kernels import paged_attention as pa
from engine.runtime.paged_cache import evict_tokens

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("mods", ["", "r", "cdw"])
@pytest.mark.parametrize("shape", [(BF16, 8, 2, 128, 16, [(100, 420), (70, 70), (3, 200)]),
                                   (FP16, 16, 2, 64, 16, [(90, 300)]),
                                   (FP32, 4, 2, 256, 16, [(70, 150)])], ids=str)  # fmt: skip
def test_weights_of_more_rows_than_a_workgroup_holds(shape, mods):
    """More query rows than the 128 or 256 that stay in registers: the keys are walked over again
    for the next ones, whose masks leave other tiles out."""
    dtype, nh, nkv, hd, bs, chunks = shape
    s = Step(dtype, nh, nkv, hd, bs, [c for _, c in chunks], [n for n, _ in chunks], seed=31)
    how = how_of(s, mods)
    lse = attention64(s, *how)[1].float()
    old = torch.rand(len(chunks), s.tables.shape[1] * bs, generator=torch.Generator().manual_seed(2))
    got = run(s, old.cuda(), how, lse, 0.5).cpu()
    want = weights64(s, old, 0.5, lse, *how)
    err = (got.double() - want).abs()
    assert bool((err <= bound(s, want, old, 0.5, how)).all()), float(err.max())
    again = run(s, old.cuda(), how, lse, 0.5).cpu()
    assert torch.equal(got, again)


@pytest.mark.parametrize("dtype,hd", [(BF16, 128), (FP16, 64), (FP32, 256)])
def test_weights_of_many_rows_over_bad_blocks(dtype, hd):
    """A block id outside the pool holds no key, in tiles that every row sees whole as in others."""
    s = Step(dtype, 4, 1, hd, 16, [300], [20], seed=33)
    lse = attention64(s)[1].float()
    old = torch.rand(1, s.tables.shape[1] * 16, generator=torch.Generator().manual_seed(3))
    want = weights64(s, old, 1.0, lse)
    for block, bad in ((2, -1), (9, 1 << 30), (18, -7)):
        want[0, 16 * block : 16 * block + 16] = old[0, 16 * block : 16 * block + 16].double()
        s.tables[0, block] = bad
    got = run(s, old.cuda(), (None, None, None), lse).cpu()
    err = (got.double() - want).abs()
    assert bool((err <= bound(s, want, old, 1.0, (None, None, None))).all())


@pytest.mark.parametrize("new", [[1, 1, 1], [40, 3, 9]])
def test_weights_captured(new):
    """One graph, other lengths, queries, normalisers and weights at every replay."""
    s = Step(BF16, 8, 2, 64, 16, [150, 60, 33], new, seed=32)
    x = {n: getattr(s, n).cuda() for n in ("q", "k", "tables", "context_lens", "cu")}
    lse = torch.zeros(s.q.shape[:2], device="cuda")
    w = torch.zeros(3, s.tables.shape[1] * 16, device="cuda")

    def call():
        pa.paged_attention_weights(w, x["q"], x["k"], x["tables"], x["context_lens"], 16, lse,
                                   x["cu"], max(new), decay=0.5)  # fmt: skip

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for i in range(4):
        s.ctx = [150 - 20 * i, 60, 33 - 5 * i]
        s.q = torch.randn(s.q.shape, generator=torch.Generator().manual_seed(i)).to(BF16)
        x["context_lens"].copy_(torch.tensor(s.ctx))
        x["q"].copy_(s.q)
        norm = attention64(s)[1].float()
        lse.copy_(norm)
        old = torch.rand(w.shape, generator=torch.Generator().manual_seed(50 + i))
        w.copy_(old)
        graph.replay()
        got = w.cpu()
        want = weights64(s, old, 0.5, norm)
        assert bool(((got.double() - want).abs() <= bound(s, want, old, 0.5, (None, None, None))).all())
        w.copy_(old)
        call()  # an eager call between the replays
        assert torch.equal(got, w.cpu())


def test_two_streams_at_once():
    """Every operator on two streams, each with inputs of its own, in flight together."""
    steps = [Step(BF16, 8, 2, 64, 16, [400, 90], [1, 1], seed=41), Step(BF16, 8, 2, 64, 16, [300, 200], [1, 1], seed=42)]
    chunks = [Step(BF16, 8, 2, 64, 16, [400, 90], [80, 30], seed=43), Step(BF16, 8, 2, 64, 16, [300, 200], [64, 99], seed=44)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    hows = [how_of(s, "cdw") for s in steps], [how_of(s, "cr") for s in chunks]
    for s in steps + chunks:  # uploads once, so that the launches follow each other closely
        s.dev = {n: getattr(s, n).cuda() for n in ("q", "k", "v", "tables", "context_lens", "cu")}
    outs = [[None] * 3, [None] * 3]
    torch.cuda.synchronize()
    for _ in range(3):
        for j, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                for at, (s, how) in enumerate(((steps[j], hows[0][j]), (chunks[j], hows[1][j]))):
                    d, (cap, slopes, ranges) = s.dev, how
                    lse = torch.empty(s.q.shape[:2], device="cuda")
                    more = {"softcap": cap, "key_ranges": ranges.cuda(),
                            "alibi_slopes": None if slopes is None else slopes.cuda()}  # fmt: skip
                    args = (d["q"], d["k"], d["v"], d["tables"], d["context_lens"], 16)
                    if at == 0:
                        outs[j][0] = (pa.paged_decode_attention(*args, lse=lse, **more), lse)
                    else:
                        out = pa.paged_prefill_attention(*args, d["cu"], max(s.new), lse=lse, **more)
                        w = torch.zeros(2, s.tables.shape[1] * 16, device="cuda")
                        pa.paged_attention_weights(w, d["q"], d["k"], d["tables"], d["context_lens"],
                                                   16, lse, d["cu"], max(s.new), **more)  # fmt: skip
                        outs[j][1], outs[j][2] = (out, lse), w
    torch.cuda.synchronize()
    for j in range(2):
        check(steps[j], *outs[j][0], hows[0][j])
        check(chunks[j], *outs[j][1], hows[1][j], True)
        s, how = chunks[j], hows[1][j]
        lse = outs[j][1][1].cpu()
        want = weights64(s, torch.zeros(outs[j][2].shape), 1.0, lse, *how)
        err = (outs[j][2].cpu().double() - want).abs()
        assert bool((err <= bound(s, want, torch.zeros(want.shape), 1.0, how)).all())


@pytest.mark.parametrize("mods", ["", "c", "d", "r", "cdw"])
def test_nothing_to_do(mods):
    """Chunks without queries, contexts without tokens, between ordinary ones."""
    s = Step(BF16, 8, 2, 64, 16, [50, 40, 33, 1], [20, 0, 33, 1], seed=45)
    how = how_of(s, mods)
    lse = torch.empty(s.q.shape[:2], device="cuda")
    check(s, prefill(s, how, lse=lse), lse, how, True)
    old = torch.rand(4, s.tables.shape[1] * 16)
    got = run(s, old.cuda(), how, lse.cpu(), 0.5).cpu()
    want = weights64(s, old, 0.5, lse.cpu(), *how)
    assert bool(((got.double() - want).abs() <= bound(s, want, old, 0.5, how)).all())
    d = Step(BF16, 8, 2, 64, 16, [50, 0, 33], [1, 0, 1], seed=46)
    d.q = torch.cat([d.q[:1], torch.randn(1, 8, 64).to(BF16), d.q[1:]])
    cap, slopes, ranges = how_of(d, mods)
    if ranges is not None:
        ranges = torch.stack([ranges[0], torch.tensor([0, 9], dtype=torch.int32), ranges[1]])
    lse = torch.empty(3, 8, device="cuda")
    out = decode(d, (cap, slopes, ranges), lse=lse).cpu()
    assert bool((out[1] == 0).all()) and bool((lse[1] == -float("inf")).all())
    d.q = d.q[[0, 2]]
    want, _ = attention64(d, cap, slopes, None if ranges is None else ranges[[0, 2]])
    assert bool(((out[[0, 2]].double() - want).abs() <= tolerance(d, want, BF16, cap, slopes)).all())


def test_two_sequences_with_one_row_of_weights_raise_under_debug_checks():
    s = Step(BF16, 4, 2, 64, 16, [40, 30], [1, 1], seed=47)
    lse = attention64(s)[1].float()
    w = torch.zeros(3, s.tables.shape[1] * 16, device="cuda")
    prev = _native.set_debug_checks(True)
    try:
        with pytest.raises(IndexError, match="one row of weights"):
            run(s, w, (None, None, None), lse, rows=torch.tensor([2, 2]), decode=True)
        with pytest.raises(IndexError, match="one row of weights"):
            evict_tokens(s.k.cuda(), s.v.cuda(), w, s.tables.cuda(), s.context_lens.cuda(), 16, 20, 4,
                         weight_rows=torch.tensor([1, 1], device="cuda"))  # fmt: skip
        run(s, w, (None, None, None), lse, rows=torch.tensor([-1, 7]), decode=True)  # both skipped
    finally:
        _native.set_debug_checks(prev)
    assert bool((w == 0).all())


def test_many_steps_of_one_budget():
    """A chat that stays at its budget: append, attend, accumulate, evict at every fourth token,
    against 64 bits from the cache that the step before left."""
    nh, nkv, hd, bs, keep = 8, 2, 64, 16, 40
    g = torch.Generator().manual_seed(48)
    s = Step(FP16, nh, nkv, hd, bs, [keep], [1], seed=48, width=4)
    s.tables[0] = torch.tensor([2, 0, 3, 1])
    k, v = torch.randn(64, nkv, hd, generator=g).to(FP16), torch.randn(64, nkv, hd, generator=g).to(FP16)
    gk, gv, w = k.cuda(), v.cuda(), torch.zeros(1, 64, device="cuda")
    ctx = torch.tensor([keep], dtype=torch.int32, device="cuda")
    tables, slopes = s.tables.cuda(), slopes_of(nh)
    for _ in range(12):
        ctx += 1
        n = int(ctx)
        slot = int(s.tables[0, (n - 1) // bs]) * bs + (n - 1) % bs
        gk[slot], gv[slot] = (torch.randn(2, nkv, hd, generator=g).to(FP16)).cuda()
        w[0, n - 1] = 0
        s.ctx, s.k, s.v = [n], gk.cpu(), gv.cpu()
        s.q = torch.randn(1, nh, hd, generator=g).to(FP16)
        lse = torch.empty(1, nh, device="cuda")
        old = w.cpu()
        out = pa.paged_decode_attention(s.q.cuda(), gk, gv, tables, ctx, bs, softcap=20.0,
                                        alibi_slopes=slopes.cuda(), lse=lse)  # fmt: skip
        check(s, out, lse, (20.0, slopes, None))
        pa.paged_attention_weights(w, s.q.cuda(), gk, tables, ctx, bs, lse, softcap=20.0,
                                   alibi_slopes=slopes.cuda())  # fmt: skip
        want = weights64(s, old, 1.0, lse.cpu(), 20.0, slopes)
        err = (w.cpu().double() - want).abs()
        assert bool((err <= bound(s, want, old, 1.0, (20.0, slopes, None))).all())
        if n == keep + 4:
            before = w.cpu()
            evict_tokens(gk, gv, w, tables, ctx, bs, keep, 8, out=ctx)
            lens, wk, wv, ww = evict64(s.k[None], s.v[None], before[None], s.tables, [n], bs, keep, 8)
            assert ctx.tolist() == lens == [keep]
            assert torch.equal(gk.cpu(), wk[0]) and torch.equal(gv.cpu(), wv[0])
            assert torch.equal(w.cpu(), ww[0])
