"""Eviction by accumulated weight: bit for bit what sorting on the host gives."""

from __future__ import annotations

import pytest
import torch
from operators64 import Step, attention64, evict64, tolerance

from engine.kernels import _native
from engine.kernels import paged_attention as pa
from engine.runtime.block_manager import BlockManager
from engine.runtime.paged_cache import KVShape, PagedKVCache, evict_tokens, evict_workspace_bytes

pytestmark = pytest.mark.gpu


def pools(layers, dtype, nkv, hd, bs, ctx, seed, width=None, spare=2):
    s = Step(dtype, nkv, nkv, hd, bs, ctx, [0] * len(ctx), seed=seed, width=width, spare=spare)
    g = torch.Generator().manual_seed(seed + 1)
    shape = (layers, s.k.shape[0], nkv, hd)
    k = torch.randn(shape, generator=g).to(dtype)
    v = torch.randn(shape, generator=g).to(dtype)
    w = torch.rand(layers, len(ctx), s.tables.shape[1] * bs, generator=g) ** 3
    for i, n in enumerate(ctx):
        w[:, i, max(n, 0) :] = 0.25  # behind a context: not the operator's
    return s, k, v, w


def check(s, k, v, w, keep, recent, rows=None, **more):
    want = evict64(k, v, w, s.tables, s.ctx, s.bs, keep, recent, rows)
    gk, gv, gw = k.cuda(), v.cuda(), w.cuda()
    lens = evict_tokens(gk, gv, gw, s.tables.cuda(), s.context_lens.cuda(), s.bs, keep, recent,
                        weight_rows=None if rows is None else rows.cuda(), **more)  # fmt: skip
    assert lens.tolist() == want[0] and lens.dtype == torch.int32
    bits = torch.int32 if k.dtype == torch.float32 else torch.int16
    assert torch.equal(gk.cpu().view(bits), want[1].view(bits))
    assert torch.equal(gv.cpu().view(bits), want[2].view(bits))
    assert torch.equal(gw.cpu().view(torch.int32), want[3].view(torch.int32))
    return lens


@pytest.mark.parametrize("keep,recent", [(64, 16), (1, 0), (1, 1), (50, 50), (33, 0), (0, 0), (200, 8)])
@pytest.mark.parametrize(
    "dtype,nkv,hd,bs",
    [(torch.bfloat16, 2, 64, 16), (torch.float16, 3, 16, 12), (torch.float32, 1, 128, 16),
     (torch.bfloat16, 8, 128, 16), (torch.float16, 1, 16, 5)],
)  # fmt: skip
def test_evict(dtype, nkv, hd, bs, keep, recent):
    ctx = [100, 65, 64, 0, 1, 63, 190, 51]
    check(*pools(2, dtype, nkv, hd, bs, ctx, seed=keep), keep, recent)


@pytest.mark.parametrize("n", [1023, 1024, 1025, 4096, 5000, 16384, 17000, 33000])
def test_evict_lengths(n):
    """Every size class of the selection, and its edges."""
    s, k, v, w = pools(1, torch.bfloat16, 1, 16, 16, [n, n // 3], seed=n)
    check(s, k, v, w, n // 2, 100)
    check(s, k, v, w, n - 1, n - 1)


@pytest.mark.parametrize("layers,batch,n,keep", [(2, 3, 1500, 1200), (4, 20, 700, 650), (16, 34, 300, 120)])
def test_evict_wide_rows(layers, batch, n, keep):
    """Rows of 1 KB, few and many sequences (each width of the move pass), batches of rows that
    overlap their own destinations."""
    g = torch.Generator().manual_seed(batch)
    ctx = [n - 7 * i % 90 for i in range(batch)]
    width = -(-n // 16)
    tables = torch.randperm(batch * width, generator=g).view(batch, width).int()
    k = torch.randint(-(2**15), 2**15, (layers, batch * width * 16, 8, 64), generator=g).to(torch.bfloat16)
    v = torch.randint(-(2**15), 2**15, k.shape, generator=g).to(torch.bfloat16)
    w = torch.rand(layers, batch, width * 16, generator=g, dtype=torch.float64).float()
    slots = (tables.long()[..., None] * 16 + torch.arange(16)).flatten(1)
    want_k, want_v, want_w = k.clone(), v.clone(), w.clone()
    for layer in range(layers):
        for b, m in enumerate(ctx):
            if m <= keep:
                continue
            old = m - 32
            heavy = torch.sort(w[layer, b, :old], descending=True, stable=True).indices[: keep - 32]
            kept = torch.cat([heavy.sort().values, torch.arange(old, m)])
            src, dst = slots[b, kept], slots[b, :keep]
            want_k[layer, dst], want_v[layer, dst] = k[layer, src], v[layer, src]
            want_w[layer, b, :keep], want_w[layer, b, keep:m] = w[layer, b, kept], 0.0
    gk, gv, gw = k.cuda(), v.cuda(), w.cuda()
    out = evict_tokens(gk, gv, gw, tables.cuda(), torch.tensor(ctx, dtype=torch.int32).cuda(), 16, keep, 32)
    assert out.tolist() == [min(m, keep) for m in ctx]
    assert torch.equal(gk.cpu(), want_k) and torch.equal(gv.cpu(), want_v)
    assert torch.equal(gw.cpu(), want_w)


def test_evict_ties_and_special_weights():
    """Equal weights, zeros of both signs, negatives, infinities and NaN: the lowest positions of
    what is equal stay, a NaN goes first."""
    ctx = [1500, 1500, 1500, 400]
    s, k, v, w = pools(3, torch.bfloat16, 2, 16, 16, ctx, seed=9)
    w[:, 0] = 1.0
    w[:, 1, :1500] = torch.randint(0, 3, (1500,), generator=torch.Generator().manual_seed(2)).float()
    w[0, 2, ::2] = -0.0
    w[0, 2, 1::4] = 0.0
    w[1, 2] -= 0.5
    w[2, 2, 5:900:7] = float("nan")
    w[2, 2, 3:1000:11] = float("inf")
    w[2, 2, 4:1000:13] = -float("inf")
    w[:, 3, :400] = float("nan")
    for keep, recent in ((700, 30), (1499, 0), (100, 0)):
        check(s, k, v, w, keep, recent)


def test_evict_rows_outside_and_bad_blocks():
    """Sequences without a row of weights are left alone; tokens whose block lies outside the pool
    are not moved; a context past its table counts as the table's."""
    s, k, v, w = pools(2, torch.bfloat16, 2, 64, 16, [100, 90, 80, 70], seed=10)
    rows = torch.tensor([3, -1, 4, 0])
    check(s, k, v, w, 40, 10, rows)
    s.tables[0, 4] = -2
    s.tables[3, 0] = 1 << 28
    check(s, k, v, w, 40, 10)
    s.ctx[1] = 100000
    s.context_lens[1] = 100000
    s, k, v, w = pools(1, torch.bfloat16, 2, 64, 16, [112, 90], seed=11)
    s.context_lens[0] = 100000
    s.ctx[0] = 100000
    check(s, k, v, w, 40, 10)


def test_evict_one_layer_strides_out_and_stream():
    s, k, v, w = pools(1, torch.float16, 2, 32, 16, [60, 45], seed=12)
    want = evict64(k, v, w, s.tables, s.ctx, 16, 20, 5)
    wide = torch.zeros(1, 2, 100)
    wide[:, :, : w.shape[2]] = w
    gk, gv, gw = k[0].cuda(), v[0].cuda(), wide[0].cuda()
    ctx = s.context_lens.cuda()
    ws = torch.empty(evict_workspace_bytes(1, 2, s.tables.shape[1], 16, 20), dtype=torch.uint8,
                     device="cuda")  # fmt: skip
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = evict_tokens(gk, gv, gw[:, : w.shape[2]], s.tables.cuda(), ctx, 16, 20, 5, out=ctx,
                           workspace=ws)  # fmt: skip
    torch.cuda.current_stream().wait_stream(stream)
    assert got is ctx and ctx.tolist() == want[0]
    assert torch.equal(gk.cpu(), want[1][0]) and torch.equal(gv.cpu(), want[2][0])
    assert torch.equal(gw[:, : w.shape[2]].cpu(), want[3][0])
    assert bool((gw[:, w.shape[2] :] == 0).all())


def test_evict_captured():
    """A graph serves other lengths and weights; every replay as an eager call."""
    s, k, v, w = pools(2, torch.bfloat16, 2, 64, 16, [200, 150, 90], seed=13)
    gk, gv, gw = k.cuda(), v.cuda(), w.cuda()
    tables, ctx = s.tables.cuda(), s.context_lens.cuda()
    out = torch.empty_like(ctx)
    evict_tokens(gk, gv, gw, tables, ctx, 16, 64, 16, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        evict_tokens(gk, gv, gw, tables, ctx, 16, 64, 16, out=out)
    for i in range(4):
        lens = [200 - 30 * i, 150, 60 + i]
        ctx.copy_(torch.tensor(lens))
        w = torch.rand(w.shape, generator=torch.Generator().manual_seed(i))
        gk.copy_(k), gv.copy_(v), gw.copy_(w)
        graph.replay()
        want = evict64(k, v, w, s.tables, lens, 16, 64, 16)
        assert out.tolist() == want[0]
        assert torch.equal(gk.cpu(), want[1]) and torch.equal(gv.cpu(), want[2])
        assert torch.equal(gw.cpu(), want[3])


def test_evict_shared_blocks_raise_under_debug_checks():
    s, k, v, w = pools(1, torch.bfloat16, 2, 16, 16, [60, 60], seed=14)
    s.tables[1, 0] = s.tables[0, 0]
    prev = _native.set_debug_checks(True)
    try:
        with pytest.raises(IndexError, match="more than one place"):
            check(s, k, v, w, 30, 4)
        check(s, k, v, w, 60, 4)  # nothing is evicted: sharing is fine
    finally:
        _native.set_debug_checks(prev)


def test_attend_accumulate_evict_attend():
    """The operators as they are used: a prompt's attention leaves its normalisers, they give the
    weights, the eviction cuts every layer down, blocks go back, and the next token's capped
    attention over what is left is that of the kept tokens in 64 bits."""
    layers, nh, nkv, hd, bs, keep, recent = 2, 8, 2, 64, 16, 48, 12
    ctx = [130, 75, 40]
    cap = 14.0
    cache = PagedKVCache(KVShape(layers, nkv, hd), 24, bs, "cuda", torch.bfloat16)
    manager = BlockManager(24, bs)
    for i, n in enumerate(ctx):
        manager.grow(i, n)
    width = 9
    tables = torch.zeros(3, width, dtype=torch.int32)
    for i in range(3):
        tables[i, : len(manager.tables[i])] = torch.tensor(manager.tables[i], dtype=torch.int32)
    gen = torch.Generator().manual_seed(4)
    steps = []
    weights = torch.zeros(layers, 3, width * bs, device="cuda")
    lens = torch.tensor(ctx, dtype=torch.int32, device="cuda")
    for layer in range(layers):
        s = Step(torch.bfloat16, nh, nkv, hd, bs, ctx, ctx, seed=20 + layer, width=width)
        s.tables = tables
        shape = (24 * bs, nkv, hd)
        s.k = torch.randn(shape, generator=gen).bfloat16()
        s.v = torch.randn(shape, generator=gen).bfloat16()
        steps.append(s)
        cache.k[layer].copy_(s.k)
        cache.v[layer].copy_(s.v)
        lse = torch.empty(sum(ctx), nh, device="cuda")
        how = {"softcap": cap}
        pa.paged_prefill_attention(s.q.cuda(), cache.k[layer], cache.v[layer], tables.cuda(), lens,
                                   bs, s.cu.cuda(), max(ctx), lse=lse, **how)  # fmt: skip
        pa.paged_attention_weights(weights[layer], s.q.cuda(), cache.k[layer], tables.cuda(), lens,
                                   bs, lse, s.cu.cuda(), max(ctx), decay=0.0, **how)  # fmt: skip
    before = weights.cpu()
    for i, n in enumerate(ctx):  # all weights of n queries and nh heads
        assert torch.allclose(before[:, i].sum(-1), torch.tensor(float(n * nh)), rtol=1e-3)
    new = cache.evict(weights, tables.cuda(), lens, keep, recent)
    assert new.tolist() == [48, 48, 40]
    free = manager.pool.num_free
    for i, n in enumerate(new.tolist()):
        manager.shrink(i, n)
    assert manager.pool.num_free == free + (9 - 3) + (5 - 3)
    manager.check_no_leaks()
    for layer, s in enumerate(steps):
        _, k, v, w = evict64(s.k[None], s.v[None], before[layer][None], tables, ctx, bs, keep, recent)
        assert torch.equal(cache.k[layer].cpu(), k[0]) and torch.equal(cache.v[layer].cpu(), v[0])
        assert torch.equal(weights[layer].cpu(), w[0])
        d = Step(torch.bfloat16, nh, nkv, hd, bs, new.tolist(), [1] * 3, seed=30, width=width)
        d.k, d.v, d.tables = k[0], v[0], tables
        got = pa.paged_decode_attention(d.q.cuda(), cache.k[layer], cache.v[layer], tables.cuda(),
                                        new, bs, softcap=cap)  # fmt: skip
        want, _ = attention64(d, cap)
        assert bool(((got.cpu().double() - want).abs() <= tolerance(d, want, torch.bfloat16, cap)).all())
