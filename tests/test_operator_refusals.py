"""What the operators beside plain causal attention refuse, on the host and at the C boundary, and
their host helpers. Runs without a GPU: CPU tensors and fake pointers never reach a launch."""

from __future__ import annotations

import ctypes

import pytest
import torch

from engine.kernels import _native
from engine.kernels import paged_attention as pa
from engine.runtime.block_manager import BlockManager
from engine.runtime.paged_cache import evict_tokens, evict_workspace_bytes, step_key_ranges

P = 1 << 20  # a 16-byte aligned address that nothing reads


def decode_args(**over):
    a = {"out": P, "dt": 2, "osb": 1024, "osh": 128, "q": P, "qsb": 1024, "qsh": 128, "k": P, "v": P,
         "kdt": 2, "kss": 256, "ksh": 128, "slots": 64, "tables": P, "ts": 4, "w": 4, "ctx": P,
         "b": 2, "nh": 8, "nkv": 2, "hd": 128, "bs": 16, "scale": 0.1, "wgs": 1, "ws": None,
         "wsb": 0, "rows": None, "nrows": 2, "cap": 5.0, "slopes": None, "ranges": None, "rs": 0,
         "lse": None, "stream": None}  # fmt: skip
    assert set(over) <= set(a)
    a.update(over)
    return list(a.values())


@pytest.mark.parametrize(
    "over,code",
    [({"cap": -1.0}, -2), ({"cap": float("nan")}, -2), ({"cap": float("inf")}, -2),
     ({"cap": 1e-35}, -2), ({"ranges": P, "rs": -2}, -2), ({"scale": 0.0}, -2),
     ({"scale": float("nan")}, -2), ({"hd": 96}, -2), ({"nh": 7}, -2), ({"kdt": 5}, -1),
     ({"dt": 1}, -1), ({"k": None}, -5), ({"ctx": None}, -5), ({"q": P + 4}, -3),
     ({"wgs": 4}, -4), ({"nrows": -1}, -2), ({"b": 0}, 0)],
)  # fmt: skip
def test_decode_entry(over, code):
    assert _native.lib().pkv_paged_decode_mod(*decode_args(**over)) == code


def prefill_args(**over):
    a = {"out": P, "dt": 2, "ost": 1024, "osh": 128, "q": P, "qst": 1024, "qsh": 128, "k": P, "v": P,
         "kdt": 2, "kss": 256, "ksh": 128, "slots": 64, "tables": P, "ts": 4, "w": 4, "ctx": P,
         "cu": P, "n": 2, "maxq": 8, "nh": 8, "nkv": 2, "hd": 128, "bs": 16, "scale": 0.1,
         "ws": None, "wsb": 0, "rows": None, "rlen": 0, "nrows": 16, "cap": 5.0, "slopes": None,
         "ranges": None, "rs": 0, "lse": None, "stream": None}  # fmt: skip
    assert set(over) <= set(a)
    a.update(over)
    return list(a.values())


@pytest.mark.parametrize(
    "over,code",
    [({"cap": -1.0}, -2), ({"cap": 1001.0}, -2), ({"ranges": P, "rs": -1}, -2),
     ({"scale": -1.0}, -2), ({"hd": 80}, -2), ({"kdt": 3}, -1), ({"cu": None}, -5),
     ({"out": P + 8}, -3), ({"wsb": 64}, -4), ({"nrows": -1}, -2), ({"n": 0}, 0), ({"maxq": 0}, 0)],
)  # fmt: skip
def test_prefill_entry(over, code):
    assert _native.lib().pkv_paged_prefill_mod(*prefill_args(**over)) == code


def weights_args(**over):
    a = {"w": P, "wst": 64, "wn": 2, "wr": None, "decay": 1.0, "q": P, "qst": 1024, "qsh": 128,
         "k": P, "kdt": 2, "kss": 256, "ksh": 128, "slots": 64, "tables": P, "ts": 4, "width": 4,
         "ctx": P, "cu": None, "n": 2, "maxq": 1, "lse": P, "nh": 8, "nkv": 2, "hd": 128, "bs": 16,
         "scale": 0.1, "cap": 0.0, "slopes": None, "ranges": None, "rs": 0, "work": None,
         "bytes": 0, "stream": None}  # fmt: skip
    assert set(over) <= set(a)
    a.update(over)
    return list(a.values())


@pytest.mark.parametrize(
    "over,code",
    [({"decay": -0.5}, -2), ({"decay": float("nan")}, -2), ({"decay": float("inf")}, -2),
     ({"wn": 1}, -2), ({"cap": -1.0}, -2), ({"hd": 48}, -2), ({"nkv": 3}, -2), ({"kdt": 9}, -1),
     ({"lse": None}, -5), ({"w": None}, -5), ({"q": P + 2}, -3), ({"kss": 100}, -3),
     ({"width": 1 << 27, "bs": 16}, -2), ({"slots": 1 << 31}, -2),
     ({"cu": P, "maxq": -1}, -2), ({"cu": P, "maxq": 5}, -4),
     ({"cu": P, "maxq": 5, "work": P, "bytes": 2 * 2 * 64 * 4 - 1}, -4), ({"bytes": -1}, -4),
     ({"work": P + 2, "bytes": 64}, -3), ({"n": 0}, 0), ({"width": 0}, 0)],
)  # fmt: skip
def test_weights_entry(over, code):
    assert _native.lib().pkv_attention_weights(*weights_args(**over)) == code


def evict_args(**over):
    a = {"k": P, "v": P, "ls": 1 << 16, "layers": 2, "row": 256, "slots": 64, "w": P, "wl": 128,
         "ws": 64, "wn": 2, "wr": None, "tables": P, "ts": 4, "width": 4, "bs": 16, "ctx": P,
         "b": 2, "keep": 20, "recent": 4, "out": P, "work": P, "bytes": 1 << 20, "stream": None}  # fmt: skip
    assert set(over) <= set(a)
    a.update(over)
    return list(a.values())


@pytest.mark.parametrize(
    "over,code",
    [({"recent": 21}, -2), ({"recent": -1}, -2), ({"keep": -1, "recent": -1}, -2), ({"row": 24}, -3),
     ({"row": 0}, -2), ({"k": P + 8}, -3), ({"ls": 8}, -3), ({"wn": 1}, -2), ({"bytes": 16}, -4),
     ({"work": None}, -5), ({"out": None}, -5), ({"slots": 1 << 31}, -2), ({"layers": 1 << 17}, -2),
     ({"b": 0}, 0), ({"layers": 0}, 0)],
)  # fmt: skip
def test_evict_entry(over, code):
    assert _native.lib().pkv_evict(*evict_args(**over)) == code


def test_workspace_queries():
    lib = _native.lib()
    assert lib.pkv_evict_workspace_bytes(2, 3, 10, 16, 50) == 256 + 2 * 3 * 50 * 4
    # no more moves than a table holds tokens
    assert lib.pkv_evict_workspace_bytes(1, 1, 2, 16, 1 << 30) == 256 + 32 * 4
    assert lib.pkv_evict_workspace_bytes(1, 1, 2, 0, 4) == -2
    assert evict_workspace_bytes(1, 1, 2, 16, 1 << 40) == 256 + 32 * 4
    with pytest.raises(ValueError):
        evict_workspace_bytes(1, 1, 2, 16, -1)
    assert lib.pkv_attention_weights_workspace_bytes(32, 8, 3, 4, 10, 16) == 0
    assert lib.pkv_attention_weights_workspace_bytes(32, 8, 3, 5, 10, 16) == 3 * 8 * 160 * 4
    assert lib.pkv_attention_weights_workspace_bytes(32, 5, 3, 5, 10, 16) == -2
    with pytest.raises(ValueError):
        pa.attention_weights_workspace_bytes(32, 8, -1, 5, 10, 16)
    assert lib.pkv_decode_mod_default_workgroups(2, 96, 24, 8, 8, 32, 16) == -2
    assert lib.pkv_decode_mod_default_workgroups(7, 128, 24, 8, 8, 32, 16) == -1
    assert ctypes.sizeof(ctypes.c_int64) == 8


def test_score_arguments():
    """The host's checks of the score arguments (as the wrappers make them, on any device)."""
    q = torch.zeros(5, 8, 64)
    cpu = q.device

    def mod(**x):
        args = {"softcap": None, "alibi_slopes": None, "key_ranges": None, "lse": None} | x
        return pa._score_mod("op", cpu, q, 5, **args)

    assert mod() is None
    assert mod(softcap=0.0) == (0.0, None, None, 0, None)
    for bad in (-1.0, float("nan"), float("inf"), 1e-31, 1000.5):
        with pytest.raises(ValueError, match="softcap"):
            mod(softcap=bad)
    for bad in (torch.zeros(7), torch.zeros(8, dtype=torch.float64), torch.zeros(16)[::2],
                torch.zeros(8, device="meta")):  # fmt: skip
        with pytest.raises(ValueError, match="alibi_slopes"):
            mod(alibi_slopes=bad)
    with pytest.raises(TypeError, match="key_ranges"):
        mod(key_ranges=torch.zeros(5, 2, dtype=torch.int64))
    for shape in ((4, 2), (5, 3), (5,)):
        with pytest.raises(ValueError, match="key_ranges"):
            mod(key_ranges=torch.zeros(shape, dtype=torch.int32))
    with pytest.raises(ValueError, match="key_ranges"):
        mod(key_ranges=torch.zeros(2, 5, dtype=torch.int32).T)
    for bad in (torch.zeros(5, 7), torch.zeros(4, 8), torch.zeros(8, 5).T,
                torch.zeros(5, 8, dtype=torch.float16)):  # fmt: skip
        with pytest.raises(ValueError, match="lse"):
            mod(lse=bad)


def test_no_cpu_path():
    q, k = torch.zeros(1, 2, 64), torch.zeros(16, 2, 64)
    tables, ctx = torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        pa.paged_decode_attention(q, k, k, tables, ctx, 16, softcap=5.0)
    with pytest.raises(ValueError, match="GPU"):
        pa.paged_attention_weights(torch.zeros(1, 16), q, k, tables, ctx, 16, torch.zeros(1, 2))
    with pytest.raises(ValueError, match="GPU"):
        evict_tokens(k, k.clone(), torch.zeros(1, 16), tables, ctx, 16, 4, 1)


def test_step_key_ranges():
    ctx, new = [9, 5, 12], [4, 1, 12]
    got = step_key_ranges(ctx, new, "cpu")
    pos = [(i, p) for i in range(3) for p in range(ctx[i] - new[i], ctx[i])]
    assert got.dtype == torch.int32 and got.tolist() == [[0, p + 1] for _, p in pos]
    assert step_key_ranges(ctx, new, "cpu", window=3).tolist() == [[max(0, p - 2), p + 1] for _, p in pos]
    starts = [[0, 6], [], [0, 1, 7]]
    docs = step_key_ranges(ctx, new, "cpu", doc_starts=starts)
    for (i, p), (lo, hi) in zip(pos, docs.tolist(), strict=True):
        assert (lo, hi) == (max([x for x in starts[i] if x <= p], default=0), p + 1)
    both = step_key_ranges(ctx, new, "cpu", window=4, doc_starts=starts, prefix_lens=[7, 0, 20])
    for (i, p), (lo, hi) in zip(pos, both.tolist(), strict=True):
        first = max(max([x for x in starts[i] if x <= p], default=0), p - 3, 0)
        n = min([7, 0, 20][i], ctx[i])
        assert (lo, hi) == (first, n if p < n else p + 1)
    assert step_key_ranges([], [], "cpu").shape == (0, 2)
    assert step_key_ranges([4], [0], "cpu").shape == (0, 2)
    for bad in ({"window": 0}, {"prefix_lens": [1]}, {"doc_starts": [[0]]}):
        with pytest.raises(ValueError):
            step_key_ranges(ctx, new, "cpu", **bad)
    with pytest.raises(ValueError):
        step_key_ranges([3], [4], "cpu")
    with pytest.raises(ValueError):
        step_key_ranges([3, 4], [1], "cpu")
    with pytest.raises(ValueError):
        step_key_ranges([9], [9], "cpu", doc_starts=[[4, 2]])


def test_shrink():
    m = BlockManager(10, 16)
    m.grow(1, 70)
    table = list(m.tables[1])
    m.fork(1, 2, 70)
    assert m.shrink(1, 33) == table[3:]
    assert m.tables[1] == table[:3] and m.pool.num_free == 5  # the fork still holds the others
    m.check_no_leaks()
    assert m.shrink(2, 48) == table[3:] and m.pool.num_free == 7
    assert m.shrink(2, 100) == [] and m.shrink(9, 5) == []
    assert m.shrink(1, 0) == table[:3]
    with pytest.raises(ValueError):
        m.shrink(1, -1)
    m.check_no_leaks()
