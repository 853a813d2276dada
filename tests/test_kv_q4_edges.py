"""KV cache held in 4 bits, at its edges: captured calls, values that must not be seen, refusals."""

from __future__ import annotations

import math

import pytest
from test_kv_q4 import DTYPES, _torch, check, expect, fill, make_cache


# ---- captured graphs -------------------------------------------------------------------------------
def _decode_case(torch, n=700, hkv=2, hq=8, hd=128):
    """A cache of two sequences, a one-row query over enough keys to be split between CTAs."""
    cache = make_cache(torch, 2, -(-n // 64), hkv, 64, hd, True, 41)
    held = fill(torch, cache, [n, n - 100], 42)
    q = torch.randn(1, hq, hd, device="cuda")
    pos = torch.tensor([n - 1], dtype=torch.int32, device="cuda")
    want = [expect(torch, q, held, [n - 1], [0], 1 / math.sqrt(hd)),
            expect(torch, q, held, [n - 101], [1], 1 / math.sqrt(hd))]
    return cache, held, q, pos, want


@pytest.mark.gpu
def test_a_captured_call_keeps_its_scratch():
    """A captured one-row call, then a call on the same stream that needs more scratch, and new
    tensors over all memory that is free: a replay gives its rows and touches nothing else."""
    torch = _torch()
    cache, held, q, pos, want = _decode_case(torch)
    side = torch.cuda.Stream()
    out = torch.empty_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        cache.attend(q, pos, 0, out=out)
    side.synchronize()
    with torch.cuda.graph(graph, stream=side):
        cache.attend(q, pos, 0, out=out)
    with torch.cuda.stream(side):
        chunk = torch.randn(200, 8, 128, device="cuda").bfloat16()
        for _ in range(2):
            cache.attend(chunk, 400, 0)
        others = [torch.full((n,), 7, dtype=torch.uint8, device="cuda")
                  for n in [64 << 20, 40 << 20, 24 << 20, 12 << 20] * 4]
    side.synchronize()
    for _ in range(3):
        out.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        check(torch, out, *want[0])
    assert all(int((t != 7).sum()) == 0 for t in others)


@pytest.mark.gpu
@pytest.mark.parametrize("order", [(1, 0), (0, 1), (1, 1, 0)])
def test_graphs_of_one_capture_stream(order):
    """Two graphs captured without a call before them, on torch's capture stream, replayed in any
    order, with eager calls between."""
    torch = _torch()
    cache, held, q, pos, want = _decode_case(torch)
    junk = torch.full((256 << 20,), 255, dtype=torch.uint8, device="cuda")
    del junk  # fresh scratch is unlikely to be zero by itself
    graphs, outs = [], []
    for slot in (0, 1):
        g, out = torch.cuda.CUDAGraph(), torch.empty_like(q)
        at = pos if slot == 0 else pos - 100
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            cache.attend(q, at, slot, out=out)
            cache.attend(q, at, slot, out=out)  # one zeroing serves both
        graphs.append((g, at))
        outs.append(out)
    for i in order:
        outs[i].fill_(math.nan)
        graphs[i][0].replay()
        check(torch, cache.attend(q, pos, 0), *want[0])
        torch.cuda.synchronize()
        check(torch, outs[i], *want[i])


@pytest.mark.gpu
def test_graphs_replayed_side_by_side():
    """Graphs captured on one stream and replayed on two at a time."""
    torch = _torch()
    cache, held, q, pos, want = _decode_case(torch, n=6000)
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in range(2)]
    for slot in (0, 1):
        g, out = torch.cuda.CUDAGraph(), torch.empty_like(q)
        at = pos if slot == 0 else pos - 100
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            for _ in range(8):
                cache.attend(q, at, slot, out=out)
        graphs.append((g, at))
        outs.append(out)
    for _ in range(10):
        for s, (g, _), out in zip(streams, graphs, outs):
            with torch.cuda.stream(s):
                out.fill_(math.nan)
                g.replay()
        torch.cuda.synchronize()
        for out, w in zip(outs, want):
            check(torch, out, *w)


# ---- values that must not be seen --------------------------------------------------------------------
# (KV heads, q heads of each, head_dim, rows, positions before them): rows of 128 or 256 on the tensor
# cores' tiles for the 16-bit types, single rows, rows packed by 2, 4 and 8 positions
CHUNKS = [(4, 8, 128, 300, 260), (8, 4, 128, 100, 0), (2, 3, 64, 400, 77), (1, 16, 64, 150, 2000),
          (2, 8, 128, 20, 100), (2, 2, 64, 9, 20), (2, 1, 128, 21, 0), (1, 4, 256, 13, 60)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hkv, rk, hd, s, past", CHUNKS)
def test_chunk_with_values_that_are_no_numbers(dtype, hkv, rk, hd, s, past):
    """NaN in a block of V at some positions of the chunk: rows that see one have NaN in its 32 dims,
    earlier rows and other dims are as ever."""
    torch = _torch()
    cache = make_cache(torch, 1, -(-(past + s) // 48), hkv, 48, hd, True, 43)
    fill(torch, cache, [past + s], 44)
    gen = torch.Generator().manual_seed(45)
    for at, dim, head in ((past + s - 2, 3, 0), (past + s // 2, 40, hkv - 1), (past + 1, hd - 1, 0)):
        x = torch.randn(1, hkv, hd, generator=gen).cuda()
        y = x.clone()
        y[0, head, dim] = math.nan
        cache.write(x, y, at, 0)
    held = [tuple(x.double() for x in cache.read(0, 0, rows=past + s))]
    q = torch.randn(s, hkv * rk, hd, generator=gen).to(getattr(torch, dtype)).cuda()
    want, tol = expect(torch, q, held, range(past, past + s), [0] * s, 1 / math.sqrt(hd))
    assert not want[0].isnan().any() and want[-1].isnan().any()
    got = cache.attend(q, past, 0)
    check(torch, got, want, tol)
    assert torch.equal(got.nan_to_num(9.0), cache.attend(q, past, 0).nan_to_num(9.0))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hkv, rk, hd, s, past", CHUNKS)
def test_chunk_whose_later_positions_are_unwritten(dtype, hkv, rk, hd, s, past):
    """The memory behind the later positions of a chunk holds whatever it held (scales that are
    infinite, NaN, or too large for f16 times a code): rows before them do not notice."""
    torch = _torch()
    cache = make_cache(torch, 1, -(-(past + s) // 48), hkv, 48, hd, True, 47)
    n = past + s // 2
    held = fill(torch, cache, [n], 48)
    q = torch.randn(s, hkv * rk, hd, generator=torch.Generator().manual_seed(49))
    q = q.to(getattr(torch, dtype)).cuda()
    rows = n - past
    want, tol = expect(torch, q[:rows], held, range(past, n), [0] * rows, 1 / math.sqrt(hd))
    check(torch, cache.attend(q, past, 0)[:rows], want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_rows_that_see_nothing_are_zero_whatever_q_holds(dtype, bad):
    """Padding rows (position -1, a slot or pages outside the cache), also those that share a tile or a
    group with rows that see keys: their q is not looked at.  Rows that see a key have no value."""
    torch = _torch()
    dt = getattr(torch, dtype)
    cache = make_cache(torch, 3, 8, 4, 64, 128, True, 51)
    held = fill(torch, cache, [400, 400, 0], 52)
    cache.pages[2] = 1000
    gen = torch.Generator().manual_seed(53)
    for rows, heads in ((4, 32), (6, 8), (300, 32)):  # single, packed, tiles (16-bit types)
        q = torch.randn(rows, heads, 128, generator=gen).to(dt).cuda()
        q[:3, 1] = bad
        q[1, :, 7] = bad
        q[rows - 1, 5, 100] = bad
        got = cache.attend(q, -3, 1)
        assert not got[:3].any()
        want, tol = expect(torch, q, held, range(-3, rows - 3), [1] * rows, 1 / math.sqrt(128))
        assert want[rows - 1, 5].isnan().all()
        check(torch, got, want, tol)
        assert not cache.attend(q, 20, 2).any()
        assert not cache.attend(q, 20, 7).any()
        pos = torch.full((rows,), -1, dtype=torch.int32, device="cuda")
        assert not cache.attend(q, pos, torch.zeros_like(pos)).any()
