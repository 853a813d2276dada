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
