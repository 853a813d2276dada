"""KV cache held in 4 bits, at its edges: captured calls, values that must not be seen, refusals."""

from __future__ import annotations

import ctypes
import gc
import math
import re
from pathlib import Path

import pytest
from test_kv_q4 import DTYPES, _c_cache, _torch, check, expect, fill, make_cache

from ggmlc_b200 import kv_q4


# ---- what a kernel may read that starts before the one that writes it has ended -----------------------
@pytest.mark.parametrize("source", ["k_attn_q4.cu", "k_attn_q4_tc.cu", "k_kv_q4.cu"])
def test_no_read_only_loads(source):
    """The cache's kernels start while the kernel before them may still run (programmatic dependent
    launch); the read-only path is for memory that nobody writes while the kernel lives."""
    code = (Path(kv_q4.__file__).parent / "csrc" / source).read_text()
    code = re.sub(r"//[^\n]*", "", code)
    assert "launch_pdl(" in code and not re.search(r"__ldg\b|ld\.global\.nc|__restrict__", code)


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


# ---- the engine's prefill form ----------------------------------------------------------------------
class Prefill:
    """gb_kv_q4_attend_prefill over a torch class's cache: f32 rows, the position read on the device."""

    def __init__(self, torch, cache, hq, rows):
        self.lib, p = kv_q4._lib, cache.pages
        self.cache = cache
        self.c = kv_q4._Cache(cache.k.data_ptr(), cache.v.data_ptr(), cache.k.shape[0],
                              cache.page_len, cache.n_kv_heads, cache.head_dim,
                              p.data_ptr() if p is not None else None,
                              p.shape[0] if p is not None else 0, p.shape[1] if p is not None else 0)
        need = self.lib.gb_kv_q4_attend_workspace_bytes(ctypes.addressof(self.c), rows, hq)
        self.work = torch.zeros(need, dtype=torch.uint8, device="cuda")
        self.pos = torch.zeros(1, dtype=torch.int64, device="cuda")
        self.hq, self.rows = hq, rows

    def __call__(self, torch, q, out, slot=0, max_kv=0):
        rc = self.lib.gb_kv_q4_attend_prefill(
            ctypes.addressof(self.c), self.rows, self.pos.data_ptr(), slot, q.data_ptr(),
            q.stride(0), q.stride(1), self.hq, max_kv, 1 / math.sqrt(self.cache.head_dim),
            out.data_ptr(), self.work.data_ptr(), self.work.numel(),
            torch.cuda.current_stream().cuda_stream)
        assert rc == 0, self.lib.gb_last_error()


def expect_prefill(torch, q, held, pos, slot):
    """f64 attention and the bound of each element where q, K and V are rounded to f16 (2^-11 of each)
    and the rest is f32: an error e in a score changes a probability by the factor exp(e), and e is at
    most scale times the sum of |q| |k| (2^-11 + 2^-11), with 2^-24 of the row's largest |q| for the
    elements that f16 does not hold beside it."""
    hd, hkv = q.shape[2], held[slot][0].shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    for r in range(q.shape[0]):
        k, v = (x[:pos + r + 1] for x in held[slot])
        qr = q[r].double().reshape(hkv, -1, hd)
        w = torch.softmax(torch.einsum("hgd,thd->hgt", qr, k) / math.sqrt(hd), -1)
        out[r] = torch.einsum("hgt,thd->hgd", w, v).reshape(-1, hd)
        off = qr.abs() * 2.0**-10 + qr.abs().amax(-1, keepdim=True) * 2.0**-24
        e = torch.einsum("hgd,thd->hgt", off, k.abs()).amax(-1) / math.sqrt(hd)
        absolute = torch.einsum("hgt,thd->hgd", w, v.abs()).reshape(-1, hd)
        tol[r] = absolute * (2.0**-11 + 2.0**-18 + 2 * e).reshape(-1, 1) + 1e-12
    return out, tol


@pytest.mark.gpu
@pytest.mark.parametrize("hkv, rk, hd", [(8, 4, 128), (8, 2, 64), (3, 3, 64), (2, 10, 128)])
@pytest.mark.parametrize("s, past, capacity", [(512, 0, 512), (500, 0, 8192), (300, 333, 700),
                                               (300, 333, 40000), (129, 2000, 4096), (512, 100, 640)])
def test_prefill_form_on_tiles(hkv, rk, hd, s, past, capacity):
    """Windows as wide as the chunk and far wider (the plan is made for the window, its runs of key
    tiles are cut by the position, which only the device knows)."""
    torch = _torch()
    cache = make_cache(torch, 2, -(-capacity // 64), hkv, 64, hd, True, 61)
    held = fill(torch, cache, [0, past + s], 62)
    q = torch.randn(s, hkv * rk, hd, generator=torch.Generator().manual_seed(63)).cuda()
    call, out = Prefill(torch, cache, hkv * rk, s), torch.empty_like(q)
    call.pos.fill_(past)
    call(torch, q, out, slot=1)
    want, tol = expect_prefill(torch, q, held, past, 1)
    check(torch, out, want, tol)
    # independent errors: 2^-11 / sqrt(3) of V, and as much of q and K each times the spread of a score
    # (1.1 here, keys of uneven channels up to 1.6), less than 1e-3 together; a tile left out or taken
    # twice would show as some percent
    err = float((out - want).norm() / want.norm())
    assert err < 2e-3
    # by rows, f32 stays below 1e-5: the tiles were what ran
    assert err > 3e-5


@pytest.mark.gpu
@pytest.mark.parametrize("contiguous", [False, True])
def test_prefill_form_in_a_graph_reads_the_position_anew(contiguous):
    """One captured call over a window of 2048 replayed at several positions."""
    torch = _torch()
    hkv, rk, hd, s, cap = 8, 4, 64, 200, 2048
    cache = make_cache(torch, 2, 1 if contiguous else cap // 64, hkv, cap if contiguous else 64, hd,
                       not contiguous, 65)
    held = fill(torch, cache, [0, cap], 66)
    q = torch.randn(s, hkv * rk, hd, generator=torch.Generator().manual_seed(67)).cuda()
    call, out = Prefill(torch, cache, hkv * rk, s), torch.empty_like(q)
    call(torch, q, out, slot=1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(torch, q, out, slot=1)
    for past in (0, 1, 120, 1000, cap - s, 0):
        call.pos.fill_(past)
        out.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        check(torch, out, *expect_prefill(torch, q, held, past, 1))
    eager = torch.empty_like(q)
    call(torch, q, eager, slot=1)
    assert torch.equal(eager, out)


def test_prefill_form_refusals():
    c, wide, p = _c_cache(kv_q4), _c_cache(kv_q4, head_dim=96), 1 << 23
    L = kv_q4._lib

    def refused(word, cache=c, n=2, step=p, q=p, row=128, hq=2, o=p, work=p, size=1 << 30):
        rc = L.gb_kv_q4_attend_prefill(ctypes.addressof(cache), n, step, 0, q, row, 64, hq, 0, 1.0, o,
                                       work, size, None)
        assert rc == -1 and word in L.gb_last_error().decode(), L.gb_last_error()

    refused("rows", n=-1)
    refused("multiple", hq=3)
    refused("strides", row=-1)
    refused("NULL", q=None)
    refused("NULL", o=None)
    refused("head_dim", cache=wide)
    refused("work", work=None)
    refused("work", work=p + 16)


# ---- a wait that runs out ----------------------------------------------------------------------------
@pytest.fixture
def no_waiting():
    """Waits inside the chunk kernel count as run out."""
    torch = _torch()
    assert kv_q4.error() == 0  # of all calls before, in whatever test
    kv_q4._lib.gb_kv_q4_expire_waits(1)
    try:
        yield
    finally:
        kv_q4._lib.gb_kv_q4_expire_waits(0)
        torch.cuda.synchronize()
        kv_q4.clear_error()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("s, past", [(512, 0), (200, 3000)])  # whole blocks; runs of key tiles and a join
def test_a_wait_that_runs_out_shows(no_waiting, dtype, s, past):
    """Rows come out NaN, never stale, the error word is set, and the next call is as ever."""
    torch = _torch()
    cache = make_cache(torch, 1, -(-(past + s) // 64), 8, 64, 128, True, 71)
    held = fill(torch, cache, [past + s], 72)
    q = torch.randn(s, 32, 128, generator=torch.Generator().manual_seed(73))
    q = q.to(getattr(torch, dtype)).cuda()
    want, tol = expect(torch, q, held, range(past, past + s), [0] * s, 1 / math.sqrt(128))
    kv_q4._lib.gb_kv_q4_expire_waits(0)
    check(torch, cache.attend(q, past, 0), want, tol)  # leaves good partials in the scratch
    assert kv_q4.error() == 0
    kv_q4._lib.gb_kv_q4_expire_waits(1)
    out = torch.zeros_like(q)
    cache.attend(q, past, 0, out=out)
    assert kv_q4.error() != 0
    assert out.isnan().all()
    kv_q4._lib.gb_kv_q4_expire_waits(0)
    kv_q4.clear_error()
    check(torch, cache.attend(q, past, 0), want, tol)
    assert kv_q4.error() == 0


# ---- scratch -------------------------------------------------------------------------------------------
@pytest.mark.gpu
def test_handles_share_the_scratch_of_a_stream():
    """A handle a layer, chunks and single rows: no more scratch than one handle holds; none is left
    when the handles are gone."""
    torch = _torch()
    gc.collect()
    none = torch.cuda.memory_allocated()
    caches = [make_cache(torch, 1, 40, 8, 64, 128, True, 81 + i) for i in range(8)]
    held = [fill(torch, c, [2500], 90 + i) for i, c in enumerate(caches)]
    q = torch.randn(100, 32, 128, device="cuda").bfloat16()
    before = torch.cuda.memory_allocated()
    outs = [caches[0].attend(q, 2400, 0)]
    one = torch.cuda.memory_allocated() - before
    assert 0 < one < 48 << 20
    outs += [c.attend(q, 2400, 0) for c in caches[1:]]
    rows = [c.attend(q[:1], 2399, 0) for c in caches]
    assert torch.cuda.memory_allocated() - before < one + 17 * outs[0].numel() * 2
    for h, o, r in zip(held, outs, rows):
        check(torch, o, *expect(torch, q, h, range(2400, 2500), [0] * 100, 1 / math.sqrt(128)))
        check(torch, r, *expect(torch, q[:1], h, [2399], [0], 1 / math.sqrt(128)))
    del caches, held, q, outs, rows, h, o, r
    gc.collect()
    assert torch.cuda.memory_allocated() <= none + 64


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_scratch_is_what_a_call_can_use(hd):
    """Single rows, calls with a position or slot each, and head_dim 256 never reach the tiles."""
    torch = _torch()
    c = _c_cache(kv_q4, head_dim=hd)
    need = lambda n: kv_q4._lib.gb_kv_q4_attend_workspace_bytes(ctypes.addressof(c), n, 4)
    assert (need(2) > need(1)) == (hd < 256) and need(1) < 20 << 20
    cache = make_cache(torch, 2, 8, 2, 64, hd, True, 95)
    held = fill(torch, cache, [500, 300], 96)
    q = torch.randn(2, 4, hd, device="cuda")
    pos = torch.tensor([499, 299], dtype=torch.int32, device="cuda")
    slot = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    work = torch.zeros(need(1), dtype=torch.uint8, device="cuda")
    out = torch.empty_like(q)
    c = kv_q4._Cache(cache.k.data_ptr(), cache.v.data_ptr(), cache.k.shape[0], 64, 2, hd,
                     cache.pages.data_ptr(), *cache.pages.shape)
    r = kv_q4._Rows(2, pos.data_ptr(), 0, slot.data_ptr(), 0)

    def call(size):
        return kv_q4._lib.gb_kv_q4_attend(
            ctypes.addressof(c), ctypes.addressof(r), 0, q.data_ptr(), q.stride(0), q.stride(1), 4, 0,
            1 / math.sqrt(hd), out.data_ptr(), work.data_ptr(), size,
            torch.cuda.current_stream().cuda_stream)

    assert call(need(1) - 1) == -1 and "work" in kv_q4._lib.gb_last_error().decode()
    assert call(need(1)) == 0
    check(torch, out, *expect(torch, q, held, [499, 299], [0, 1], 1 / math.sqrt(hd)))


# ---- refusals ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("scale", [math.nan, math.inf, -math.inf])
def test_a_scale_that_is_no_number_is_refused(scale):
    """(It came out as a scale too small to tell scores apart: the mean of V.)"""
    c, p, L = _c_cache(kv_q4), 1 << 23, kv_q4._lib
    r = kv_q4._Rows(1, None, 0, None, 0)
    assert L.gb_kv_q4_attend(ctypes.addressof(c), ctypes.addressof(r), 0, p, 128, 64, 2, 0, scale, p, p,
                             1 << 30, None) == -1
    assert "scale" in L.gb_last_error().decode()
    assert L.gb_kv_q4_attend_prefill(ctypes.addressof(c), 1, p, 0, p, 128, 64, 2, 0, scale, p, p, 1 << 30,
                                     None) == -1
    assert "scale" in L.gb_last_error().decode()


@pytest.mark.parametrize("per_slot, ok", [((2**31 - 1) // 64, False), ((2**31 - 4096) // 64 + 1, False),
                                          ((2**31 - 4097) // 64, True)])
def test_a_capacity_near_two_to_the_31(per_slot, ok):
    """Positions are ints in the kernels, and tiles of keys run past a sequence's end: the last 4096
    below 2^31 are refused (page tables can repeat pages, so no memory stands in the way)."""
    c, L = _c_cache(kv_q4, pages_per_slot=per_slot), kv_q4._lib
    none = kv_q4._Rows(0, None, 0, None, 0)  # no rows: nothing is launched
    rc = L.gb_kv_q4_read(ctypes.addressof(c), ctypes.addressof(none), 0, None, None, None)
    assert rc == (0 if ok else -1), L.gb_last_error()
    assert ok or "2^31" in L.gb_last_error().decode()
