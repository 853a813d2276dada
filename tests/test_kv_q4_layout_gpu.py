"""Laying out the engine's KV cache: refusals and failures, and the type that is held."""

from __future__ import annotations

import numpy as np
import pytest
from test_kv_q4_engine_gpu import _step

from conftest import GOLDEN, cuda_available

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not cuda_available(), reason="needs a CUDA device")]

MODEL = "tiny_llama_q8_0"


def _executor():
    from ggmlc_b200._runtime import ModelExecutor, ModelLoader

    g = ModelLoader.load_from_file(str(GOLDEN / f"{MODEL}.gguf"))
    return g, ModelExecutor(g, "cuda")


def _paged_row(g, ex, prompt):
    """Last logits of a prompt prefilled into slot 0."""
    ex.set_logits_last_only(True)
    ex.prepare({"s": len(prompt), "pos": 0, "slot": 0, **{s: len(prompt) for s in g.symbol_table}})
    ex.set_input_by_id(g.inputs[0], np.asarray(prompt, np.int32))
    ex.run()
    return np.array(ex.get_output_array(g.outputs[0])).ravel()


def test_a_refused_layout_leaves_the_cache_in_place():
    """A paged f16 cache whose pages are too small for 4 bits: asking for 4 bits is refused, and the
    cache, its slot and its pages are as before."""
    prompt = [int(t) for t in np.load(GOLDEN / f"{MODEL}.npz")["prompt"]][:20]
    g, ex = _executor()
    ex.set_tokens_per_page(8)
    ex.init_paged_kv_cache(2, 64)
    ex.paged_kv_alloc_slot(0)
    ex.paged_kv_ensure_tokens(0, 40)
    before, bytes_ = _paged_row(g, ex, prompt), ex.get_paged_active_vram_bytes()
    ex.set_kv_cache_type("q4_0")
    with pytest.raises(RuntimeError, match="tokens_per_page"):
        ex.init_paged_kv_cache(2, 64)
    assert ex.is_paged_kv_cache_enabled() and ex.has_kv_cache()
    assert ex.get_paged_active_vram_bytes() == bytes_
    assert np.array_equal(_paged_row(g, ex, prompt), before)


def test_pages_too_small_for_the_held_type_are_refused():
    """set_tokens_per_page lays an idle pool out again; pages of 8 positions of 4 bits are refused, and
    the pool of 16 stays."""
    _, ex = _executor()
    ex.set_kv_cache_type("q4_0")
    ex.set_tokens_per_page(16)
    ex.init_paged_kv_cache(2, 64)
    with pytest.raises(RuntimeError, match="tokens_per_page"):
        ex.set_tokens_per_page(8)
    ex.paged_kv_alloc_slot(0)
    ex.paged_kv_ensure_tokens(0, 16)
    page = ex.get_paged_active_vram_bytes()
    ex.paged_kv_ensure_tokens(0, 17)
    assert 0 < page == ex.get_paged_active_vram_bytes() - page


@pytest.mark.parametrize("kv_type", ["f16", "q4_0"])
def test_a_layout_that_does_not_fit_leaves_nothing_behind(kv_type):
    """More positions than any memory holds: an error, and the next layout runs as a first one does
    (the decode chain of the f16 cache among it)."""
    from ggmlc_b200.runner import load

    gold = np.load(GOLDEN / f"{MODEL}.npz")
    V, prompt = gold["full_logits"].shape[1], [int(t) for t in gold["prompt"]][:9]
    rows = []
    for fail in (False, True):
        r = load(str(GOLDEN / f"{MODEL}.gguf"), device="cuda")
        if fail:
            r.executor.set_kv_cache_type(kv_type)
            with pytest.raises(RuntimeError):
                r.init_kv_cache(1 << 40)
            assert not r.executor.has_kv_cache()
            r.executor.set_kv_cache_type("f16")
        r.init_kv_cache(64)
        _step(r, prompt[:8], 0, V)
        rows.append(_step(r, prompt[8:], 8, V))
        rows.append(r.executor.launches_per_run())
    assert np.array_equal(rows[0], rows[2]) and rows[1] == rows[3]


def test_the_type_is_that_of_the_cache_that_is_held():
    """A runner that goes from f16 to 4 bits and back computes what fresh runners of each type do."""
    from ggmlc_b200.runner import load

    gold = np.load(GOLDEN / f"{MODEL}.npz")
    V, prompt = gold["full_logits"].shape[1], [int(t) for t in gold["prompt"]]
    fresh = {}
    for kv_type in ("f16", "q4_0"):
        r = load(str(GOLDEN / f"{MODEL}.gguf"), device="cuda")
        r.init_kv_cache(64, kv_type)
        fresh[kv_type] = _step(r, prompt, 0, V)
    assert not np.array_equal(fresh["f16"], fresh["q4_0"])
    r = load(str(GOLDEN / f"{MODEL}.gguf"), device="cuda")
    assert r.executor.kv_cache_type() == "f16"
    r.executor.set_kv_cache_type("q4_0")
    assert r.executor.kv_cache_type() == "q4_0"  # nothing is held yet
    r.executor.set_kv_cache_type("f16")
    r.init_kv_cache(64)
    for kv_type, before in (("q4_0", "f16"), ("f16", "q4_0"), ("q4_0", "f16")):
        r.executor.set_kv_cache_type(kv_type)
        assert r.executor.kv_cache_type() == before
        r.init_kv_cache(64, kv_type)
        assert r.executor.kv_cache_type() == kv_type
        assert np.array_equal(_step(r, prompt, 0, V), fresh[kv_type])
        r.init_kv_cache(64, kv_type)  # the same type: kept, with what it holds
        assert r.executor.has_kv_cache()


def test_the_type_of_a_paged_cache():
    """init_kv_cache does not replace a paged cache by a contiguous one of another type, and a pool that
    set_tokens_per_page lays out again keeps its type."""
    _, ex = _executor()
    ex.set_tokens_per_page(16)
    ex.init_paged_kv_cache(2, 64)
    ex.set_kv_cache_type("q4_0")
    with pytest.raises(RuntimeError, match="paged"):
        ex.init_kv_cache(64)
    ex.set_tokens_per_page(32)
    assert ex.is_paged_kv_cache_enabled() and ex.kv_cache_type() == "f16"
    ex.init_paged_kv_cache(2, 64)
    assert ex.kv_cache_type() == "q4_0"
    ex.init_kv_cache(64)  # the type that is held: nothing to do, as ever
    assert ex.is_paged_kv_cache_enabled()
