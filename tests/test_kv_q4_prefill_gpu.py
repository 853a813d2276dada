"""The engine over a 4-bit KV cache with prompts long enough for the attention's tensor-core tiles
(the fixtures' prompts are not): a synthesized two-layer Llama with 16 heads on 8, against the CPU
oracle with the same quantisation in its cache, at the bar of test_kv_q4_engine_gpu.py."""

from __future__ import annotations

import numpy as np
import pytest
from test_kv_q4_engine_gpu import COS_MIN, Q4Oracle, _step, cos

from conftest import cuda_available

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not cuda_available(), reason="needs a CUDA device")]

VOCAB, TOKENS = 512, 400


@pytest.fixture(scope="module", params=[64, 128])
def model(request, tmp_path_factory):
    """The model's file, a prompt, and the oracle's logits of all its rows."""
    from ggmlc_b200 import synth

    hd = request.param
    path = tmp_path_factory.mktemp("synth") / f"llama_hd{hd}.gguf"
    synth.synth_llama(path, synth.LlamaShape(2, 512, 16, 8, hd, 1024, VOCAB, 10000.0), synth.Q8_0)
    prompt = np.random.default_rng(hd).integers(1, VOCAB, TOKENS).astype(np.int32)
    M = Q4Oracle(path)
    M.init_kv_cache(TOKENS + 8)
    rows = M.forward(prompt, pos=0).reshape(-1, VOCAB)
    step = M.forward(np.array([int(rows[-1].argmax())]), pos=TOKENS).ravel()
    return path, prompt, rows, step


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("chunk", [TOKENS, TOKENS // 2])
@pytest.mark.parametrize("window", [512, 8192])
def test_long_prompts_follow_the_oracle(model, window, chunk, graph):
    """A chunk of 400 or two of 200 (one program, run at both positions), in a window that fits and in
    one whose plan cuts the keys into runs.  200 rows of these heads: 16.6 us by rows, 15 by tiles in
    a window of 512, by the launcher's rule; 67 and 38 in one of 8192."""
    from ggmlc_b200.runner import load

    path, prompt, rows, step = model
    r = load(str(path), device="cuda")
    r.executor.set_enable_cuda_graph(graph)
    r.init_kv_cache(window, "q4_0")
    got = np.concatenate([_step(r, prompt[i:i + chunk], i, VOCAB) for i in range(0, TOKENS, chunk)])
    assert cos(got, rows) >= COS_MIN
    assert min(cos(a, b) for a, b in zip(got[::37], rows[::37])) >= COS_MIN - 0.002
    token = int(rows[-1].argmax())
    assert cos(_step(r, [token], TOKENS, VOCAB), step) >= COS_MIN


def test_a_wait_that_runs_out_is_raised(model):
    """Reading the outputs of a prefill whose attention gave up raises once; the next prefill is as
    ever."""
    from ggmlc_b200 import kv_q4
    from ggmlc_b200.runner import load

    path, prompt, rows, _ = model
    r = load(str(path), device="cuda")
    r.executor.set_enable_cuda_graph(False)
    r.init_kv_cache(512, "q4_0")
    try:
        kv_q4._lib.gb_kv_q4_expire_waits(1)
        with pytest.raises(RuntimeError, match="4-bit KV cache"):
            _step(r, prompt, 0, VOCAB)
    finally:
        kv_q4._lib.gb_kv_q4_expire_waits(0)
        kv_q4.clear_error()
    assert cos(_step(r, prompt, 0, VOCAB), rows) >= COS_MIN
    assert kv_q4.error() == 0
