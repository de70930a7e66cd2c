"""Cached prefix pages and a change of the sliding window: K/V that a step wrote
under another window is refused at admission, K/V of the same one is shared."""
import ctypes as C

import numpy as np
import pytest

from mini_serve_rs_b200 import engine as E
from oracle.qwen_ref import random_weights
from tests.gpu_util import need_gpu
from tests.test_gpu_engine_window import SHAPES

pytestmark = pytest.mark.gpu
CFG = SHAPES["qwen3"]


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    need_gpu()


@pytest.fixture
def eng():
    e = E.Engine(CFG, pool_blocks=64, max_seqs=8, max_tokens_per_step=512, max_blocks_per_seq=16, dtype=E.MS_DTYPE_F32)
    e.load_weights(random_weights(CFG, 6, norm_std=0.1))
    yield e
    e.close()


def toks(n, seed=0):
    return np.random.default_rng(seed).integers(0, CFG.vocab_size, n).tolist()


def run(eng, sid, prompt, blocks, cached=0, budget=0):
    eng.admit(sid, prompt, blocks, num_cached=cached)
    for _ in range(20):
        _, flags = eng.step([sid], flags=E.MS_STEP_KEEP_LOGITS, token_budget=budget)
        if flags[0] & E.MS_FLAG_PREFILLED:
            return eng.logits(1)[0].copy()
    raise AssertionError("prompt not done")


def refused(eng, prompt, blocks, cached):
    with pytest.raises(E.EngineError, match="window"):
        eng.admit(99, prompt, blocks, num_cached=cached)
    assert eng.is_healthy()


def test_pages_of_another_window_are_refused(eng):
    prompt = toks(100)
    pages = E.Pages(64, 16, max_chunks=32)
    blocks, cached = pages.admit(1, prompt)
    assert cached == 0
    full = run(eng, 1, prompt, blocks)
    pages.publish(1, prompt)
    longer = prompt[:96] + toks(20, 1)
    b2, c2 = pages.admit(2, longer)
    assert c2 == 96
    eng.set_window(30, 2, 0)
    refused(eng, longer, b2, c2)
    # on pages of its own the prompt is computed under the window, and shared from then on
    own = list(range(40, 48))
    want = run(eng, 2, longer, own)
    again = run(eng, 3, longer, own[:6] + [50, 51], cached=96)
    assert np.abs(want - again).max() <= 1e-4
    for other in ((30, 0, 0), (31, 2, 0), (30, 2, 1), (0, 0, 0)):
        eng.set_window(*other)
        refused(eng, longer, own, 96)
    # back to no window: the first sequence's pages are what they were
    got = run(eng, 4, prompt, blocks[:6] + [52], cached=96)
    assert np.abs(got - full).max() <= 1e-4


def test_settings_without_effect_are_the_same_setting(eng):
    prompt, blocks = toks(100), list(range(8))
    full = run(eng, 1, prompt, blocks)
    for same in ((256, 0, 0), (56, 200, 0), (30, 0, 3), (0, 5, 1)):  # as wide as the table, no layer, no window
        eng.set_window(*same)
        got = run(eng, 2, prompt, blocks[:6] + [20], cached=96)
        assert np.abs(got - full).max() <= 1e-4
        eng.release(2)


def test_pages_written_in_part_under_each(eng):
    """A prompt whose first page is half computed under one window and half under another."""
    prompt, blocks = toks(40), [0, 1, 2]
    eng.admit(1, prompt, blocks)
    eng.step([1], token_budget=8)
    eng.set_window(12, 0, 0)
    eng.step([1], token_budget=8)
    refused(eng, prompt, blocks, 16)
    eng.set_window(0)
    refused(eng, prompt, blocks, 16)
    eng.release(1)
    want = run(eng, 2, prompt, blocks, budget=24)  # written anew from its first slot on
    got = run(eng, 3, prompt, [0, 1, 7], cached=32)
    assert np.abs(want - got).max() <= 1e-4


def test_pages_filled_by_the_caller_are_accepted(eng):
    """K/V that no step wrote (a caller's own prefill) belongs to whatever window is set."""
    # the layers' pools lie one behind the other
    rt = C.CDLL("libcudart.so.12")
    rt.cudaMemset.argtypes = [C.c_void_p, C.c_int, C.c_size_t]
    assert rt.cudaMemset(eng.pool_ptr(0, 0), 0, eng.memory()["pool"]) == 0
    eng.set_window(30, 0, 0)
    eng.admit(1, toks(100), list(range(8)), num_cached=99)
    eng.step([1])
    eng.set_window(20, 0, 0)
    eng.admit(2, toks(50), list(range(10, 14)), num_cached=49)
    refused(eng, toks(100), list(range(8)), 100)  # its last token is a step's


def test_live_sequences_go_on(eng):
    prompt = toks(60)
    run(eng, 1, prompt, list(range(5)))
    eng.set_window(16, 0, 0)
    for k in range(6):  # eager, captured, replayed: over the K/V the sequence has
        eng.step([1], [3], [60 + k])
    assert eng.cached_tokens(1) == 66
    refused(eng, prompt, list(range(5)), 48)
