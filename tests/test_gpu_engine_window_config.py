"""What of a configuration turns a sliding window on, and windows that cannot
bind: those steps are the steps without one, bit for bit."""
import dataclasses

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


def logits(cfg, windows=(), dtype=E.MS_DTYPE_BF16, steps=4):
    """Logits of a prompt of 100 tokens and of decode steps (eager, captured, replayed) in a
    table row of 16 pages, after set_window(*w) for each of `windows`."""
    eng = E.Engine(cfg, pool_blocks=16, max_seqs=2, max_tokens_per_step=256, max_blocks_per_seq=16, dtype=dtype)
    eng.load_weights(random_weights(CFG, 6, norm_std=0.1))
    for w in windows:
        eng.set_window(*w)
    prompt = np.random.default_rng(3).integers(0, cfg.vocab_size, 100).tolist()
    eng.admit(1, prompt, list(range(8)))
    eng.step([1], flags=E.MS_STEP_KEEP_LOGITS)
    out = [eng.logits(1).copy()]
    for k in range(steps):
        eng.step([1], [7], [100 + k], flags=E.MS_STEP_KEEP_LOGITS)
        out.append(eng.logits(1).copy())
    eng.close()
    return np.stack(out)


@pytest.mark.parametrize("first", [3, 4, 99])
def test_no_layer_from_max_window_layers_on(first):
    """max_window_layers at or above the layer count: no layer has the window."""
    cfg = dataclasses.replace(CFG, sliding_window=30, max_window_layers=first)
    assert np.array_equal(logits(cfg), logits(CFG))


def test_use_sliding_window_off():
    cfg = dataclasses.replace(CFG, sliding_window=30, max_window_layers=1, use_sliding_window=False)
    assert np.array_equal(logits(cfg), logits(CFG))
    on = dataclasses.replace(cfg, use_sliding_window=True)
    assert np.array_equal(logits(on), logits(CFG, [(30, 0, 1)]))
    assert not np.array_equal(logits(on), logits(CFG))
