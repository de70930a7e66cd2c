"""Engine steps with a sliding window (ms_engine_set_window, ModelConfig.sliding_window)
against the CPU oracle with the same mask: packed and chunked prompts, decode
steps eager and replayed, f32 and bf16, layers below first_layer untouched.
Tolerances are the other engine tests': f32 logits 2e-4 max-abs, bf16 0.25
max-abs and 0.04 RMS."""
import dataclasses
import math

import numpy as np
import pytest
import torch

from mini_serve_rs_b200 import engine as E
from mini_serve_rs_b200.config import ModelConfig
from oracle.qwen_ref import QwenRef, SeqState, apply_rope, linear, random_weights, rms_norm, softmax_last
from tests.gpu_util import need_gpu

pytestmark = pytest.mark.gpu
SHAPES = {"qwen3": ModelConfig(640, 256, 512, 3, 4, 2, 512, 128, 1e6, 1e-6, True, False, True),
          "qwen2 gqa 7": ModelConfig(512, 448, 640, 3, 7, 1, 512, 64, 1e6, 1e-6, False, True, False)}


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    need_gpu()


class WindowRef(QwenRef):
    """The oracle with layers >= first_layer attending to j <= p with p - j < window or j < sinks."""

    window, sinks, first_layer = 0, 0, 0

    def _attn(self, l, xs, state, offset):
        if self.window == 0 or l < self.first_layer:
            return super()._attn(l, xs, state, offset)
        cfg, w = self.cfg, self.w
        p = f"model.layers.{l}.self_attn."
        t, d, hq, hkv = xs.shape[0], cfg.hd(), cfg.num_attention_heads, cfg.num_key_value_heads
        q, k, v = (linear(xs, w[p + f"{n}_proj.weight"], w.get(p + f"{n}_proj.bias")).reshape(t, h, d)
                   for n, h in (("q", hq), ("k", hkv), ("v", hkv)))
        if cfg.qk_norm:
            q = rms_norm(q, w[p + "q_norm.weight"], cfg.rms_norm_eps)
            k = rms_norm(k, w[p + "k_norm.weight"], cfg.rms_norm_eps)
        cos, sin = self.cos[offset:offset + t], self.sin[offset:offset + t]
        kk, vv = state.append(l, apply_rope(k.transpose(0, 1), cos, sin), v.transpose(0, 1))
        q = apply_rope(q.transpose(0, 1), cos, sin)
        g = hq // hkv
        att = torch.matmul(q, kk.repeat_interleave(g, 0).transpose(1, 2)) / math.sqrt(d)
        pos, j = torch.arange(offset, offset + t)[:, None], torch.arange(offset + t)[None]
        see = (j <= pos) & ((pos - j < self.window) | (j < self.sinks))
        att = softmax_last(att.masked_fill(~see, float("-inf")))
        out = torch.matmul(att, vv.repeat_interleave(g, 0)).transpose(0, 1).reshape(t, hq * d)
        return linear(out, w[p + "o_proj.weight"])


def _close(got, want, dtype):
    err = np.abs(got.astype(np.float64) - want)
    print(f"logits: max {err.max():.2e} rms {math.sqrt((err ** 2).mean()):.2e}")
    if dtype == E.MS_DTYPE_F32:
        assert err.max() <= 2e-4
    else:
        assert err.max() <= 0.25 and math.sqrt((err ** 2).mean()) <= 0.04


@pytest.mark.parametrize("shape", list(SHAPES))
@pytest.mark.parametrize("dtype", [E.MS_DTYPE_F32, E.MS_DTYPE_BF16])
@pytest.mark.parametrize("window,sinks,first_layer,budget", [(24, 0, 0, 0), (33, 4, 1, 0), (16, 20, 0, 50), (1, 0, 2, 0)])
def test_steps_match_the_oracle(shape, dtype, window, sinks, first_layer, budget):
    cfg = SHAPES[shape]
    w = random_weights(cfg, 5, norm_std=0.1)
    ref = WindowRef(cfg, w)
    ref.window, ref.sinks, ref.first_layer = window, sinks, first_layer
    rng = np.random.default_rng(2)
    prompts = [rng.integers(0, cfg.vocab_size, n).tolist() for n in (90, 1, 17, 130)]
    eng = E.Engine(cfg, pool_blocks=64, max_seqs=8, max_tokens_per_step=512, max_blocks_per_seq=16, dtype=dtype)
    eng.load_weights(w)
    eng.set_window(window, sinks, first_layer)
    ids = [1, 2, 3, 4]
    for i, (sid, p) in enumerate(zip(ids, prompts)):
        eng.admit(sid, p, list(range(12 * i, 12 * i + 12)))
    states = [SeqState(cfg, 200) for _ in ids]
    done = [False] * 4
    for _ in range(20):
        run = [i for i in range(4) if not done[i]]
        toks, flags = eng.step([ids[i] for i in run], flags=E.MS_STEP_KEEP_LOGITS, token_budget=budget)
        lg = eng.logits(len(run))
        row = 0  # a prompt that the budget cuts comes last, behind those that finish
        for k, i in enumerate(run):
            if flags[k] & E.MS_FLAG_PREFILLED:
                _close(lg[row], ref.forward(prompts[i], states[i], 0).numpy(), dtype)
                done[i] = True
                row += 1
        if all(done):
            break
    assert all(done)
    pos = [len(p) for p in prompts]
    for step in range(6):  # the first eager, the second captured, the others replayed
        inputs = rng.integers(0, cfg.vocab_size, 4).tolist()
        eng.step(ids, inputs, pos, flags=E.MS_STEP_KEEP_LOGITS)
        lg = eng.logits(4)
        for i in range(4):
            _close(lg[i], ref.forward([inputs[i]], states[i], pos[i]).numpy(), dtype)
            pos[i] += 1
    assert eng.graph_stats()[1] > 0
    eng.close()


def test_window_off_is_the_step_without_it_and_config_turns_it_on():
    cfg = SHAPES["qwen3"]
    w = random_weights(cfg, 6, norm_std=0.1)
    prompt = np.random.default_rng(3).integers(0, cfg.vocab_size, 100).tolist()

    def logits(c, set_window=()):
        eng = E.Engine(c, pool_blocks=16, max_seqs=2, max_tokens_per_step=256, max_blocks_per_seq=16, dtype=E.MS_DTYPE_BF16)
        eng.load_weights(w)
        for args in set_window:
            eng.set_window(*args)
        eng.admit(1, prompt, list(range(8)))
        eng.step([1], flags=E.MS_STEP_KEEP_LOGITS)
        out = [eng.logits(1).copy()]
        for k in range(3):
            eng.step([1], [7], [100 + k], flags=E.MS_STEP_KEEP_LOGITS)
            out.append(eng.logits(1).copy())
        eng.close()
        return np.stack(out)

    plain = logits(cfg)
    assert np.array_equal(plain, logits(cfg, [(30, 2, 0), (0, 0, 0)]))
    on = dataclasses.replace(cfg, sliding_window=30, max_window_layers=1)
    windowed = logits(on)
    assert np.array_equal(windowed, logits(cfg, [(30, 0, 1)]))
    assert not np.array_equal(windowed, plain)


def test_bad_windows_are_refused():
    cfg = SHAPES["qwen3"]
    eng = E.Engine(cfg, pool_blocks=16, max_seqs=2, max_tokens_per_step=64, max_blocks_per_seq=8, dtype=E.MS_DTYPE_F32)
    for bad in ((-1, 0, 0), (8, -1, 0), (8, 0, -1), (8, 0, 4)):
        with pytest.raises(E.BackendError):
            eng.set_window(*bad)
    assert eng.is_healthy()
    eng.set_window(8, 0, 3)
    eng.close()
