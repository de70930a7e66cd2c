"""Refusals of the cache-bounding operators: out-of-range host arguments return
cudaErrorInvalidValue before anything is launched (no GPU needed), empty calls
succeed, and the workspace formulas hold.  The pointers passed are never read."""
import ctypes as C

import pytest

from mini_serve_rs_b200 import engine as E

INVALID = 1  # cudaErrorInvalidValue
P = 0x7f0000000000  # a 16-byte aligned address nobody dereferences


def rows(**kw):
    a = dict(q=P, k=P, v=P, pool=64, tables=P, table_rows=8, blocks=40, row_table=P, ctx=P, n=4, max_ctx=600, window=100,
             sinks=4, out=P, hq=16, hkv=8, d=128, bs=16, scale=0.1, dtype=1, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return E.lib().ms_launch_window_attention(*a.values())


def chunk(**kw):
    a = dict(q=P, k=P, v=P, pool=64, tables=P, table_rows=8, blocks=40, tiles=P, n=4, window=100, sinks=4, out=P, hq=16, hkv=8,
             d=128, bs=16, scale=0.1, dtype=1, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return E.lib().ms_launch_window_prefill(*a.values())


def weights(**kw):
    a = dict(q=P, k=P, v=P, pool=64, tables=P, table_rows=8, blocks=40, row_table=P, ctx=P, n=4, max_ctx=600, out=P, w=P,
             stride=600, hq=16, hkv=8, d=128, bs=16, scale=0.1, ws=P, ws_bytes=1 << 40, dtype=1, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return E.lib().ms_launch_attention_weights(*a.values())


def evict(**kw):
    a = dict(k=P, v=P, pool=64, tables=P, table_rows=8, blocks=40, row_table=P, ctx=P, next=P, known=P, n=4, max_ctx=600,
             keep=500, sinks=4, recent=100, w=P, w_out=P, pos=P, pos_out=P, stride=600, hkv=8, d=128, bs=16, ws=P,
             ws_bytes=1 << 40, dtype=1, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return E.lib().ms_launch_evict(*a.values())


COMMON = [dict(k=None), dict(v=None), dict(tables=None), dict(k=P + 8), dict(v=P + 8), dict(pool=0), dict(pool=-1),
          dict(pool=1 << 31), dict(pool=1 << 40), dict(table_rows=0), dict(blocks=0), dict(blocks=-4), dict(d=96), dict(d=0),
          dict(bs=32), dict(dtype=3), dict(dtype=-1), dict(hkv=0), dict(n=-1), dict(sinks=-1)]
HEADS = [dict(hq=0), dict(hq=24), dict(hq=17), dict(hq=128), dict(q=None), dict(q=P + 8), dict(out=None), dict(out=P + 4), dict(scale=0.0),
         dict(scale=-0.1), dict(scale=float("nan")), dict(scale=float("inf"))]


@pytest.mark.parametrize("bad", COMMON + HEADS + [
    dict(ctx=None), dict(max_ctx=-1), dict(max_ctx=641), dict(window=-1), dict(row_table=None, n=9)], ids=str)
def test_window_attention_refuses(bad):
    assert rows(**bad) == INVALID


@pytest.mark.parametrize("bad", COMMON + HEADS + [dict(tiles=None), dict(window=-1), dict(dtype=0), dict(n=65536)], ids=str)
def test_window_prefill_refuses(bad):
    assert chunk(**bad) == INVALID


@pytest.mark.parametrize("bad", [b for b in COMMON if "sinks" not in b] + HEADS + [
    dict(ctx=None), dict(max_ctx=641), dict(w=None), dict(stride=599), dict(ws=None), dict(ws=P + 4), dict(ws_bytes=0),
    dict(ws_bytes=4 * 16 * 600 * 4 - 1)], ids=str)
def test_attention_weights_refuses(bad):
    assert weights(**bad) == INVALID


@pytest.mark.parametrize("bad", COMMON + [
    dict(ctx=None), dict(next=None), dict(pos=None), dict(w=None), dict(w_out=None), dict(pos_out=None), dict(stride=599),
    dict(max_ctx=641), dict(max_ctx=-1), dict(blocks=1 << 20, max_ctx=262145, stride=262145), dict(keep=0), dict(keep=-1),
    dict(recent=-1), dict(sinks=401), dict(recent=497), dict(sinks=2 ** 31 - 1, recent=2 ** 31 - 1), dict(ws=None),
    dict(ws_bytes=0), dict(row_table=None, n=9)], ids=str)
def test_evict_refuses(bad):
    assert evict(**bad) == INVALID


def test_empty_calls_succeed():
    assert rows(n=0) == 0 and chunk(n=0) == 0 and weights(n=0) == 0 and evict(n=0) == 0


def test_workspace_formulas():
    lib = E.lib()
    assert lib.ms_attention_weights_workspace_bytes(0, 16, 100) == 0
    assert lib.ms_attention_weights_workspace_bytes(3, 16, 0) == 0
    # one f32 score per (row, query head, key) at least; no 32-bit overflow
    for r, h, c in ((1, 16, 1), (64, 28, 4097), (256, 32, 131072)):
        assert lib.ms_attention_weights_workspace_bytes(r, h, c) >= 4 * r * h * c
    assert lib.ms_evict_workspace_bytes(0, 8, 100) == 0
    assert lib.ms_evict_workspace_bytes(256, 8, 262144) > 0
