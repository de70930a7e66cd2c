"""Attention over a bounded part of the paged cache (ms_launch_window_attention,
ms_launch_window_prefill, ms_launch_attention_weights) against the 64-bit
reference.  Keys that a row does not see hold NaN, table entries of pages it
does not see are out of range, and the status word must stay clear.  Tolerances
are oracle.bounded_cache_ref.bound's, per element."""
import math

import pytest
import torch

from mini_serve_rs_b200 import engine as E
from oracle import bounded_cache_ref as ref
from tests.gpu_util import dt_code, need_gpu, ptr, sync_ok

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    need_gpu()
    E.kernel_status(0)


def cache(ctx, first, window, sinks, hkv, d, dt, seed, spare=3, nan=True):
    """Pools, tables and row table for sequences of ctx[i] tokens of which the
    rows at positions first[i].. see some: what none of them sees is NaN in
    the pools and out of range in the tables."""
    g = torch.Generator().manual_seed(seed)
    n = len(ctx)
    blocks = max(1, max(-(-c // 16) for c in ctx)) + 1
    pool = sum(-(-c // 16) for c in ctx) + spare
    perm = torch.randperm(pool, generator=g).to(torch.int32)
    tables = torch.full((n, blocks), -5 if nan else 0, dtype=torch.int32)
    k = torch.full((pool, hkv, 16, d), math.nan if nan else 0.0)
    v = k.clone()
    row_table = torch.randperm(n, generator=g).to(torch.int32)
    off = 0
    for i, c in enumerate(ctx):
        t = int(row_table[i])
        see = torch.zeros(c, dtype=torch.bool)
        for p in range(first[i], c):
            see[:p + 1] |= ref.visible(p, window, sinks)
        for b in range(-(-c // 16)):
            if see[16 * b:16 * b + 16].any():
                tables[t, b] = perm[off]
                off += 1
        for j in torch.nonzero(see).flatten().tolist():
            page = int(tables[t, j // 16])
            k[page, :, j % 16] = torch.randn(hkv, d, generator=g)
            v[page, :, j % 16] = torch.randn(hkv, d, generator=g)
    return k.to(dt), v.to(dt), tables, row_table


def want_rows(q, k, v, tables, row_table, ctx, window, sinks):
    z = lambda t: torch.nan_to_num(t.float(), nan=0.0)  # what is not seen has weight 0
    return ref.window_rows(q, z(k), z(v), tables.clamp(min=0), row_table, ctx, window, sinks, ref.scale_of(q.shape[-1]))


def run_rows(q, k, v, tables, row_table, ctx, window, sinks, out, max_ctx=None, stream=None):
    dev = [x.to(DEV) for x in (q, k, v, tables, row_table, torch.tensor(ctx, dtype=torch.int32))]
    qd, kd, vd, td, rd, cd = dev
    return E.lib().ms_launch_window_attention(
        ptr(qd), ptr(kd), ptr(vd), k.shape[0], ptr(td), tables.shape[0], tables.shape[1], ptr(rd), ptr(cd), len(ctx),
        max_ctx or max(1, max(ctx)), window, sinks, ptr(out), q.shape[1], k.shape[1], q.shape[2], 16,
        ref.scale_of(q.shape[2]), dt_code(q), stream)


def check(got, want, absv, smax, n, dt, rounds_p=True, exp_err=2.0 ** -20):
    tol = ref.bound(dt, want, absv, smax, n, want.shape[-1], rounds_p, exp_err)
    err = (got.cpu().double() - want).abs()
    worst = float((err / tol).max())
    print(f"worst error / bound {worst:.3f}")
    assert torch.isfinite(got).all() and worst <= 1.0, worst


LENS = [0, 1, 2, 15, 16, 17, 31, 33, 100, 129, 255, 256, 700]


@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (1, 1), (16, 0), (17, 4), (100, 16), (97, 20), (64, 200),
                                          (1000, 4), (33, 1 << 30)])
@pytest.mark.parametrize("name,group,hkv,d", [("bf16", 2, 2, 128), ("f16", 7, 1, 64), ("f32", 2, 3, 128)])
def test_rows_at_every_edge(name, group, hkv, d, window, sinks):
    dt = DTYPES[name]
    k, v, tables, rt = cache(LENS, [max(0, c - 1) for c in LENS], window, sinks, hkv, d, dt, window * 7 + sinks % 1000)
    q = (2 * torch.randn(len(LENS), hkv * group, d, generator=torch.Generator().manual_seed(1))).to(dt)
    out = torch.full(q.shape, math.nan, dtype=dt, device=DEV)
    sync_ok(run_rows(q, k, v, tables, rt, LENS, window, sinks, out))
    assert E.kernel_status(0) == 0
    want, _, absv, smax = want_rows(q, k, v, tables, rt, LENS, window, sinks)
    check(out, want, absv, smax, max(LENS), dt)
    assert (out[0] == 0).all()  # a row that sees nothing


@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("group", [1, 2, 4, 7, 8])
@pytest.mark.parametrize("d", [64, 128])
def test_rows_every_head_layout(name, group, d):
    dt = DTYPES[name]
    lens = [3, 77, 400]
    k, v, tables, rt = cache(lens, [c - 1 for c in lens], 200, 5, 2, d, dt, group)
    q = (2 * torch.randn(len(lens), 2 * group, d, generator=torch.Generator().manual_seed(d))).to(dt)
    out = torch.full(q.shape, math.nan, dtype=dt, device=DEV)
    sync_ok(run_rows(q, k, v, tables, rt, lens, 200, 5, out))
    assert E.kernel_status(0) == 0
    want, _, absv, smax = want_rows(q, k, v, tables, rt, lens, 200, 5)
    check(out, want, absv, smax, max(lens), dt)


@pytest.mark.parametrize("rows", [1, 3, 40, 300])
def test_rows_split_and_long(rows):
    """Few rows split a long window over CTAs, many rows do not."""
    ctx = [max(1, 5003 - 61 * (i % 80)) for i in range(rows)]
    if rows == 300:
        ctx = [1 + 7 * (i % 60) for i in range(rows)]
    hkv, d, dt = 2, 64, torch.bfloat16
    window, sinks = 4001, 20
    g = torch.Generator().manual_seed(rows)
    blocks = -(-max(ctx) // 16)
    pool = 700
    k, v = torch.randn(pool, hkv, 16, d, generator=g).to(dt), torch.randn(pool, hkv, 16, d, generator=g).to(dt)
    tables = torch.randint(0, pool, (rows, blocks), generator=g).to(torch.int32)
    rt = torch.arange(rows, dtype=torch.int32)
    q = (2 * torch.randn(rows, 4, d, generator=g)).to(dt)
    out = torch.full(q.shape, math.nan, dtype=dt, device=DEV)
    sync_ok(run_rows(q, k, v, tables, rt, ctx, window, sinks, out, max_ctx=blocks * 16))
    assert E.kernel_status(0) == 0
    want, _, absv, smax = ref.window_rows(q, k, v, tables, rt, ctx, window, sinks, ref.scale_of(d))
    check(out, want, absv, smax, max(ctx), dt)


def test_rows_extreme_scores():
    """Scores far apart: one key takes all the weight, and it is the first, the last, a sink."""
    hkv, d, n = 1, 128, 90
    for name in ("bf16", "f32"):
        dt = DTYPES[name]
        for at in (0, 2, 60, 75, 89):
            k, v, tables, rt = cache([n], [n - 1], 40, 3, hkv, d, dt, at)
            q = torch.full((1, 2, d), 3.0).to(dt)
            if (n - 1 - at < 40) or at < 3:
                k[int(tables[0, at // 16]), 0, at % 16] = 60.0
            out = torch.full(q.shape, math.nan, dtype=dt, device=DEV)
            sync_ok(run_rows(q, k, v, tables, rt, [n], 40, 3, out))
            want, _, absv, smax = want_rows(q, k, v, tables, rt, [n], 40, 3)
            check(out, want, absv, torch.minimum(smax, torch.full_like(smax, 2500.0)), n, dt)
    assert E.kernel_status(0) == 0


# ---- prefill tiles ----------------------------------------------------------------

def tiles_of(chunks, row_table, group):
    size = 256 // (1 << (group - 1).bit_length())
    rows, r0 = [], 0
    for i, (start, n) in enumerate(chunks):
        rows += [(r0 + j, min(size, n - j), start + j, int(row_table[i])) for j in range(0, n, size)]
        r0 += n
    return torch.tensor(rows, dtype=torch.int32)


@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (1, 3), (16, 0), (50, 4), (130, 16), (127, 33), (300, 140),
                                          (5000, 4), (90, 1 << 30)])
@pytest.mark.parametrize("name,group,hkv,d", [("bf16", 2, 2, 128), ("f16", 1, 2, 64), ("bf16", 7, 1, 128)])
def test_chunks_at_every_edge(name, group, hkv, d, window, sinks):
    dt = DTYPES[name]
    chunks = [(0, 1), (0, 37), (200, 2), (333, 130), (640, 65), (511, 257), (7, 9)]
    ctx = [s + n for s, n in chunks]
    k, v, tables, rt = cache(ctx, [s for s, _ in chunks], window, sinks, hkv, d, dt, window + sinks % 1000, nan=True)
    T = sum(n for _, n in chunks)
    q = (2 * torch.randn(T, hkv * group, d, generator=torch.Generator().manual_seed(5))).to(dt)
    out = torch.full((T + 4, hkv * group, d), 7.0, dtype=dt, device=DEV)
    tl = tiles_of(chunks, rt, group)
    rc = E.lib().ms_launch_window_prefill(ptr(q.to(DEV)), ptr(k.to(DEV)), ptr(v.to(DEV)), k.shape[0],
                                          ptr(tables.to(DEV)), tables.shape[0], tables.shape[1], ptr(tl.to(DEV)),
                                          len(tl), window, sinks, ptr(out), hkv * group, hkv, d, 16, ref.scale_of(d),
                                          dt_code(q), None)
    sync_ok(rc)
    assert E.kernel_status(0) == 0
    assert (out[T:] == 7.0).all()  # rows behind the last one
    rows, rrt, r = [], [], 0
    for i, (s, n) in enumerate(chunks):
        rows += [s + j + 1 for j in range(n)]
        rrt += [int(rt[i])] * n
    want, _, absv, smax = want_rows(q, k, v, tables, torch.tensor(rrt), rows, window, sinks)
    # 2^x of some scores comes from a cubic good to 7.5e-5
    check(out[:T], want, absv, smax, max(ctx), dt, exp_err=8e-5)


@pytest.mark.parametrize("group", [1, 2, 4, 7, 8])
@pytest.mark.parametrize("d", [64, 128])
def test_chunks_every_head_layout(group, d):
    for dt in (torch.bfloat16, torch.float16):
        chunks = [(100, 300), (0, 20)]
        ctx = [s + n for s, n in chunks]
        k, v, tables, rt = cache(ctx, [s for s, _ in chunks], 150, 5, 2, d, dt, group)
        q = (2 * torch.randn(320, 2 * group, d, generator=torch.Generator().manual_seed(d))).to(dt)
        out = torch.full(q.shape, math.nan, dtype=dt, device=DEV)
        tl = tiles_of(chunks, rt, group)
        rc = E.lib().ms_launch_window_prefill(ptr(q.to(DEV)), ptr(k.to(DEV)), ptr(v.to(DEV)), k.shape[0],
                                              ptr(tables.to(DEV)), 2, tables.shape[1], ptr(tl.to(DEV)), len(tl), 150, 5,
                                              ptr(out), 2 * group, 2, d, 16, ref.scale_of(d), dt_code(q), None)
        sync_ok(rc)
        assert E.kernel_status(0) == 0
        rows = [s + j + 1 for s, n in chunks for j in range(n)]
        rrt = torch.tensor([int(rt[i]) for i, (s, n) in enumerate(chunks) for _ in range(n)])
        want, _, absv, smax = want_rows(q, k, v, tables, rrt, rows, 150, 5)
        check(out, want, absv, smax, max(ctx), dt, exp_err=8e-5)


@pytest.mark.parametrize("window,sinks", [(0, 0), (2500, 4), (2047, 130), (1100, 0)])
@pytest.mark.parametrize("name,group,hkv,d", [("bf16", 2, 1, 128), ("f16", 1, 2, 64), ("bf16", 7, 2, 64)])
def test_chunks_of_few_tiles_are_split(name, group, hkv, d, window, sinks):
    """Few tiles share their keys among the CTAs of a cluster; a short one leaves some without any."""
    dt = DTYPES[name]
    chunks = [(3000, 90), (0, 5), (1500, 1)]
    ctx = [s + n for s, n in chunks]
    k, v, tables, rt = cache(ctx, [s for s, _ in chunks], window, sinks, hkv, d, dt, window)
    T = sum(n for _, n in chunks)
    q = (2 * torch.randn(T, hkv * group, d, generator=torch.Generator().manual_seed(6))).to(dt)
    out = torch.full(q.shape, math.nan, dtype=dt, device=DEV)
    tl = tiles_of(chunks, rt, group)
    sync_ok(E.lib().ms_launch_window_prefill(ptr(q.to(DEV)), ptr(k.to(DEV)), ptr(v.to(DEV)), k.shape[0],
                                             ptr(tables.to(DEV)), tables.shape[0], tables.shape[1], ptr(tl.to(DEV)),
                                             len(tl), window, sinks, ptr(out), hkv * group, hkv, d, 16, ref.scale_of(d),
                                             dt_code(q), None))
    assert E.kernel_status(0) == 0
    rows = [s + j + 1 for s, n in chunks for j in range(n)]
    rrt = torch.tensor([int(rt[i]) for i, (s, n) in enumerate(chunks) for _ in range(n)])
    want, _, absv, smax = want_rows(q, k, v, tables, rrt, rows, window, sinks)
    check(out, want, absv, smax, max(ctx), dt, exp_err=8e-5)


# ---- attention weights ------------------------------------------------------------

def run_weights(q, k, v, tables, rt, ctx, out, w, max_ctx=None, ws=None, stream=None):
    lib = E.lib()
    mc = max_ctx or max(ctx)
    need = lib.ms_attention_weights_workspace_bytes(len(ctx), q.shape[1], mc)
    ws = torch.empty(need, dtype=torch.uint8, device=DEV) if ws is None else ws
    return lib.ms_launch_attention_weights(ptr(q), ptr(k), ptr(v), k.shape[0], ptr(tables), tables.shape[0],
                                           tables.shape[1], ptr(rt),
                                           ptr(torch.tensor(ctx, dtype=torch.int32, device=DEV)), len(ctx), mc, ptr(out),
                                           ptr(w), w.shape[-1], q.shape[1], k.shape[1], q.shape[2], 16,
                                           ref.scale_of(q.shape[2]), ptr(ws), ws.numel(), dt_code(q), stream)


@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("group,hkv,d", [(1, 2, 64), (2, 2, 128), (4, 1, 64), (7, 2, 128), (8, 1, 128)])
@pytest.mark.parametrize("odd", [3, 2])  # the stride: a multiple of 4, and not
def test_weights_accumulate(name, group, hkv, d, odd):
    dt = DTYPES[name]
    ctx = LENS + [1301]
    k, v, tables, rt = cache(ctx, [max(0, c - 1) for c in ctx], 0, 0, hkv, d, dt, 3)
    q = (2 * torch.randn(len(ctx), hkv * group, d, generator=torch.Generator().manual_seed(9))).to(dt)
    out = torch.full(q.shape, math.nan, dtype=dt, device=DEV)
    stride = max(ctx) + odd
    w0 = torch.rand(len(ctx), hkv, stride, generator=torch.Generator().manual_seed(2))
    wd = w0.to(DEV)
    dev = [x.to(DEV) for x in (q, k, v, tables, rt)]
    for _ in range(2):
        sync_ok(run_weights(*dev, ctx, out, wd))
    assert E.kernel_status(0) == 0
    want, add, absv, smax = want_rows(q, k, v, tables, rt, ctx, 0, 0)
    check(out, want, absv, smax, max(ctx), dt)
    worst = 0.0
    for r, n in enumerate(ctx):
        t = int(rt[r])
        got, base = wd[t].cpu().double(), w0[t].double()
        assert torch.equal(got[:, n:], base[:, n:])  # behind the row's context
        if n == 0:
            continue
        rel = 2 * 2.0 ** -20 + 2 * (d + 4) * 2.0 ** -23 * float(smax[r].max()) + (n + 64) * 2.0 ** -23
        tol = 2 * add[r] * rel + 2 * 2.0 ** -24 * (base[:, :n] + 2 * add[r]) + 1e-37
        worst = max(worst, float(((got[:, :n] - base[:, :n] - 2 * add[r]).abs() / tol).max()))
        # the weights of a head sum to one
        assert abs(float((got[:, :n] - base[:, :n]).sum()) - 2 * hkv * group) < 1e-3 * hkv * group
    print(f"weights: worst error / bound {worst:.3f}")
    assert worst <= 1.0


def test_weights_equal_calls_give_equal_bits():
    ctx = [4000, 37, 900]
    hkv, group, d, dt = 4, 7, 128, torch.bfloat16
    g = torch.Generator().manual_seed(0)
    k, v = (torch.randn(400, hkv, 16, d, generator=g).to(dt).to(DEV) for _ in range(2))
    tables = torch.randperm(400, generator=g)[:3 * 130].reshape(3, 130).to(torch.int32)
    tables = torch.cat([tables, tables[:, :130]], 1).to(DEV)
    q = (2 * torch.randn(3, hkv * group, d, generator=g)).to(dt).to(DEV)
    rt = torch.tensor([2, 0, 1], dtype=torch.int32, device=DEV)
    first = None
    for _ in range(4):
        out, w = torch.empty_like(q), torch.zeros(3, hkv, 4000, device=DEV)
        sync_ok(run_weights(q, k, v, tables, rt, ctx, out, w))
        if first is None:
            first = (out, w)
        assert torch.equal(out, first[0]) and torch.equal(w, first[1])


def test_weights_with_nothing_cached():
    q = torch.randn(2, 4, 64, device=DEV).bfloat16()
    pool = torch.zeros(1, 2, 16, 64, dtype=torch.bfloat16, device=DEV)
    out, w = torch.full_like(q, 5.0), torch.full((2, 2, 8), 3.0, device=DEV)
    tables, zero = torch.zeros(2, 1, dtype=torch.int32, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV)
    rc = E.lib().ms_launch_attention_weights(ptr(q), ptr(pool), ptr(pool), 1, ptr(tables), 2, 1, None, ptr(zero), 2, 0, ptr(out),
                                             ptr(w), 8, 4, 2, 64, 16, 0.125, None, 0, 1, None)
    sync_ok(rc)
    assert E.kernel_status(0) == 0 and (out == 0).all() and (w == 3.0).all()


def test_pages_whose_elements_pass_32_bits():
    """A pool of 2^31 elements and more: its last pages, in every operator that reads them."""
    hkv, d, dt, n = 8, 128, torch.bfloat16, 100
    pool = (2 ** 31 // (hkv * 16 * d)) + 40
    k, v = (torch.zeros(pool, hkv, 16, d, dtype=dt, device=DEV) for _ in range(2))
    assert k.numel() > 2 ** 31
    g = torch.Generator().manual_seed(8)
    pages = torch.tensor([pool - 1, 3, pool - 9, pool // 2, pool - 2, 0, pool - 30], dtype=torch.int32)
    small_k, small_v = (torch.randn(7, hkv, 16, d, generator=g).to(dt) for _ in range(2))
    k[pages.long().to(DEV)], v[pages.long().to(DEV)] = small_k.to(DEV), small_v.to(DEV)
    tables, rt = pages[None].clone(), torch.zeros(1, dtype=torch.int32)
    q = (2 * torch.randn(1, 16, d, generator=g)).to(dt)
    local = torch.arange(7, dtype=torch.int32)[None]
    qd, td, rd = q.to(DEV), tables.to(DEV), rt.to(DEV)
    for window, sinks in ((0, 0), (40, 3)):
        out = torch.full(q.shape, math.nan, dtype=dt, device=DEV)
        sync_ok(run_rows(qd, k, v, td, rd, [n], window, sinks, out))
        want, _, absv, smax = ref.window_rows(q, small_k, small_v, local, rt, [n], window, sinks, ref.scale_of(d))
        check(out, want, absv, smax, n, dt)
        tl = torch.tensor([[0, 1, n - 1, 0]], dtype=torch.int32, device=DEV)
        out = torch.full(q.shape, math.nan, dtype=dt, device=DEV)
        sync_ok(E.lib().ms_launch_window_prefill(ptr(qd), ptr(k), ptr(v), pool, ptr(td), 1, 7, ptr(tl), 1, window, sinks,
                                                 ptr(out), 16, hkv, d, 16, ref.scale_of(d), dt_code(q), None))
        check(out, want, absv, smax, n, dt, exp_err=8e-5)
    out, w = torch.full(q.shape, math.nan, dtype=dt, device=DEV), torch.zeros(1, hkv, n, device=DEV)
    sync_ok(run_weights(qd, k, v, td, rd, [n], out, w))
    want, add, absv, smax = ref.window_rows(q, small_k, small_v, local, rt, [n], 0, 0, ref.scale_of(d))
    check(out, want, absv, smax, n, dt)
    assert float((w[0].cpu().double() - add[0]).abs().max()) < 1e-5
    assert E.kernel_status(0) == 0


# ---- values in device memory that are out of range ----------------------------------

def test_bad_rows_are_skipped_and_flagged():
    hkv, d, dt = 2, 64, torch.bfloat16
    ctx = [40, 50, 60]
    k, v, tables, rt = cache(ctx, [0, 0, 0], 0, 0, hkv, d, dt, 11)
    q = torch.randn(3, 4, d).to(dt)
    good = torch.full(q.shape, 5.0, dtype=dt, device=DEV)
    sync_ok(run_rows(q, k, v, tables, rt, ctx, 30, 2, good))
    assert E.kernel_status(0) == 0
    for bad_ctx, bad_rt in (([40, -1, 60], rt), ([40, 61, 60], rt), (ctx, torch.tensor([rt[0], 3, rt[2]], dtype=torch.int32)),
                            (ctx, torch.tensor([rt[0], -1, rt[2]], dtype=torch.int32))):
        out = torch.full(q.shape, 5.0, dtype=dt, device=DEV)
        sync_ok(run_rows(q, k, v, tables, bad_rt, bad_ctx, 30, 2, out, max_ctx=60))
        assert E.kernel_status(0) == 2
        assert (out[1] == 5.0).all() and torch.equal(out[0], good[0]) and torch.equal(out[2], good[2])
    # a page out of range: that row alone is unspecified
    for page in (-1, k.shape[0], 2 ** 31 - 1, -2 ** 31):
        t = tables.clone()
        t[int(rt[1]), 2] = page
        out = torch.full(q.shape, 5.0, dtype=dt, device=DEV)
        sync_ok(run_rows(q, k, v, t, rt, ctx, 30, 2, out))
        assert E.kernel_status(0) == 2
        assert torch.equal(out[0], good[0]) and torch.equal(out[2], good[2])


def test_bad_tiles_are_skipped_and_flagged():
    hkv, d, dt = 1, 128, torch.bfloat16
    k, v, tables, rt = cache([200], [0], 0, 0, hkv, d, dt, 12)
    q = torch.randn(200, 2, d).to(dt).to(DEV)
    kd, vd, td = k.to(DEV), v.to(DEV), tables.to(DEV)

    def go(tl, tab=td):
        out = torch.full(q.shape, 5.0, dtype=dt, device=DEV)
        t = torch.tensor(tl, dtype=torch.int32, device=DEV)
        sync_ok(E.lib().ms_launch_window_prefill(ptr(q), ptr(kd), ptr(vd), k.shape[0], ptr(tab), 1, tables.shape[1],
                                                 ptr(t), len(tl), 64, 4, ptr(out), 2, hkv, d, 16, ref.scale_of(d),
                                                 dt_code(q), None))
        return out, E.kernel_status(0)

    good, st = go([(0, 128, 0, 0), (128, 72, 128, 0)])
    assert st == 0
    for bad in ((128, 129, 0, 0), (128, -1, 0, 0), (128, 72, -1, 0), (128, 72, 10 ** 9, 0), (128, 72, 128, 1),
                (128, 72, 128, -1), (-3, 72, 128, 0), (128, 72, 2 ** 31 - 1, 0)):
        out, st = go([(0, 128, 0, 0), bad])
        assert st == 2 and torch.equal(out[:128], good[:128]) and (out[128:] == 5.0).all(), bad
    for page in (-1, k.shape[0], 2 ** 31 - 1, -2 ** 31):
        t = tables.clone()
        t[0, 10] = page
        out, st = go([(0, 128, 0, 0), (128, 72, 128, 0)], t.to(DEV))
        assert st == 2 and torch.equal(out[:128], good[:128]), page
    out, st = go([(0, 0, 0, 0), (0, 128, 0, 0)])  # an empty tile is no error
    assert st == 0 and torch.equal(out[:128], good[:128]) and (out[128:] == 5.0).all()


def test_weights_of_a_repeated_table_row_are_flagged():
    hkv, d, dt = 2, 64, torch.bfloat16
    ctx = [40, 50, 60]
    k, v, tables, rt = cache(ctx, [0, 0, 0], 0, 0, hkv, d, dt, 11)
    q = torch.randn(3, 4, d).to(dt)
    dev = [x.to(DEV) for x in (q, k, v, tables)]
    out, w = torch.full(q.shape, 5.0, dtype=dt, device=DEV), torch.zeros(3, hkv, 64, device=DEV)
    sync_ok(run_weights(*dev, rt.to(DEV), ctx, out, w))
    assert E.kernel_status(0) == 0
    out2, w2 = torch.full(q.shape, 5.0, dtype=dt, device=DEV), torch.zeros(3, hkv, 64, device=DEV)
    twice = torch.tensor([rt[0], rt[1], rt[1]], dtype=torch.int32, device=DEV)
    sync_ok(run_weights(*dev, twice, [40, 50, 50], out2, w2, max_ctx=60))
    assert E.kernel_status(0) == 2
    assert torch.equal(out2[:2], out[:2]) and (out2[2] == 5.0).all()
    assert torch.equal(w2[rt[0].long()], w[rt[0].long()]) and torch.equal(w2[rt[1].long()], w[rt[1].long()])
    assert (w2[rt[2].long()] == 0).all()


def test_padded_batches():
    """Empty rows and tiles may name any table row, a used one or none."""
    hkv, d, dt = 2, 64, torch.bfloat16
    ctx = [40, 50]
    k, v, tables, rt = cache(ctx, [0, 0], 0, 0, hkv, d, dt, 11)
    q = torch.randn(5, 4, d).to(dt)
    dev = [x.to(DEV) for x in (q, k, v, tables)]
    real = [1, 3]
    plain = [dev[0][real].contiguous()] + dev[1:]
    out, w = torch.full((2, 4, d), 5.0, dtype=dt, device=DEV), torch.zeros(2, hkv, 64, device=DEV)
    sync_ok(run_weights(*plain, rt.to(DEV), ctx, out, w))
    padded_rt = torch.tensor([rt[0], rt[0], -7, rt[1], rt[1]], dtype=torch.int32, device=DEV)
    out2, w2 = torch.full(q.shape, 5.0, dtype=dt, device=DEV), torch.zeros(2, hkv, 64, device=DEV)
    sync_ok(run_weights(*dev, padded_rt, [0, 40, 0, 50, 0], out2, w2))
    assert E.kernel_status(0) == 0
    assert torch.equal(out2[real], out) and torch.equal(w2, w) and (out2[[0, 2, 4]] == 0).all()
    out3 = torch.full(q.shape, 5.0, dtype=dt, device=DEV)
    sync_ok(run_rows(*dev, padded_rt, [0, 40, 0, 50, 0], 0, 0, out3))
    assert E.kernel_status(0) == 0 and torch.equal(out3[real], out) and (out3[[0, 2, 4]] == 0).all()
    chunk = torch.full((2, 4, d), 5.0, dtype=dt, device=DEV)
    tl = torch.tensor([[0, 1, 39, rt[0]], [-9, 0, -1, 77], [1, 1, 49, rt[1]], [0, 0, 1 << 30, -1]], dtype=torch.int32, device=DEV)
    sync_ok(E.lib().ms_launch_window_prefill(ptr(plain[0]), ptr(dev[1]), ptr(dev[2]), k.shape[0], ptr(dev[3]), 2,
                                             tables.shape[1], ptr(tl), 4, 0, 0, ptr(chunk), 4, hkv, d, 16, ref.scale_of(d),
                                             dt_code(q), None))
    assert E.kernel_status(0) == 0
    want, _, absv, smax = want_rows(q[real], k, v, tables, rt, ctx, 0, 0)
    check(chunk, want, absv, smax, 50, dt, exp_err=8e-5)


def test_no_row_table_and_very_many_rows():
    hkv, d, dt = 1, 64, torch.bfloat16
    k, v, tables, _ = cache([40, 50, 60], [0, 0, 0], 0, 0, hkv, d, dt, 13)
    rt = torch.arange(3, dtype=torch.int32)
    order = torch.argsort(cache([40, 50, 60], [0, 0, 0], 0, 0, hkv, d, dt, 13)[3])
    ctx = [[40, 50, 60][int(i)] for i in order]  # of table rows 0, 1, 2
    q = torch.randn(3, 4, d).to(dt)
    dev = [x.to(DEV) for x in (q, k, v, tables, rt)]
    named, unnamed = (torch.full(q.shape, 5.0, dtype=dt, device=DEV) for _ in range(2))
    sync_ok(run_rows(*dev, ctx, 30, 2, named))
    cd = torch.tensor(ctx, dtype=torch.int32, device=DEV)
    call = (ptr(dev[1]), ptr(dev[2]), k.shape[0], ptr(dev[3]), 3, tables.shape[1])
    rc = E.lib().ms_launch_window_attention(ptr(dev[0]), *call, None, ptr(cd), 3, 60, 30, 2, ptr(unnamed), 4, hkv, d, 16,
                                            ref.scale_of(d), 1, None)
    sync_ok(rc)
    assert E.kernel_status(0) == 0 and torch.equal(named, unnamed)
    rows = 70001  # more than a grid's y or z holds
    many_q = dev[0][:1].expand(rows, -1, -1).contiguous()
    out = torch.full(many_q.shape, 5.0, dtype=dt, device=DEV)
    zeros, many_ctx = torch.zeros(rows, dtype=torch.int32, device=DEV), torch.full((rows,), ctx[0], dtype=torch.int32, device=DEV)
    sync_ok(E.lib().ms_launch_window_attention(ptr(many_q), ptr(dev[1]), ptr(dev[2]), k.shape[0], ptr(dev[3]), 3,
                                               tables.shape[1], ptr(zeros), ptr(many_ctx), rows, 60, 30, 2, ptr(out), 4, hkv, d,
                                               16, ref.scale_of(d), 1, None))
    assert E.kernel_status(0) == 0 and (out == out[:1]).all()
    want, _, absv, smax = want_rows(q[:1], k, v, tables, rt, ctx[:1], 30, 2)
    check(out[:1], want, absv, smax, 60, dt)


# ---- streams and graphs ---------------------------------------------------------------

def test_streams_and_graph_replay():
    hkv, group, d, dt = 2, 2, 128, torch.bfloat16
    ctx = [700, 60, 300]
    k, v, tables, rt = cache(ctx, [0, 0, 0], 0, 0, hkv, d, dt, 4)
    q = (2 * torch.randn(3, hkv * group, d, generator=torch.Generator().manual_seed(0))).to(dt)
    kd, vd, td, rd, qd = (x.to(DEV) for x in (k, v, tables, rt, q))
    cd = torch.tensor(ctx, dtype=torch.int32, device=DEV)
    chunks = [(s, 60) for s in (640, 0, 240)]
    tl = tiles_of(chunks, rt, group).to(DEV)
    qc = (2 * torch.randn(180, hkv * group, d, generator=torch.Generator().manual_seed(1))).to(dt).to(DEV)
    lib = E.lib()
    need = lib.ms_attention_weights_workspace_bytes(3, hkv * group, 700)

    def calls(stream, o):
        pools = (ptr(kd), ptr(vd), k.shape[0], ptr(td), 3, tables.shape[1])
        tail = (hkv * group, hkv, d, 16, ref.scale_of(d))
        assert lib.ms_launch_window_attention(ptr(qd), *pools, ptr(rd), ptr(cd), 3, 700, 128, 4, ptr(o["row"]), *tail,
                                              dt_code(q), stream) == 0
        assert lib.ms_launch_window_prefill(ptr(qc), *pools, ptr(tl), len(tl), 128, 4, ptr(o["chunk"]), *tail,
                                            dt_code(q), stream) == 0
        assert lib.ms_launch_attention_weights(ptr(qd), *pools, ptr(rd), ptr(cd), 3, 700, ptr(o["wrow"]), ptr(o["w"]), 700,
                                               *tail, ptr(o["ws"]), need, dt_code(q), stream) == 0

    def buffers():
        return {"row": torch.zeros_like(qd), "chunk": torch.zeros_like(qc), "wrow": torch.zeros_like(qd),
                "w": torch.zeros(3, hkv, 700, device=DEV), "ws": torch.empty(need, dtype=torch.uint8, device=DEV)}

    want = buffers()
    calls(None, want)
    torch.cuda.synchronize()
    # two streams at once, each with its own workspace
    side = [torch.cuda.Stream() for _ in range(2)]
    got = [buffers() for _ in side]
    torch.cuda.synchronize()
    for s, o in zip(side, got):
        calls(s.cuda_stream, o)
    torch.cuda.synchronize()
    for o in got:
        assert all(torch.equal(o[n], want[n]) for n in ("row", "chunk", "wrow", "w"))
    # captured once, replayed with other inputs in the same buffers
    o = buffers()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls(torch.cuda.current_stream().cuda_stream, o)
    o["w"].zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o[n], want[n]) for n in ("row", "chunk", "wrow", "w"))
    qd.mul_(-0.5)
    cd.copy_(torch.tensor([313, 60, 1], dtype=torch.int32))
    again = buffers()
    calls(None, again)
    torch.cuda.synchronize()
    o["w"].zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o[n], again[n]) for n in ("row", "chunk", "wrow", "w"))
    assert not torch.equal(o["row"], want["row"])
    assert E.kernel_status(0) == 0


def test_a_wait_that_runs_out_is_reported():
    """The poll limit set to zero: no copy has landed at the first poll, every
    one still lands before the CTA leaves; nothing is written, the status says so."""
    lib = E.lib()
    hkv, d, dt = 2, 128, torch.bfloat16
    for rows in (1, 200):  # split over a cluster, and not
        ctx = [3000] * rows
        g = torch.Generator().manual_seed(0)
        k, v = (torch.randn(400, hkv, 16, d, generator=g).to(dt).to(DEV) for _ in range(2))
        tables = torch.randint(0, 400, (rows, 188), generator=g).to(torch.int32).to(DEV)
        q = torch.randn(rows, 4, d, generator=g).to(dt).to(DEV)
        rt = torch.arange(rows, dtype=torch.int32, device=DEV)
        good, out, w = torch.full_like(q, 5.0), torch.full_like(q, 5.0), torch.zeros(rows, hkv, 3000, device=DEV)
        try:
            lib.ms_test_set_attention_wait_limit(0)
            sync_ok(run_rows(q, k, v, tables, rt, ctx, 2000, 4, out))
            assert E.kernel_status(0) == 1 and (out == 5.0).all()
            sync_ok(run_weights(q, k, v, tables, rt, ctx, out, w))
            assert E.kernel_status(0) == 1 and (out == 5.0).all() and (w == 0).all()
        finally:
            lib.ms_test_set_attention_wait_limit(-1)
        sync_ok(run_rows(q, k, v, tables, rt, ctx, 2000, 4, good))
        assert E.kernel_status(0) == 0 and not (good == 5.0).any()
