"""Values that test the arithmetic of ms_launch_window_attention,
ms_launch_window_prefill and ms_launch_attention_weights: weights far below the
heaviest one, NaN and infinity where a row sees them, large numbers where it
does not."""
import math

import pytest
import torch

from mini_serve_rs_b200 import engine as E
from oracle import bounded_cache_ref as ref
from tests.gpu_util import dt_code, need_gpu, ptr, sync_ok
from tests.test_gpu_window import DEV, DTYPES, run_rows, run_weights, tiles_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    need_gpu()
    E.kernel_status(0)


def one_sequence(k, v):
    """Keys and values [n, Hkv, D] as pools, block table and row table of one sequence."""
    n, hkv, d = k.shape
    blocks = -(-n // 16)
    pools = []
    for x in (k, v):
        p = torch.zeros(blocks * 16, hkv, d, dtype=x.dtype)
        p[:n] = x
        pools.append(p.reshape(blocks, 16, hkv, d).transpose(1, 2).contiguous())
    perm = torch.randperm(blocks, generator=torch.Generator().manual_seed(n))
    tables = torch.empty(1, blocks, dtype=torch.int32)
    tables[0] = perm.to(torch.int32)
    for i, p in enumerate(pools):
        pools[i] = torch.empty_like(p)
        pools[i][perm] = p
    return pools[0], pools[1], tables, torch.zeros(1, dtype=torch.int32)


def run_chunk(q, k, v, tables, tl, window, sinks, out):
    return E.lib().ms_launch_window_prefill(
        ptr(q.to(DEV)), ptr(k.to(DEV)), ptr(v.to(DEV)), k.shape[0], ptr(tables.to(DEV)), tables.shape[0], tables.shape[1],
        ptr(tl.to(DEV)), len(tl), window, sinks, ptr(out), q.shape[1], k.shape[1], q.shape[2], 16,
        ref.scale_of(q.shape[2]), dt_code(q), None)


def tails(dt, d, far, heavy, n=16384):
    """One key that takes nearly all the weight and whose value is 0, and n keys 2^far below it
    whose values are 16 to 32: what a row returns is the light keys' share alone."""
    g = torch.Generator().manual_seed(int(far * 10))
    k, v = torch.zeros(n + 1, 1, d), 16 + 16 * torch.rand(n + 1, 1, d, generator=g)
    k[:, 0, 0] = -far * math.log(2.0) * math.sqrt(d) / 8
    k[heavy], v[heavy] = 0.0, 0.0
    q = torch.zeros(1, 2, d)
    q[..., 0] = 8.0
    return q.to(dt), k.to(dt), v.to(dt)


def tail_tolerance(dt, want, absv, n, exp_err):
    """oracle.bounded_cache_ref.bound without its constant term: each weight keeps the relative
    precision of its type however light it is, the result is rounded once (half a subnormal step
    at least).  Sums of n f32 terms of one sign: 2^-23 each.  The scores are one exact product each."""
    half = torch.finfo(dt).eps / 2
    rel = 2 * exp_err + (n + 64) * 2.0 ** -23 + 2 * 2.0 ** -23 * 64 + (half if dt != torch.float32 else 0.0)
    step = torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
    return half * want.abs() * 1.001 + rel * absv + step / 2


@pytest.mark.parametrize("name,d", [("f16", 128), ("f16", 64), ("bf16", 128), ("f32", 64)])
@pytest.mark.parametrize("far", [8.0, 15.3, 20.7, 25.5, 28.0])
@pytest.mark.parametrize("heavy", [0, 16384])
def test_rows_keep_light_weights(name, d, far, heavy):
    dt = DTYPES[name]
    q, k, v = tails(dt, d, far, heavy)
    n = k.shape[0]
    kp, vp, tables, rt = one_sequence(k, v)
    want, add, absv, _ = ref.window_rows(q, kp, vp, tables, rt, [n], 0, 0, ref.scale_of(d))
    tol = tail_tolerance(dt, want, absv, n, 2.0 ** -20)
    assert float((tol / want).max()) < 0.02  # far below what is measured
    w = torch.zeros(1, 1, n + 3, device=DEV)
    for op in ("window", "sinks and window", "weights"):
        out = torch.full(q.shape, math.nan, dtype=dt, device=DEV)
        if op == "weights":
            sync_ok(run_weights(q.to(DEV), kp.to(DEV), vp.to(DEV), tables.to(DEV), rt.to(DEV), [n], out, w))
        else:
            sync_ok(run_rows(q, kp, vp, tables, rt, [n], 0 if op == "window" else n - 16, 0 if op == "window" else 16, out))
        worst = float(((out.cpu().double() - want).abs() / tol).max())
        print(f"{op}: worst error / bound {worst:.3f}")
        assert worst <= 1.0, op
    got = w[0, :, :n].cpu().double()
    assert float(((got - add[0]).abs() / add[0]).max()) < 2 * 2.0 ** -20 + (n + 200) * 2.0 ** -23
    assert E.kernel_status(0) == 0


@pytest.mark.parametrize("name,d", [("f16", 128), ("f16", 64), ("bf16", 128)])
@pytest.mark.parametrize("far", [8.0, 15.3, 20.7, 24.5])
@pytest.mark.parametrize("heavy", [0, 16350])
@pytest.mark.parametrize("window,sinks", [(0, 0), (16300, 100)])
def test_chunks_keep_light_weights(name, d, far, heavy, window, sinks):
    """The tiles' reference may lie 2^4 below the maximum: weights from 2^-25 on are as precise as any."""
    dt = DTYPES[name]
    q, k, v = tails(dt, d, far, heavy)
    n = k.shape[0]
    kp, vp, tables, rt = one_sequence(k, v)
    rows = 3
    q = q.expand(rows, 2, d).contiguous()
    tl = tiles_of([(n - rows, rows)], rt, 2)
    out = torch.full(q.shape, math.nan, dtype=dt, device=DEV)
    sync_ok(run_chunk(q, kp, vp, tables, tl, window, sinks, out))
    assert E.kernel_status(0) == 0
    want, _, absv, _ = ref.window_rows(q, kp, vp, tables, rt.expand(rows), [n - rows + 1 + i for i in range(rows)], window,
                                       sinks, ref.scale_of(d))
    tol = tail_tolerance(dt, want, absv, n, 8e-5)
    worst = float(((out.cpu().double() - want).abs() / tol).max())
    print(f"worst error / bound {worst:.3f}")
    assert worst <= 1.0


@pytest.mark.parametrize("name", ["f16", "bf16"])
@pytest.mark.parametrize("step", [0.5, 3.9, 4.1, 7.9, 8.1])
def test_chunks_whose_scores_climb(name, step):
    """Each group of 128 keys is 2^step heavier than the one before it."""
    dt, d, n = DTYPES[name], 64, 128 * 9 + 5
    g = torch.Generator().manual_seed(2)
    k, v = torch.zeros(n, 1, d), torch.randn(n, 1, d, generator=g)
    k[:, 0, 0] = (torch.arange(n) // 128) * step * math.log(2.0) * math.sqrt(d) / 8
    k[:, 0, 1] = 0.02 * torch.randn(n, generator=g)
    q = torch.zeros(40, 2, d)
    q[..., 0] = 8.0
    q[..., 1] = torch.randn(40, 2, generator=g)
    q, k, v = q.to(dt), k.to(dt), v.to(dt)
    kp, vp, tables, rt = one_sequence(k, v)
    for window in (0, 700):
        tl = tiles_of([(n - 40, 40)], rt, 2)
        out = torch.full(q.shape, math.nan, dtype=dt, device=DEV)
        sync_ok(run_chunk(q, kp, vp, tables, tl, window, 0, out))
        want, _, absv, _ = ref.window_rows(q, kp, vp, tables, rt.expand(40), [n - 39 + i for i in range(40)], window, 0,
                                           ref.scale_of(d))
        # scores up to 65 in two exact products: 2^-23 of that, twice
        tol = tail_tolerance(dt, want, absv, n, 8e-5) + 4 * 65 * 2.0 ** -23 * absv
        worst = float(((out.cpu().double() - want).abs() / tol).max())
        print(f"window {window}: worst error / bound {worst:.3f}")
        assert worst <= 1.0
    assert E.kernel_status(0) == 0


def same_nans(got, want, other, tol):
    """NaN exactly where the formula has it; elsewhere within tol of it and the bits of `other`."""
    got, nan = got.cpu(), want.isnan()
    assert torch.equal(got.isnan(), nan)
    assert torch.equal(got[~nan], other.cpu()[~nan])
    assert bool(((got.double() - want).abs()[~nan] <= tol[~nan]).all())


@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("window", [32, 2000])  # one CTA a row, a cluster
@pytest.mark.parametrize("where", ["query", "key", "first key", "value", "infinite query"])
def test_rows_that_see_a_nan(name, window, where):
    dt, d, hkv, group = DTYPES[name], 64, 2, 2
    g = torch.Generator().manual_seed(4)
    ctx = [2500, 40, 2300, 1, 0]
    rows, blocks = len(ctx), 160
    k, v = (torch.randn(rows * blocks, hkv, 16, d, generator=g).to(dt) for _ in range(2))
    tables = torch.arange(rows * blocks, dtype=torch.int32).reshape(rows, blocks)
    rt = torch.arange(rows, dtype=torch.int32)
    q = torch.randn(rows, hkv * group, d, generator=g).to(dt)
    clean = torch.full(q.shape, 5.0, dtype=dt, device=DEV)
    sync_ok(run_rows(q, k, v, tables, rt, ctx, window, 0, clean))
    w_clean = torch.zeros(rows, hkv, 2500, device=DEV)
    sync_ok(run_weights(q.to(DEV), k.to(DEV), v.to(DEV), tables.to(DEV), rt.to(DEV), ctx, torch.empty_like(clean), w_clean))
    for row in range(3 if where == "infinite query" else 4):  # (one key's score alone may be -infinity)
        qq, kk, vv = q.clone(), k.clone(), v.clone()
        at = ctx[row] - 1 if where != "first key" else max(0, ctx[row] - window)
        page = int(tables[row, at // 16])
        if where == "query":
            qq[row, 1, 7] = math.nan
        elif where == "infinite query":
            qq[row, 1, 7] = math.inf  # scores of both signs: infinity less infinity
        elif where == "value":
            vv[page, 0, at % 16, 9] = math.nan
        else:
            kk[page, 0, at % 16, 9] = math.nan
        out = torch.full(q.shape, 5.0, dtype=dt, device=DEV)
        sync_ok(run_rows(qq, kk, vv, tables, rt, ctx, window, 0, out))
        want, _, absv, smax = ref.window_rows(qq, kk, vv, tables, rt, ctx, window, 0, ref.scale_of(d))
        assert want.isnan().any()
        same_nans(out, want, clean, ref.bound(dt, want, absv, smax, max(ctx), d))
        # every key of a head whose sum is NaN gets NaN, no other key does
        w, o = torch.zeros_like(w_clean), torch.full(q.shape, 5.0, dtype=dt, device=DEV)
        sync_ok(run_weights(qq.to(DEV), kk.to(DEV), vv.to(DEV), tables.to(DEV), rt.to(DEV), ctx, o, w))
        want, add, _, _ = ref.window_rows(qq, kk, vv, tables, rt, ctx, 0, 0, ref.scale_of(d))
        assert torch.equal(o.cpu().isnan(), want.isnan())
        for r, n in enumerate(ctx):
            nan = add[r].isnan()
            got, base = w[r, :, :n].cpu(), w_clean[r, :, :n].cpu()
            assert torch.equal(got.isnan(), nan) and torch.equal(got[~nan], base[~nan])
    assert E.kernel_status(0) == 0


@pytest.mark.parametrize("name,group,hkv,d", [("bf16", 2, 2, 64), ("f16", 1, 2, 128)])
@pytest.mark.parametrize("window", [300, 2600])  # one CTA a tile, a cluster
def test_chunks_that_see_a_nan(name, group, hkv, d, window):
    dt, start, rows = DTYPES[name], 3000, 150
    g = torch.Generator().manual_seed(4)
    n = start + rows
    k, v = (torch.randn(n, hkv, d, generator=g).to(dt) for _ in range(2))
    q = torch.randn(rows, hkv * group, d, generator=g).to(dt)
    kp, vp, tables, rt = one_sequence(k, v)
    tl = tiles_of([(start, rows)], rt, group)

    def go(q, kp, vp):
        out = torch.full(q.shape, 5.0, dtype=dt, device=DEV)
        sync_ok(run_chunk(q, kp, vp, tables, tl, window, 0, out))
        return out

    def want(q, kp, vp):
        return ref.window_rows(q, kp, vp, tables, rt.expand(rows), [start + i + 1 for i in range(rows)], window, 0,
                               ref.scale_of(d))

    clean = go(q, kp, vp)
    base, _, absv, smax = want(q, kp, vp)
    tol = ref.bound(dt, base, absv, smax, n, d, exp_err=8e-5)
    assert bool(((clean.cpu().double() - base).abs() <= tol).all())
    for row in (0, 77, rows - 1):
        for bad in (math.nan, math.inf):
            qq = q.clone()
            qq[row, 1, 3] = bad
            exp = base.clone()
            exp[row, 1] = math.nan
            same_nans(go(qq, kp, vp), exp, clean, tol)
    # a key of each of 16 columns next to one another, seen by all rows and by some
    for key in [*range(start - 130, start - 114), start, start + 20, n - 1, start - window + 3]:
        kk = kp.clone()
        kk[int(tables[0, key // 16]), 0, key % 16, 5] = math.nan
        exp = base.clone()
        for i in range(rows):
            if key <= start + i and start + i - key < window:
                exp[i, :group] = math.nan
        got = go(q, kk, vp)
        same_nans(got, exp, clean, tol)
    assert E.kernel_status(0) == 0


@pytest.mark.parametrize("name,group,hkv,d", [("bf16", 2, 2, 64), ("bf16", 1, 2, 128)])
@pytest.mark.parametrize("window", [300, 2600])  # one CTA a tile, a cluster
def test_chunks_of_huge_scores(name, group, hkv, d, window):
    """Finite scores of any size: the key that is ahead takes the row, the ones behind have no part."""
    dt, start, rows = DTYPES[name], 3000, 150
    g = torch.Generator().manual_seed(4)
    n = start + rows
    k, v = (torch.randn(n, hkv, d, generator=g).to(dt) for _ in range(2))
    q = torch.randn(rows, hkv * group, d, generator=g).to(dt)
    kp, vp, tables, rt = one_sequence(k, v)
    tl = tiles_of([(start, rows)], rt, group)

    def go(q, kp, vp):
        out = torch.full(q.shape, 5.0, dtype=dt, device=DEV)
        sync_ok(run_chunk(q, kp, vp, tables, tl, window, 0, out))
        return out

    # finite numbers whose product is infinite (not in f16: its products fit f32)
    for key in range(start - 130, start - 126):
        qq, kk = q.clone(), kp.clone()
        qq[40, 0, 5], kk[int(tables[0, key // 16]), 0, key % 16, 5] = 1e30, 1e30
        got = go(qq, kk, vp)
        assert got[40, 0].isnan().all() and not got[41].isnan().any()
    compared = 0
    # one key of each of 16 neighbouring columns, many keys (each a multiple of the last), all keys
    for size in (1e5, 3e7, 1e12, 1e30):
        for keys in [[start - 130 + i] for i in range(16)] + [list(range(start - 200, start, 16)), list(range(0, start - 20))]:
            kk = kp.clone()
            for i, key in enumerate(keys):
                kk[int(tables[0, key // 16]), 0, key % 16, 5] = size * (1 + i % 7) * (1 if len(keys) < 100 else -1)
            got = go(q, kk, vp).cpu().double()
            assert torch.isfinite(got).all()
            # Rows whose largest score stands 2^-14 of its size before the next (f32 scores are good to
            # d 2^-23 of it) are one value, rounded once with a weight rounded once.
            half = torch.finfo(dt).eps / 2
            pos, at = torch.arange(start, n)[:, None], torch.arange(n)[None]
            seen = (at <= pos) & (pos - at < window)
            for h in range(group):
                s = (q[:, h].double() @ ref.paged(kk, tables[0], 0, n).double().T * ref.scale_of(d)).masked_fill(~seen, -math.inf)
                top = s.topk(2, -1)
                ahead = top.values[:, 0] - top.values[:, 1] > (2.0 ** -14 * s.masked_fill(~seen, 0).abs().amax(-1)).clamp(min=60.0)
                val = ref.paged(vp, tables[0], 0, n).double()[top.indices[:, 0]]
                off = (got[:, h] - val).abs() <= 2.02 * half * val.abs() + 1e-30
                assert bool(off[ahead].all()), (size, keys[:2], h)
                compared += int(ahead.sum())
    assert compared > 1000
    assert E.kernel_status(0) == 0


@pytest.mark.parametrize("name", ["bf16", "f32"])
@pytest.mark.parametrize("window", [60, 2000])  # one CTA a row, a cluster
def test_scores_of_minus_infinity_have_no_weight(name, window):
    """Finite keys whose product with the query is below the f32 range: weight 0, whole pages of
    them too, wherever they lie."""
    dt, d, n = DTYPES[name], 64, 2100
    g = torch.Generator().manual_seed(6)
    k, v = (torch.randn(n, 1, d, generator=g).to(dt) for _ in range(2))
    q = torch.randn(1, 2, d, generator=g).to(dt)
    q[..., 5] = 1e3
    k[..., 5] = 0.0
    for keys in (range(n - 60, n - 30), range(n - 20, n), range(0, n - 30), [n - 1], range(n - 40, n, 2)):
        kk = k.clone()
        kk[list(keys), :, 5] = -3e38
        kp, vp, tables, rt = one_sequence(kk, v)
        out = torch.full(q.shape, math.nan, dtype=dt, device=DEV)
        sync_ok(run_rows(q, kp, vp, tables, rt, [n], window, 0, out))
        # the reference without those keys' huge components: a score 10^4 below all others
        kk[list(keys), :, 5] = -80.0
        kp2 = one_sequence(kk, v)[0]
        want, _, absv, smax = ref.window_rows(q, kp2, vp, tables, rt, [n], window, 0, ref.scale_of(d))
        tol = ref.bound(dt, want, absv, torch.full_like(smax, 100.0), n, d)
        assert bool(((out.cpu().double() - want).abs() <= tol).all()), keys
        want, add, absv, smax = ref.window_rows(q, kp2, vp, tables, rt, [n], 0, 0, ref.scale_of(d))
        w = torch.zeros(1, 1, n, device=DEV)
        sync_ok(run_weights(q.to(DEV), kp.to(DEV), vp.to(DEV), tables.to(DEV), rt.to(DEV), [n], out, w))
        assert bool(((out.cpu().double() - want).abs() <= tol).all()), keys
        assert float((w[0].cpu().double() - add[0]).abs().max()) < 1e-4
        assert (w[0, 0, list(keys)] == 0).all()
        if dt != torch.float32:
            o = torch.full(q.shape, math.nan, dtype=dt, device=DEV)
            sync_ok(run_chunk(q, kp, vp, tables, tiles_of([(n - 1, 1)], rt, 2), 0, 0, o))
            assert bool(((o.cpu().double() - want).abs() <= tol + 2e-4 * absv).all()), keys
    assert E.kernel_status(0) == 0


@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
def test_large_numbers_that_no_row_sees(name):
    """Keys and values between the sinks and the window, on pages that hold seen keys too, change no bit."""
    dt, d, n, window, sinks = DTYPES[name], 128, 90, 40, 3
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(n, 2, d, generator=g).to(dt) for _ in range(2))
    q = torch.randn(5, 4, d, generator=g).to(dt)
    big = torch.finfo(dt).max

    def go(k, v, first):
        kp, vp, tables, rt = one_sequence(k, v)
        out = torch.full(q.shape, math.nan, dtype=dt, device=DEV)
        if first == n - 1:
            sync_ok(run_rows(q[:1], kp, vp, tables, rt, [n], window, sinks, out))
            return out[:1]
        tl = tiles_of([(first, n - first)], rt, 2)
        sync_ok(run_chunk(q, kp, vp, tables, tl, window, sinks, out))
        return out

    for first in [n - 1] + ([n - 5] if dt != torch.float32 else []):  # the row at n - 1; the rows from n - 5 on
        base = go(k, v, first)
        low = first + 1 - window  # the first key of the first row's window
        assert torch.isfinite(base).all() and low > 40
        for at in (3, 15, 16, 30, 40, low - 1):
            for sign in (1, -1):
                kk, vv = k.clone(), v.clone()
                kk[at], vv[at] = sign * big, -sign * big
                assert torch.equal(go(kk, vv, first), base), (first, at)
    # keys that the chunk's first rows see and its last do not, and the other way round
    if dt != torch.float32:
        first = n - 5
        base = go(k, v, first)
        for at, sees in ((first + 1 - window, [0]), (n - 2, [3, 4])):
            vv = v.clone()
            vv[at] = big
            got = go(k, vv, first)
            for r in range(5):
                assert torch.equal(got[r], base[r]) == (r not in sees), (at, r)
    assert E.kernel_status(0) == 0
