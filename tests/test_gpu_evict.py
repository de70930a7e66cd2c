"""Eviction from the paged cache (ms_launch_evict): which slots stay, where the
others go, and what is left alone, all bit for bit against the definition
restated in oracle.bounded_cache_ref; then the operators together, as a
sequence with a bounded cache uses them."""
import math

import numpy as np
import pytest
import torch

from mini_serve_rs_b200 import engine as E
from oracle import bounded_cache_ref as ref
from tests.gpu_util import dt_code, need_gpu, ptr, sync_ok
from tests.test_gpu_window import check, run_rows, run_weights, tiles_of

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    need_gpu()
    E.kernel_status(0)


def state(ctx, hkv, d, dt, seed, extra=5, tables_extra=2):
    g = torch.Generator().manual_seed(seed)
    n = len(ctx)
    blocks = -(-max(ctx) // 16) + 1
    pool = n * blocks + 3
    s = {"tables": torch.randperm(pool, generator=g)[:n * blocks].reshape(n, blocks).to(torch.int32)}
    s["tables"] = torch.cat([s["tables"], torch.full((tables_extra, blocks), -1, dtype=torch.int32)])
    s["rt"] = torch.randperm(n, generator=g).to(torch.int32)
    if dt == torch.float32:
        s["k"], s["v"] = (torch.randn(pool, hkv, 16, d, generator=g) for _ in range(2))
    else:  # any bit pattern is moved as it is
        s["k"], s["v"] = (torch.randint(-2 ** 15, 2 ** 15, (pool, hkv, 16, d), generator=g).to(torch.int16).view(dt)
                          for _ in range(2))
    stride = max(ctx) + extra
    rows = n + tables_extra
    s["w"] = torch.exp(2 * torch.randn(rows, hkv, stride, generator=g))
    s["pos"] = torch.zeros(rows, hkv, stride, dtype=torch.int32)
    s["ctx"] = ctx
    return s


def launch(s, keep, sinks, recent, nxt, known, w_in, w_out, pos_in, pos_out, k, v, dt, max_ctx=None, ws=None, stream=None,
           rt=None, tables=None):
    lib = E.lib()
    i32 = lambda x: torch.as_tensor(x, dtype=torch.int32).to(DEV)
    rows, hkv, mc = len(s["ctx"]), k.shape[1], max_ctx or max(s["ctx"])
    need = lib.ms_evict_workspace_bytes(rows, hkv, mc)
    ws = torch.empty(max(need, 1), dtype=torch.uint8, device=DEV) if ws is None else ws
    tables = s["tables"] if tables is None else tables
    rt = s["rt"] if rt is None else rt
    return lib.ms_launch_evict(ptr(k), ptr(v), k.shape[0], ptr(tables.to(DEV)), tables.shape[0], tables.shape[1],
                               ptr(rt.to(DEV)), ptr(i32(s["ctx"])), ptr(i32(nxt)),
                               ptr(None if known is None else i32(known)), rows, mc, keep, sinks, recent, ptr(w_in),
                               ptr(w_out), ptr(pos_in), ptr(pos_out), w_in.shape[-1], hkv, k.shape[-1], 16, ptr(ws),
                               ws.numel(), {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[dt], stream)


def expect(s, keep, sinks, recent, nxt, known, w_out, pos_out):
    k, v = s["k"].clone(), s["v"].clone()
    w_out, pos_out = w_out.clone(), pos_out.clone()
    for r, n in enumerate(s["ctx"]):
        t = int(s["rt"][r])
        page = lambda j: s["tables"][t][torch.as_tensor(j) // 16].long()
        for h in range(k.shape[1]):
            src, place = ref.evict(s["w"][t, h].numpy(), s["pos"][t, h].numpy(), n, nxt[r], known[r], keep, sinks, recent)
            m = min(n, keep)
            to = np.flatnonzero(src != np.arange(m))
            of = src[to]
            k[page(to), h, to % 16] = s["k"][page(of), h, of % 16]
            v[page(to), h, to % 16] = s["v"][page(of), h, of % 16]
            w_out[t, h, :m], w_out[t, h, m:n] = s["w"][t, h][src], 0
            pos_out[t, h, :m] = torch.from_numpy(place.astype(np.int32))
    return k, v, w_out, pos_out


def bits(t):
    return t.contiguous().view(torch.uint8).cpu()


def run(s, keep, sinks, recent, nxt, known, dt, in_place):
    w = s["w"].to(DEV)
    pos = s["pos"].to(DEV)
    w_out = w if in_place else torch.full_like(w, 9.0)
    pos_out = pos if in_place else torch.full_like(pos, -9)
    want = expect(s, keep, sinks, recent, nxt, known or [0] * len(nxt), w_out.cpu(), pos_out.cpu())
    k, v = s["k"].to(DEV), s["v"].to(DEV)
    sync_ok(launch(s, keep, sinks, recent, nxt, known, w, w_out, pos, pos_out, k, v, dt))
    assert E.kernel_status(0) == 0
    for got, exp, name in zip((pos_out, w_out, k, v), (want[3], want[2], want[0], want[1]), ("pos", "weight", "k", "v")):
        assert torch.equal(bits(got), bits(exp)), name


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("keep,sinks,recent", [(1, 0, 0), (1, 1, 0), (16, 0, 16), (33, 4, 5), (100, 0, 0), (100, 100, 0),
                                               (129, 4, 64), (700, 4, 100), (5000, 1, 1)])
@pytest.mark.parametrize("extra", [3, 5])  # the stride: a multiple of 4, and not
def test_first_eviction(keep, sinks, recent, in_place, extra):
    ctx = [0, 1, 2, 16, 17, 34, 101, 130, 700, 1025]
    s = state(ctx, 3, 64, torch.bfloat16, keep, extra=extra)
    run(s, keep, sinks, recent, ctx, None, torch.bfloat16, in_place)


@pytest.mark.parametrize("name,d", [("f32", 128), ("f32", 64), ("bf16", 128), ("f16", 64)])
def test_types(name, d):
    dt = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]
    s = state([300, 450], 2, d, dt, d)
    run(s, 256, 4, 32, s["ctx"], None, dt, True)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("extra", [4, 5])
def test_later_eviction_goes_by_positions(in_place, extra):
    """Slots below row_known hold their own positions, in any order."""
    ctx, known = [300, 260, 200, 77], [256, 256, 0, 77]
    nxt = [900, 260 + 44, 200, 500]
    s = state(ctx, 2, 64, torch.bfloat16, 5, extra=extra)
    g = torch.Generator().manual_seed(1)
    for r, (c, kn, nx) in enumerate(zip(ctx, known, nxt)):
        for h in range(2):
            s["pos"][int(s["rt"][r]), h, :kn] = torch.randperm(nx - (c - kn), generator=g)[:kn].to(torch.int32)
    run(s, 250, 4, 100, nxt, known, torch.bfloat16, in_place)


@pytest.mark.parametrize("kind", ["zero", "one", "two values", "signed zeros", "nan and infinity", "negative", "denormal"])
def test_ties_and_special_weights(kind):
    s = state([513, 1100], 2, 64, torch.bfloat16, 3)
    w = s["w"]
    g = torch.Generator().manual_seed(2)
    pick = torch.randint(0, 4, w.shape, generator=g)
    if kind in ("zero", "one"):
        w.fill_(0.0 if kind == "zero" else 1.0)
    elif kind == "two values":
        w.copy_(torch.where(pick == 0, 2.0, 1.0))
    elif kind == "signed zeros":
        w.copy_(torch.where(pick < 2, -0.0, 0.0))
    elif kind == "nan and infinity":
        w.copy_(torch.where(pick == 0, math.nan, torch.where(pick == 1, math.inf, torch.where(pick == 2, -math.inf, w))))
        w[0, 0, ::7] = -math.nan
    elif kind == "negative":
        w.neg_()
    else:
        w.mul_(1e-42)
    run(s, 500, 3, 40, s["ctx"], None, torch.bfloat16, True)


@pytest.mark.parametrize("ctx,keep", [([5000, 4097], 4096), ([20000], 513), ([9000, 33], 8999), ([70000, 40000], 30001),
                                      ([140001], 1000), ([262144], 130000)])
def test_long(ctx, keep):
    s = state(ctx, 2, 64, torch.float16, keep)
    run(s, keep, 4, min(200, keep // 2), ctx, None, torch.float16, True)


def test_pages_whose_elements_pass_32_bits():
    hkv, d, dt, n, keep = 8, 128, torch.bfloat16, 100, 60
    pool = (2 ** 31 // (hkv * 16 * d)) + 40
    k, v = (torch.zeros(pool, hkv, 16, d, dtype=dt, device=DEV) for _ in range(2))
    assert k.numel() > 2 ** 31
    g = torch.Generator().manual_seed(8)
    pages = torch.tensor([pool - 1, 3, pool - 9, pool // 2, pool - 2, 0, pool - 30])
    s = {"tables": pages[None].to(torch.int32), "rt": torch.zeros(1, dtype=torch.int32), "ctx": [n],
         "w": torch.rand(1, hkv, n, generator=g), "pos": torch.zeros(1, hkv, n, dtype=torch.int32)}
    small_k, small_v = (torch.randn(7, hkv, 16, d, generator=g).to(dt) for _ in range(2))
    k[pages.to(DEV)], v[pages.to(DEV)] = small_k.to(DEV), small_v.to(DEV)
    w, pos = s["w"].to(DEV), s["pos"].to(DEV)
    sync_ok(launch(s, keep, 2, 5, [n], None, w, w, pos, pos, k, v, dt))
    assert E.kernel_status(0) == 0
    local = dict(s, k=small_k, v=small_v, tables=torch.arange(7, dtype=torch.int32)[None])
    want = expect(local, keep, 2, 5, [n], [0], s["w"], s["pos"])
    for got, exp in ((k[pages.to(DEV)], want[0]), (v[pages.to(DEV)], want[1]), (w, want[2]), (pos, want[3])):
        assert torch.equal(bits(got), bits(exp))


def test_many_rows():
    ctx = [40 + (i * 37) % 300 for i in range(200)]
    s = state(ctx, 2, 64, torch.bfloat16, 8)
    run(s, 128, 4, 32, ctx, None, torch.bfloat16, True)


def test_padded_batch():
    """Empty rows may name any table row, a used one or none, before it or after."""
    ctx = [100, 120]
    s = state(ctx, 2, 64, torch.bfloat16, 6)
    want = expect(s, 64, 4, 16, ctx, [0, 0], s["w"], s["pos"])
    w, pos, k, v = (s[n].to(DEV) for n in ("w", "pos", "k", "v"))
    padded = dict(s, ctx=[0, 100, 0, 120, 0])
    rt = torch.tensor([s["rt"][0], s["rt"][0], -7, s["rt"][1], s["rt"][1]], dtype=torch.int32)
    sync_ok(launch(padded, 64, 4, 16, [0, 100, -3, 120, 9], [0, 0, -1, 0, 0], w, w, pos, pos, k, v, torch.bfloat16, rt=rt))
    assert E.kernel_status(0) == 0
    for got, exp in ((k, want[0]), (v, want[1]), (w, want[2]), (pos, want[3])):
        assert torch.equal(bits(got), bits(exp))


def test_bad_rows_are_skipped_and_flagged():
    ctx = [100, 120, 140]
    s = state(ctx, 2, 64, torch.bfloat16, 6)
    w, pos, k, v = (s[n].to(DEV) for n in ("w", "pos", "k", "v"))
    launch_ok = dict(w_in=w, pos_in=None, dt=torch.bfloat16)

    def go(nxt=ctx, known=None, rt=None, c=None, tables=None):
        wo, po, kk, vv = torch.full_like(w, 9.0), torch.full_like(pos, -9), k.clone(), v.clone()
        t = dict(s, ctx=c or ctx)
        pin = torch.zeros_like(pos) if known is not None else None
        sync_ok(launch(t, 64, 4, 16, nxt, known, w, wo, pin, po, kk, vv, torch.bfloat16, max_ctx=140, rt=rt, tables=tables))
        return (wo, po, kk, vv), E.kernel_status(0)

    assert launch_ok
    good, st = go()
    assert st == 0
    t1 = int(s["rt"][1])
    twice = s["rt"].clone()
    twice[1] = twice[0]
    outside = s["rt"].clone()
    outside[1] = s["tables"].shape[0]
    below = s["rt"].clone()
    below[1] = -1
    for kw in (dict(c=[100, 141, 140]), dict(c=[100, -1, 140]), dict(nxt=[100, 119, 140]), dict(known=[0, -1, 0]),
               dict(rt=twice), dict(rt=outside), dict(rt=below)):
        got, st = go(**kw)
        assert st == 2, kw
        for a, b, first in zip(got[:2], good[:2], (9.0, -9)):
            assert (a[t1] == first).all()
            for r in (0, 2):
                assert torch.equal(a[int(s["rt"][r])], b[int(s["rt"][r])]), kw
        for a, b, start in zip(got[2:], good[2:], (k, v)):
            for r in range(3):
                pages = s["tables"][int(s["rt"][r])].long()
                assert torch.equal(bits(a[pages]), bits((start if r == 1 else b)[pages])), kw
    for page in (-1, k.shape[0], 2 ** 31 - 1, -2 ** 31):  # never dereferenced; the other rows are as before
        tables = s["tables"].clone()
        tables[t1, :4] = page
        got, st = go(tables=tables)
        assert st == 2
        for r in (0, 2):
            pages = s["tables"][int(s["rt"][r])].long()
            for a, b in zip(got[2:], good[2:]):
                assert torch.equal(bits(a[pages]), bits(b[pages]))


@pytest.mark.parametrize("n,keep", [(400, 200), (4000, 1500)])  # one launch, two launches
def test_stream_and_graph_replay(n, keep):
    ctx = [n, n - 67]
    s = state(ctx, 2, 64, torch.bfloat16, 7)
    want = expect(s, keep, 4, 50, ctx, [0, 0], torch.full_like(s["w"], 9.0), torch.full_like(s["pos"], -9))
    dev = {x: s[x].to(DEV) for x in ("w", "pos", "k", "v", "tables", "rt")}
    c = torch.tensor(ctx, dtype=torch.int32, device=DEV)
    lib = E.lib()
    need = lib.ms_evict_workspace_bytes(2, 2, n)

    def call(stream, o):
        assert lib.ms_launch_evict(ptr(o["k"]), ptr(o["v"]), s["k"].shape[0], ptr(dev["tables"]), s["tables"].shape[0],
                                   s["tables"].shape[1], ptr(dev["rt"]), ptr(c), ptr(c), None, 2, n, keep, 4, 50,
                                   ptr(dev["w"]), ptr(o["w"]), None, ptr(o["pos"]), s["w"].shape[-1], 2, 64, 16,
                                   ptr(o["ws"]), need, 1, stream) == 0

    def buffers():
        return {"k": s["k"].to(DEV), "v": s["v"].to(DEV), "w": torch.full_like(dev["w"], 9.0),
                "pos": torch.full_like(dev["pos"], -9), "ws": torch.empty(need, dtype=torch.uint8, device=DEV)}

    def check_all(o):
        for x, exp in zip(("k", "v", "w", "pos"), want):
            assert torch.equal(bits(o[x]), bits(exp)), x

    side = [torch.cuda.Stream() for _ in range(2)]
    got = [buffers() for _ in side]
    torch.cuda.synchronize()
    for st, o in zip(side, got):
        call(st.cuda_stream, o)
    torch.cuda.synchronize()
    for o in got:
        check_all(o)
    # one after the other in a stream, through the same workspace
    first, second = buffers(), buffers()
    second["ws"] = first["ws"]
    torch.cuda.synchronize()
    for o in (first, second):
        call(None, o)
    torch.cuda.synchronize()
    check_all(first)
    check_all(second)
    o = buffers()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(torch.cuda.current_stream().cuda_stream, o)
    graph.replay()
    graph.replay()  # the same weights again: the same moves of the same values
    torch.cuda.synchronize()
    check_all(o)
    assert E.kernel_status(0) == 0


@pytest.mark.parametrize("name", ["bf16", "f32"])
def test_the_operators_together(name):
    """A bounded cache from prompt to decode: a windowed prompt chunk (16-bit),
    decode steps that track weights, an eviction, appended tokens, a second
    eviction, and decode over what is left; against the reference run on the
    kept tokens themselves."""
    dt = {"bf16": torch.bfloat16, "f32": torch.float32}[name]
    hkv, group, d = 2, 2, 64
    hq, lens, keep, sinks, recent = hkv * group, [200, 90], 96, 4, 32
    g = torch.Generator().manual_seed(3)
    n, blocks = len(lens), 20
    tables = torch.randperm(n * blocks, generator=g).reshape(n, blocks).to(torch.int32)
    rt = torch.tensor([1, 0], dtype=torch.int32)
    total = [c + 40 for c in lens]
    keys = [torch.randn(t, hkv, d, generator=g).to(dt) for t in total]
    vals = [torch.randn(t, hkv, d, generator=g).to(dt) for t in total]
    k, v = (torch.zeros(n * blocks, hkv, 16, d, dtype=dt) for _ in range(2))
    ctx, seen = list(lens), list(lens)
    kd, vd, td, rd = k.to(DEV), v.to(DEV), tables.to(DEV), rt.to(DEV)
    held = [[list(range(c)) for _ in range(hkv)] for c in lens]  # position in each slot

    def put(i, slot, pos):
        page = int(tables[int(rt[i]), slot // 16])
        kd[page, :, slot % 16] = keys[i][pos].to(DEV)
        vd[page, :, slot % 16] = vals[i][pos].to(DEV)

    for i, c in enumerate(lens):
        for j in range(c):
            put(i, j, j)
    T = sum(lens)
    qp = (2 * torch.randn(T, hq, d, generator=g)).to(dt)
    rows = [j + 1 for c in lens for j in range(c)]
    rrt = torch.tensor([int(rt[i]) for i, c in enumerate(lens) for _ in range(c)], dtype=torch.int32)
    out = torch.zeros_like(qp).to(DEV)
    if name == "bf16":
        tl = tiles_of([(0, c) for c in lens], rt, group).to(DEV)
        sync_ok(E.lib().ms_launch_window_prefill(ptr(qp.to(DEV)), ptr(kd), ptr(vd), kd.shape[0], ptr(td), n, blocks, ptr(tl),
                                                 len(tl), 64, sinks, ptr(out), hq, hkv, d, 16, ref.scale_of(d), dt_code(qp),
                                                 None))
    else:  # f32 chunks run as rows
        sync_ok(run_rows(qp, kd, vd, td, rrt, rows, 64, sinks, out))
    want, _, absv, smax = ref.window_rows(qp, kd.cpu(), vd.cpu(), tables, rrt, rows, 64, sinks, ref.scale_of(d))
    check(out, want, absv, smax, max(lens), dt, exp_err=8e-5 if name == "bf16" else 2.0 ** -20)

    w = torch.zeros(n, hkv, blocks * 16, device=DEV)
    pos = torch.zeros(n, hkv, blocks * 16, dtype=torch.int32, device=DEV)
    known = [0, 0]
    for step in range(40):
        for i in range(n):  # the step's token
            put(i, ctx[i], seen[i])
            for h in range(hkv):
                held[i][h].append(seen[i])
            ctx[i] += 1
            seen[i] += 1
        q = (2 * torch.randn(n, hq, d, generator=g)).to(dt)
        o = torch.full(q.shape, math.nan, dtype=dt, device=DEV)
        before = w.clone()
        sync_ok(run_weights(q.to(DEV), kd, vd, td, rd, ctx, o, w))
        for i in range(n):  # on the held tokens, whatever their slots
            for h in range(hkv):
                at = torch.tensor(held[i][h])
                sl = slice(h * group, (h + 1) * group)
                want, p, absv, smax = ref.attend(q[i, sl], keys[i][at, h], vals[i][at, h],
                                                 torch.ones(len(at), dtype=torch.bool), ref.scale_of(d))
                check(o[i, sl], want, absv, smax, len(at), dt)
                add = (w - before)[int(rt[i]), h, :ctx[i]].cpu().double()
                assert float((add - p.sum(0)).abs().max()) < 1e-4
        if step in (7, 25):
            weights = w.cpu()
            s = dict(ctx=list(ctx), rt=rt, tables=tables)
            sync_ok(launch(s, keep, sinks, recent, seen, known, w, w, pos, pos, kd, vd, dt))
            for i in range(n):
                t = int(rt[i])
                for h in range(hkv):
                    src, place = ref.evict(weights[t, h].numpy(), held[i][h], ctx[i], seen[i], ctx[i], keep, sinks, recent)
                    held[i][h] = place.tolist()
                    m = min(ctx[i], keep)
                    assert pos[t, h, :m].tolist() == place.tolist()
                    assert set(range(sinks)) <= set(place.tolist())
                    assert set(range(seen[i] - recent, seen[i])) <= set(place.tolist())
            ctx = [min(c, keep) for c in ctx]
            known = list(ctx)
    assert E.kernel_status(0) == 0
