"""Cases of the operators that bound a sequence's KV cache, with their plain forms.

Four operators over the paged pools (k_pool / v_pool [pool_blocks, kv heads, 16, head_dim], block tables
[sequences, max_blocks] of page ids):

* "window":  attention of single tokens with a sliding window and sink tokens;
* "chunk":   attention of chunks of new tokens with a sliding window and sink tokens;
* "weights": attention of single tokens over the whole cache, adding each key's weight to an accumulator;
* "evict":   eviction from the cache by accumulated weight.

`own` false: elementary torch operations in 32 bits, rounded once.  `own` true: the library's calls.
"""
import math
import random

import numpy as np
import torch

own = False

PAGE = 16
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
CODES = {"f32": 0, "bf16": 1, "f16": 2}


def listed():
    return [
        # one chat, the smallest call: a decode step of Qwen3-0.6B's heads inside a 1024-token window
        dict(name="window 1 row", op="window", dtype="bf16", rows=1, hq=16, hkv=8, d=128, lo=1500, hi=1500, window=1024, sinks=4),
        # a serving batch of Qwen2.5-7B's heads, contexts up to 16k, a 4096-token window
        dict(name="window 64 rows", op="window", dtype="bf16", rows=64, hq=28, hkv=4, d=128, lo=700, hi=16384, window=4096, sinks=4),
        # the f32 parity mode, an odd window that ends inside a page, no sinks
        dict(name="window f32 24 rows", op="window", dtype="f32", rows=24, hq=16, hkv=8, d=128, lo=1, hi=2999, window=1001, sinks=0),
        # a chunked-prefill step: the next 512 tokens of one long prompt
        dict(name="chunk 512 of 8192", op="chunk", dtype="bf16", seqs=1, hq=16, hkv=8, d=128, lo=512, hi=512, start=7680, window=4096, sinks=4),
        # whole prompts of 4096 tokens prefilled in one step
        dict(name="chunk 4 x 4096", op="chunk", dtype="bf16", seqs=4, hq=16, hkv=8, d=128, lo=4096, hi=4096, start=0, window=2048, sinks=4),
        # a ragged step of a small model with 64-wide heads in f16, odd starts and lengths
        dict(name="chunk ragged f16", op="chunk", dtype="f16", seqs=9, hq=8, hkv=8, d=64, lo=5, hi=801, start=333, window=500, sinks=17),
        # one chat whose cache is tracked, the smallest call
        dict(name="weights 1 row", op="weights", dtype="bf16", rows=1, hq=16, hkv=8, d=128, lo=2177, hi=2177),
        # a serving batch at the budget of its caches
        dict(name="weights 64 rows", op="weights", dtype="bf16", rows=64, hq=16, hkv=8, d=128, lo=2048, hi=4608),
        # long caches of Qwen2.5-7B's heads in f16, before their first eviction
        dict(name="weights 12 long rows", op="weights", dtype="f16", rows=12, hq=28, hkv=4, d=128, lo=9000, hi=16385),
        # one chat that outgrew its budget by eight pages
        dict(name="evict 1 to 2048", op="evict", dtype="bf16", rows=1, hkv=8, d=128, lo=2176, hi=2176, keep=2048, sinks=4, recent=128, known=2048),
        # a serving batch that outgrew its budget
        dict(name="evict 64 to 4096", op="evict", dtype="bf16", rows=64, hkv=8, d=128, lo=3900, hi=4608, keep=4096, sinks=4, recent=256, known=0),
        # long prompts cut to an eighth, 7B heads
        dict(name="evict 6 long prompts", op="evict", dtype="f16", rows=6, hkv=4, d=128, lo=20011, hi=32768, keep=4000, sinks=4, recent=500, known=0),
    ]


def _spread(rng, lo, hi):
    """A whole number whose logarithm is uniform in [lo, hi]."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["window", "chunk", "weights", "evict"])
    hq, hkv = rng.choice([(16, 8), (28, 4), (8, 8), (14, 2), (32, 4), (8, 2)])
    d = rng.choice([64, 128, 128])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op in ("window", "weights"):
        rows = _spread(rng, 1, 64)
        # at most about 120k keys in all: below the listed batches' work
        hi = _spread(rng, 1, min(16384, 120000 // rows))
        lo = rng.randint(1, hi)
        c = dict(op=op, dtype=dtype, rows=rows, hq=hq, hkv=hkv, d=d, lo=lo, hi=hi)
        if op == "window":
            c |= dict(window=_spread(rng, 1, 4096), sinks=rng.choice([0, 1, 4, 16, 33, 130]))
        return c
    if op == "chunk":
        seqs = rng.randint(1, 6)
        hi = _spread(rng, 1, 2048)
        return dict(op=op, dtype=rng.choice(["bf16", "f16"]), seqs=seqs, hq=hq, hkv=hkv, d=d, lo=rng.randint(1, hi), hi=hi,
                    start=rng.choice([0, rng.randint(1, 2500)]), window=_spread(rng, 1, 4096),
                    sinks=rng.choice([0, 1, 4, 16, 33, 130]))
    rows = _spread(rng, 1, 24)
    hi = _spread(rng, 2, min(32768, 200000 // rows))
    lo = rng.randint(1, hi)
    keep = rng.randint(1, hi)
    recent = rng.randint(0, keep // 2)
    return dict(op=op, dtype=dtype, rows=rows, hkv=hkv, d=d, lo=lo, hi=hi, keep=keep, sinks=min(rng.choice([0, 1, 4, 16]), keep - recent),
                recent=recent, known=rng.choice([0, rng.randint(0, lo)]))


def _lengths(case):
    """The sequences' lengths: fixed by the case, both ends of its range among them."""
    n = case.get("rows") or case["seqs"]
    lo, hi = case["lo"], case["hi"]
    r = random.Random("%d %d %d" % (n, lo, hi))
    got = [hi] + [r.randint(lo, hi) for _ in range(n - 2)] + [lo]
    return got[:n]


def _visible(ctx, case):
    """How many keys a token at position ctx - 1 sees."""
    w, s = case.get("window", 0), case.get("sinks", 0)
    low = max(0, ctx - w) if w > 0 else 0
    return ctx - low + min(s, low)


def work(case):
    es = 4 if case["dtype"] == "f32" else 2
    hkv, d, lens = case["hkv"], case["d"], _lengths(case)
    if case["op"] == "evict":
        b = 0
        for n in lens:
            keep = min(case["keep"], n)
            free = n - min(n, case["sinks"] + case["recent"])  # slots that the weights decide about
            share = max(0, keep - (n - free)) / free if free else 0
            tail = n - keep
            moved = min(keep, min(tail, case["recent"]) + max(0, tail - case["recent"]) * share)
            b += hkv * (4 * n + 4 * min(n, case["known"]) + 4 * n + 4 * keep + moved * 2 * d * es * 2)
        return {"bytes": b, "flops": 0}
    hq = case["hq"]
    if case["op"] == "chunk":
        b = f = 0
        for n in lens:
            end = case["start"] + n
            b += (_visible(case["start"] + 1, case) + n - 1) * hkv * d * 2 * es + 2 * n * hq * d * es
            p = np.arange(case["start"], end, dtype=np.int64) + 1
            low = np.maximum(0, p - case["window"])
            f += int((p - low + np.minimum(case["sinks"], low)).sum()) * hq * 4 * d
        return {"bytes": b, "flops": f}
    keys = sum(_visible(n, case) for n in lens)
    b = keys * hkv * d * 2 * es + 2 * len(lens) * hq * d * es + keys // PAGE * 4
    if case["op"] == "weights":
        b += keys * hkv * 8
    return {"bytes": b, "flops": keys * hq * 4 * d}


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    hkv, d, lens = case["hkv"], case["d"], _lengths(case)
    n = len(lens)
    ctx = [case["start"] + t for t in lens] if case["op"] == "chunk" else lens
    blocks = -(-max(ctx) // PAGE)
    pool = n * blocks + 5
    s = dict(case=dict(case), n=n, lens=lens, max_ctx=max(ctx), pool=pool, blocks=blocks)
    # pages of the sequences lie scattered over the pool, each with one owner
    s["tables"] = torch.randperm(pool, generator=g, device=dev)[: n * blocks].reshape(n, blocks).to(torch.int32).contiguous()
    for k in ("k", "v"):
        s[k] = torch.empty(pool, hkv, PAGE, d, dtype=dt, device=dev).normal_(generator=g)
    s["ctx"] = torch.tensor(ctx, dtype=torch.int32, device=dev)
    s["row_table"] = torch.randperm(n, generator=g, device=dev).to(torch.int32)
    if case["op"] == "evict":
        stride = -(-max(ctx) // 4) * 4
        # accumulated weights are heavy-tailed; a tenth of the slots has seen no query yet
        w = torch.exp(2 * torch.randn(n, hkv, stride, generator=g, device=dev))
        s["w"] = torch.where(torch.rand(n, hkv, stride, generator=g, device=dev) < 0.1, torch.zeros_like(w), w)
        s["w_out"], s["stride"] = torch.zeros_like(w), stride
        # positions of the slots that an earlier eviction left: some of the first, in any order
        s["next"] = s["ctx"] + (37 if case["known"] else 0)
        s["known"] = torch.full((n,), case["known"], dtype=torch.int32, device=dev)
        span = case["known"] + 37
        s["pos"] = torch.argsort(torch.rand(n, hkv, span, generator=g, device=dev), -1)[..., :stride].to(torch.int32)
        s["pos"] = torch.nn.functional.pad(s["pos"], (0, stride - s["pos"].shape[-1])).contiguous()
        s["pos_out"] = torch.zeros_like(s["pos"])
    else:
        # scores with a spread of about two, as after a query norm
        t = sum(lens) if case["op"] == "chunk" else n
        s["q"] = (2 * torch.randn(t, case["hq"], d, generator=g, device=dev)).to(dt)
        s["out"] = torch.zeros_like(s["q"])
    if case["op"] == "weights":
        s["stride"] = -(-max(ctx) // 4) * 4
        s["w"] = torch.rand(n, hkv, s["stride"], generator=g, device=dev)
    if case["op"] == "chunk":
        s["row0"] = [sum(lens[:i]) for i in range(n)]
        s["seq"] = torch.repeat_interleave(torch.arange(n, device=dev), torch.tensor(lens, device=dev))
        s["step"] = torch.cat([torch.arange(t, device=dev) for t in lens])
        # the prefill tiles of the step: at most 256 query rows of one kv head each, those that end last first
        group = case["hq"] // hkv
        size = 256 // (1 << (group - 1).bit_length())
        tiles = [(s["row0"][i] + j, min(size, lens[i] - j), case["start"] + j, t) for i, t in enumerate(s["row_table"].tolist())
                 for j in range(0, lens[i], size)]
        s["tiles"] = torch.tensor(sorted(tiles, key=lambda a: -a[1] - a[2]), dtype=torch.int32, device=dev)
    return s


_scratch = {}  # device -> the workspace that the program keeps for its calls, as large as its largest step


def _workspace(s, lib):
    c = s["case"]
    if c["op"] == "weights":
        need = lib.ms_attention_weights_workspace_bytes(s["n"], c["hq"], s["max_ctx"])
    else:
        need = lib.ms_evict_workspace_bytes(s["n"], c["hkv"], s["max_ctx"])
    dev = s["k"].device
    if dev not in _scratch or _scratch[dev].numel() < need:
        _scratch[dev] = torch.empty(need, dtype=torch.uint8, device=dev)
    return _scratch[dev]


def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    from mini_serve_rs_b200 import engine as E
    c, lib = s["case"], E.lib()
    stream = torch.cuda.current_stream().cuda_stream
    p = lambda t: t.data_ptr()  # noqa: E731
    code, scale = CODES[c["dtype"]], 1.0 / math.sqrt(c["d"])
    pools = (p(s["k"]), p(s["v"]), s["pool"], p(s["tables"]), s["n"], s["blocks"])
    if c["op"] == "window":
        rc = lib.ms_launch_window_attention(p(s["q"]), *pools, p(s["row_table"]), p(s["ctx"]), s["n"], s["max_ctx"], c["window"], c["sinks"],
                                            p(s["out"]), c["hq"], c["hkv"], c["d"], PAGE, scale, code, stream)
        got = s["out"]
    elif c["op"] == "chunk":
        rc = lib.ms_launch_window_prefill(p(s["q"]), *pools, p(s["tiles"]), len(s["tiles"]), c["window"], c["sinks"], p(s["out"]), c["hq"],
                                          c["hkv"], c["d"], PAGE, scale, code, stream)
        got = s["out"]
    elif c["op"] == "weights":
        ws = _workspace(s, lib)
        rc = lib.ms_launch_attention_weights(p(s["q"]), *pools, p(s["row_table"]), p(s["ctx"]), s["n"], s["max_ctx"], p(s["out"]), p(s["w"]),
                                             s["stride"], c["hq"], c["hkv"], c["d"], PAGE, scale, p(ws), ws.numel(), code, stream)
        got = (s["out"], s["w"])
    else:
        ws = _workspace(s, lib)
        rc = lib.ms_launch_evict(*pools, p(s["row_table"]), p(s["ctx"]), p(s["next"]), p(s["known"]), s["n"], s["max_ctx"], c["keep"], c["sinks"],
                                 c["recent"], p(s["w"]), p(s["w_out"]), p(s["pos"]), p(s["pos_out"]), s["stride"], c["hkv"], c["d"], PAGE,
                                 p(ws), ws.numel(), code, stream)
        got = (s["k"], s["v"], s["w_out"], s["pos_out"])
    if rc != 0:
        raise RuntimeError("%s returned %d" % (c["op"], rc))
    return got


def _rows(pool, table, keys):
    """Rows [n, m, kv heads, d] of a pool in 32 bits: keys [n, m] of the sequences with block-table rows `table` [n, blocks]."""
    page = torch.gather(table.long(), 1, keys // PAGE)
    return pool[page, :, keys % PAGE].float()


def _run_plain(s):
    return {"window": _plain_rows, "weights": _plain_rows, "chunk": _plain_chunk, "evict": _plain_evict}[s["case"]["op"]](s)


def _plain_rows(s):
    c, dev = s["case"], s["q"].device
    n, hkv, d = s["n"], c["hkv"], c["d"]
    ctx = s["ctx"].long()[:, None]
    w, sinks = c.get("window", 0), c.get("sinks", 0)
    low = (ctx - w).clamp(min=0) if w > 0 else torch.zeros_like(ctx)
    first = low.clamp(max=sinks)  # sink keys below the window
    most = min(s["max_ctx"], w + sinks) if w > 0 else s["max_ctx"]
    at = torch.arange(most, device=dev)[None]
    keys = torch.where(at < first, at, low + at - first)
    live = at < first + ctx - low
    keys = torch.where(live, keys, torch.zeros_like(keys))
    table = s["tables"][s["row_table"].long()]
    q = s["q"].float().reshape(n, hkv, -1, d)
    k, v = _rows(s["k"], table, keys).transpose(1, 2), _rows(s["v"], table, keys).transpose(1, 2)
    score = torch.matmul(q, k.transpose(2, 3)) * (1.0 / math.sqrt(d))
    score = score.masked_fill(~live[:, None, None], -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    out = torch.matmul(p, v).reshape(n, -1, d).to(s["q"].dtype)
    if c["op"] == "window":
        return out
    s["w"][s["row_table"].long(), :, : s["max_ctx"]] += p.sum(2)
    return out, s["w"]


def _plain_chunk(s):
    c, dev = s["case"], s["q"].device
    n, hkv, d = s["n"], c["hkv"], c["d"]
    most = max(s["lens"])
    keys = torch.arange(s["max_ctx"], device=dev)
    live = keys[None] < s["ctx"].long()[:, None]
    table = s["tables"][s["row_table"].long()]
    at = torch.where(live, keys[None], torch.zeros_like(keys)[None])
    k, v = _rows(s["k"], table, at).transpose(1, 2), _rows(s["v"], table, at).transpose(1, 2)
    q = torch.zeros(n, most, hkv, c["hq"] // hkv, d, device=dev)
    q[s["seq"], s["step"]] = s["q"].float().reshape(-1, hkv, c["hq"] // hkv, d)
    q = q.permute(0, 2, 3, 1, 4).reshape(n, hkv, -1, d)
    score = torch.matmul(q, k.transpose(2, 3)).reshape(n, hkv, -1, most, s["max_ctx"])
    score *= 1.0 / math.sqrt(d)
    pos = c["start"] + torch.arange(most, device=dev)[:, None]
    seen = (keys <= pos) & ((keys < c["sinks"]) | (pos - keys < c["window"]))
    score.masked_fill_(~seen, -math.inf)
    score -= score.amax(-1, keepdim=True)
    p = score.exp_()
    p /= p.sum(-1, keepdim=True)
    o = torch.matmul(p.reshape(n, hkv, -1, s["max_ctx"]), v).reshape(n, hkv, -1, most, d)
    return o.permute(0, 3, 1, 2, 4)[s["seq"], s["step"]].reshape(s["q"].shape).to(s["q"].dtype)


def _plain_evict(s):
    c, dev = s["case"], s["k"].device
    n, hkv, m = s["n"], c["hkv"], s["max_ctx"]
    rt = s["row_table"].long()
    at = torch.arange(m, device=dev)
    ctx, known, nxt = (s[k].long()[:, None, None] for k in ("ctx", "known", "next"))
    w, pos = s["w"][rt, :, :m], s["pos"][rt, :, :m].long()
    pos = torch.where(at < known, pos, nxt - (ctx - at))
    live = at < ctx
    rank = torch.where((pos < c["sinks"]) | (pos >= nxt - c["recent"]), torch.full_like(w, math.inf), w)
    rank = torch.where(live, rank, torch.full_like(w, -math.inf))
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices
    kept = torch.zeros_like(live.expand(n, hkv, m)).scatter(-1, order[..., : c["keep"]], True) & live
    # the kept slots from `keep` on, in order, and the slot that each evicted one below takes
    high = at >= c["keep"]
    mover = torch.sort(torch.where(kept & high, at, torch.full_like(at, m)), -1).values
    hole = ~kept & ~high & live
    nth = (hole.cumsum(-1) - 1).clamp(min=0)
    src = torch.where(hole, torch.gather(mover, -1, nth), at.expand(n, hkv, m))
    top = min(c["keep"], m)
    src, keepers = src[..., :top], at[:top].expand(n, hkv, top)
    table = s["tables"][rt].long()[:, None].expand(n, hkv, -1)
    heads = torch.arange(hkv, device=dev)[None, :, None]
    to, of = torch.gather(table, 2, keepers // PAGE), torch.gather(table, 2, src // PAGE)
    for name in ("k", "v"):
        s[name][to, heads, keepers % PAGE] = s[name][of, heads, src % PAGE]
    head = torch.where(live[..., :top], torch.gather(w, -1, src), s["w_out"][rt, :, :top])
    rest = torch.where(live[..., top:], torch.zeros_like(w[..., top:]), s["w_out"][rt, :, top:m])
    s["w_out"][rt, :, :m] = torch.cat([head, rest], -1)
    s["pos_out"][rt, :, :top] = torch.where(live[..., :top], torch.gather(pos, -1, src).to(torch.int32), s["pos_out"][rt, :, :top])
    return s["k"], s["v"], s["w_out"], s["pos_out"]


def exact(case, seed):
    """The definition in 64 bits, one sequence (and query head) at a time."""
    s = prepare(case, seed)
    if case["op"] == "evict":
        return _exact_evict(s)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    rt = s["row_table"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    add = s["w"].double() if case["op"] == "weights" else None
    row = 0
    for i, n in enumerate(s["lens"]):
        chunk = case["op"] == "chunk"
        count, end = (n, case["start"] + n) if chunk else (1, n)
        pages = s["tables"][rt[i], : -(-end // PAGE)].long()
        p = torch.arange(end - count, end, device=out.device)[:, None]
        j = torch.arange(end, device=out.device)[None]
        see = j <= p
        if "window" in case:
            see = see & ((j < case["sinks"]) | (j > p - case["window"]))
        for h in range(hq):
            kv = h // (hq // hkv)
            k = s["k"][pages, kv].reshape(-1, d)[:end].double()
            v = s["v"][pages, kv].reshape(-1, d)[:end].double()
            a = torch.where(see, (s["q"][row: row + count, h].double() @ k.T) / math.sqrt(d), -math.inf)
            a = torch.softmax(a, -1)
            out[row: row + count, h] = a @ v
            if add is not None:
                add[rt[i], kv, :end] += a[0]
        row += count
    return (out, add) if add is not None else out


def _exact_evict(s):
    c = s["case"]
    rt = s["row_table"].tolist()
    w, pos, tables = s["w"].cpu().numpy(), s["pos"].cpu().numpy(), s["tables"].cpu().numpy()
    w_out, pos_out = s["w_out"].double().cpu().numpy(), s["pos_out"].cpu().numpy()
    ctx, nxt, known = s["ctx"].tolist(), s["next"].tolist(), s["known"].tolist()
    moves = []  # (page to, page from, head, slot to, slot from)
    for i, t in enumerate(rt):
        n, keep = ctx[i], min(c["keep"], ctx[i])
        for h in range(c["hkv"]):
            place = np.arange(n) - n + nxt[i]
            place[: known[i]] = pos[t, h, : min(known[i], n)]
            safe = (place < c["sinks"]) | (place >= nxt[i] - c["recent"])
            best = np.lexsort((np.arange(n), -w[t, h, :n].astype(np.float64), ~safe))[:keep]
            stay = np.zeros(n, bool)
            stay[best] = True
            src = np.arange(keep)
            src[~stay[:keep]] = keep + np.flatnonzero(stay[keep:])
            w_out[t, h, :n] = 0
            w_out[t, h, :keep], pos_out[t, h, :keep] = w[t, h, src], place[src]
            to = np.flatnonzero(src != np.arange(keep))
            moves.append(np.stack([tables[t, to // PAGE], tables[t, src[to] // PAGE], np.full(len(to), h), to % PAGE, src[to] % PAGE]))
    to, of, h, at, was = torch.from_numpy(np.concatenate(moves, 1).astype(np.int64)).to(s["k"].device)
    k, v = s["k"].clone(), s["v"].clone()
    k[to, h, at], v[to, h, at] = s["k"][of, h, was], s["v"][of, h, was]
    return k, v, torch.from_numpy(w_out), torch.from_numpy(pos_out)
