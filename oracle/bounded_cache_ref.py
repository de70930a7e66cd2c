"""64-bit references of the operators that bound a sequence's cache: windowed
attention with sink tokens, attention weights, eviction (test infrastructure
only).  Each follows the operator's definition one row and head at a time."""
from __future__ import annotations

import math

import numpy as np
import torch


def visible(pos: int, window: int, sinks: int) -> torch.Tensor:
    """Mask over keys 0..pos of what the token at position pos sees."""
    j = torch.arange(pos + 1)
    if window <= 0:
        return torch.ones(pos + 1, dtype=torch.bool)
    return (j < sinks) | (pos - j < window)


def attend(q, k, v, see, scale):
    """One row of one kv head in f64.  q [G, D], k / v [n, D], see [n] bool.
    Returns out [G, D], weights [G, n], and for the error bounds
    sum_j p_j |v_j| [G, D] and max_j scale * sum_d |q_d k_jd| [G]."""
    q, k, v = q.double(), k.double()[see], v.double()[see]
    g, d = q.shape
    p_all = torch.zeros(g, see.numel(), dtype=torch.float64)
    if k.shape[0] == 0:
        z = torch.zeros(g, d, dtype=torch.float64)
        return z, p_all, z, torch.zeros(g, dtype=torch.float64)
    p = torch.softmax(q @ k.T * scale, -1)
    p_all[:, see] = p
    return p @ v, p_all, p @ v.abs(), (q.abs() @ k.abs().T).amax(-1) * abs(scale)


def bound(dtype, out, absv, smax, n, d, rounds_p=True, exp_err=2.0 ** -20):
    """Largest error of one f32 attention row whose result is rounded once to
    `dtype`, per element.  eps / 2 of the result for that rounding; relative to
    sum p |v|: eps / 2 where the kernel rounds p to the 16-bit type for the P.V
    product, exp_err twice (numerator and sum), each score's error twice
    (d products and their sums, one 2^-23 step each at most: the tensor cores
    may truncate), and one 2^-23 step per addition of the n terms and of the
    joins."""
    half = torch.finfo(dtype).eps / 2
    rel = 2 * exp_err + 2 * (d + 4) * 2.0 ** -23 * smax + (n + 64) * 2.0 ** -23
    if dtype != torch.float32 and rounds_p:
        rel = rel + half
    tiny = torch.finfo(dtype).smallest_normal
    return half * out.abs() * 1.001 + rel[..., None] * absv + tiny


def paged(pool, table, h, n):
    """Keys (values) 0..n-1 of kv head h through one block-table row."""
    return pool[table[: -(-n // 16)].long(), h].reshape(-1, pool.shape[-1])[:n]


def window_rows(q, k_pool, v_pool, tables, row_table, ctx, window, sinks, scale):
    """q [R, Hq, D].  Returns out, weights (list of [Hkv, ctx] sums over the kv
    head's query heads), absv, smax as attend()."""
    R, hq, d = q.shape
    hkv = k_pool.shape[1]
    g = hq // hkv
    out, absv = torch.zeros(R, hq, d, dtype=torch.float64), torch.zeros(R, hq, d, dtype=torch.float64)
    smax, weights = torch.zeros(R, hq, dtype=torch.float64), []
    for r in range(R):
        n = int(ctx[r])
        w = torch.zeros(hkv, n, dtype=torch.float64)
        for h in range(hkv):
            if n == 0:
                continue
            see = visible(n - 1, window, sinks)
            t = tables[int(row_table[r])]
            sl = slice(h * g, (h + 1) * g)
            out[r, sl], p, absv[r, sl], smax[r, sl] = attend(q[r, sl], paged(k_pool, t, h, n), paged(v_pool, t, h, n),
                                                             see, scale)
            w[h] = p.sum(0)
        weights.append(w)
    return out, weights, absv, smax


def evict(weight, pos, n, nxt, known, keep, sinks, recent):
    """One (sequence, kv head).  weight [n] f32, pos [>= known] int.  Returns
    (source slot of each slot of the first min(n, keep), their positions)."""
    place = np.arange(n, dtype=np.int64) - n + nxt
    place[:min(known, n)] = np.asarray(pos)[:min(known, n)]
    if n <= keep:
        return np.arange(n), place
    w = np.asarray(weight[:n], np.float64)
    safe = (place < sinks) | (place >= nxt - recent)
    rank = [(0 if safe[j] else 1, 0 if np.isnan(w[j]) else 1, 0.0 if np.isnan(w[j]) else -w[j], j) for j in range(n)]
    stay = np.zeros(n, bool)
    stay[[r[-1] for r in sorted(rank)[:keep]]] = True
    src = np.arange(keep)
    src[~stay[:keep]] = keep + np.flatnonzero(stay[keep:])
    return src, place[src]


def scale_of(d: int) -> float:
    return 1.0 / math.sqrt(d)
