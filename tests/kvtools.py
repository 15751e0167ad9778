"""Workloads and plain 64-bit forms of the paged-KV operators, for the tests."""
import math

import numpy as np
import torch

from tensorcast_b200.kvcache import KvWorkload


def tables(tokens, page=16, kv_heads=2, dim=64, planes=2, spare=0, seed=0, extra=3, taken=0):
    """A workload of sequences of `tokens` tokens, each with `spare` unused pages more, in permuted
    slots; `extra` slots of the pool and the last `taken` of the permutation stay free. Returns it
    and the free slots."""
    pages = [-(-n // page) + spare for n in tokens]
    total = sum(pages)
    slots = np.random.default_rng(seed).permutation(total + extra + taken).astype(np.uint32)
    offs = np.concatenate([[0], np.cumsum(pages)]).astype(np.uint64)
    w = KvWorkload(planes, total + extra + taken, page, kv_heads * dim * 2, np.array(tokens, np.uint32), offs,
                   slots[:total].copy())
    return w, slots[total:].copy()


def make_pool(w, kv_heads, dim, dtype, seed=0, fill=None):
    """[planes, slots * page_tokens, kv_heads, dim] normal values; with `fill`, only the rows that a
    sequence of `w` holds are normal and every other value is `fill`."""
    g = torch.Generator().manual_seed(seed)
    pool = torch.randn((w.planes, w.pool_pages * w.page_tokens, kv_heads, dim), generator=g).to(dtype)
    if fill is not None:
        used = np.zeros(w.pool_pages * w.page_tokens, bool)
        for s in range(w.n_seq):
            used[token_rows(w, s)] = True
        pool[:, torch.from_numpy(~used)] = fill
    return pool


def token_rows(w, s, n=None):
    n = int(w.seq_tokens[s]) if n is None else n
    at = np.arange(n)
    table = w.page_table[int(w.page_offsets[s]):int(w.page_offsets[s + 1])].astype(np.int64)
    return table[at // w.page_tokens] * w.page_tokens + at % w.page_tokens


def attention(w, pool, layer, q, counts, window=0, sinks=0, scale=None, prefix_rows=None, tokens=None):
    """The definition in 64 bits: out, lse, weights (per sequence, [kv_heads, tokens]) and, for the
    error bounds, sum p |v| for every output element and the largest scaled sum |q||k| of every row."""
    pre = np.zeros(0, np.int64) if prefix_rows is None else prefix_rows
    q = q.double()
    heads, dim = q.shape[1:]
    kv_heads = pool.shape[2]
    group = heads // kv_heads
    scale = dim ** -0.5 if scale is None else scale
    out, mass = torch.zeros_like(q), torch.zeros_like(q)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)
    size = torch.zeros_like(lse)
    weights, first = [], 0
    for s, m in enumerate(counts):
        n = int(w.seq_tokens[s]) if tokens is None else int(tokens[s])
        rows = torch.from_numpy(np.concatenate([pre, token_rows(w, s, n)])).to(pool.device)
        k, v = (pool[2 * layer + i][rows].double() for i in range(2))
        at = torch.arange(len(pre) + n, device=pool.device)
        added = torch.zeros((kv_heads, n), dtype=torch.float64, device=pool.device)
        for i in range(m):
            pos = len(pre) + n - m + i
            see = at <= pos
            if window:
                see &= (at > pos - window) | (at < sinks)
            if not bool(see.any()):
                continue
            for h in range(heads):
                kk, vv, row = k[see, h // group], v[see, h // group], q[first + i, h]
                z = kk @ row * scale
                lse[first + i, h] = torch.logsumexp(z, 0)
                p = torch.exp(z - lse[first + i, h])
                out[first + i, h] = p @ vv
                mass[first + i, h] = p @ vv.abs()
                size[first + i, h] = (kk.abs() @ row.abs()).max() * scale
                added[h // group, (see.nonzero()[:, 0] - len(pre))[see.nonzero()[:, 0] >= len(pre)]] += \
                    p[see.nonzero()[:, 0] >= len(pre)]
        weights.append(added)
        first += m
    return out, lse, weights, mass, size


def bounds(ref, dtype, longest):
    """Elementwise bounds of out, lse, and the relative one of a weight.

    A score is a sum of `dim` exact products in 32 bits: whatever the order, and with a last place
    twice that of rounding to nearest, off by at most (dim + 8) 2^-23 of the sum of |q||k| (scaled).
    A weight then is off by twice that (its own score and lse), an exponential in 32 bits by 2^-21,
    and sums of `longest` terms by longest 2^-24. An output adds the rounding of each probability
    and of itself to the type, half a step each, and as much again as 2^-18 of the terms' size."""
    out, lse, _, mass, size = ref
    dim = out.shape[-1]
    score = (dim + 8) * 2.0 ** -23 * size
    weight = 2 * score + 2.0 ** -20 + longest * 2.0 ** -24
    half = torch.finfo(dtype).eps / 2
    # a subnormal result is off by half of the smallest subnormal step
    tiny = torch.finfo(dtype).smallest_normal * half
    return half * out.abs() * 1.01 + (half + weight[..., None] + 2.0 ** -18) * mass + tiny, \
        score + 2.0 ** -20 + longest * 2.0 ** -24 + lse.abs().nan_to_num(0, posinf=0) * 2.0 ** -22, weight


def evict(weights, n, budget, sinks, recent):
    """The kept indices, in order."""
    w = np.asarray(weights, np.float64).copy()
    if n <= budget:
        return np.arange(n)
    first, newest = min(sinks, budget), min(recent, max(budget - sinks, 0))
    middle = np.arange(first, n - newest)
    key = np.where(np.isnan(w[middle]), -np.inf, w[middle])
    nan_last = np.isnan(w[middle])
    order = np.lexsort((middle, nan_last, -key))
    best = middle[order][: budget - first - newest]
    return np.sort(np.concatenate([np.arange(first), best, np.arange(n - newest, n)]))
