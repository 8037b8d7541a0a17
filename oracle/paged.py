"""Oracle: paged KV cache of the attention layers -- TEST INFRASTRUCTURE ONLY.

Plain sequential restatements, float64 arithmetic: page tables and maps from
request lengths, causal attention of new tokens over the cache, and the
accepted path's rows moved to the tree's first positions.
"""
from __future__ import annotations

import numpy as np


def page_plan(cached, fresh, rows, table, held, stack, page):
    """Lists / arrays of one plan; table [R, max_pages] and held are changed in
    place, `stack` (list of free pages, top last) too.  Returns qo_indptr,
    kv_indptr, kv_indices, slot_map, positions as lists, or None (nothing
    changed) when the stack does not hold enough pages."""
    B = len(cached)
    need = [-(-(int(c) + int(f)) // page) for c, f in zip(cached, fresh)]
    back = sum(max(int(held[r]) - n, 0) for r, n in zip(rows, need))
    take = sum(max(n - int(held[r]), 0) for r, n in zip(rows, need))
    if take > len(stack) + back:
        return None
    for b in range(B):
        for p in range(need[b], int(held[rows[b]])):
            stack.append(int(table[rows[b]][p]))
    for b in range(B):
        for p in range(int(held[rows[b]]), need[b]):
            table[rows[b]][p] = stack.pop()
        held[rows[b]] = need[b]
    qo, kv, idx, slots, pos = [0], [0], [], [], []
    for b in range(B):
        n = int(cached[b]) + int(fresh[b])
        at = [int(table[rows[b]][j // page]) * page + j % page for j in range(n)]
        idx += at
        slots += at[int(cached[b]):]
        pos += range(int(cached[b]), n)
        qo.append(qo[-1] + int(fresh[b]))
        kv.append(kv[-1] + n)
    return qo, kv, idx, slots, pos


def chunk_attention(q, k_cache, v_cache, qo_indptr, kv_indptr, kv_indices, scale, bound_unit=None):
    """q [T, Hq, D], caches [slots, Hkv, D]; float64 o [T, Hq, D] (NaN rows stay
    NaN; rows outside every request NaN, rows that see nothing 0).

    With bound_unit u (half a step of the 16-bit type) also the error bound of
    a kernel that keeps scores, softmax and sums in fp32, rounds P to the type
    and rounds o once.  With w the weights, A = sum_j w_j |v_j|, per element:
      u |o|                   the output's rounding
      u A                     P's rounding, each w_j by at most u (l sums the unrounded P)
      2 (ds + 2^-20) A        a score off by ds moves every weight and their sum by e^ds - 1 each;
                              2^-20: the exponential's and the scaling's own few fp32 roundings,
                              at exponents up to 2^4 past the running maximum
      L 2^-23 A               the fp32 sums over L keys, twice 2^-24 for truncating adders
      L 2^-31 max|v|          float16 P: its smallest step against the largest weight
    ds = D 2^-23 scale max_j sum_d |q_d k_jd|: the dot products' fp32 sums.
    First order; u^2 terms are covered by a factor 1.01."""
    q, kc, vc = (np.asarray(x, np.float64) for x in (q, k_cache, v_cache))
    T, Hq, D = q.shape
    G = Hq // kc.shape[1]
    o = np.full((T, Hq, D), np.nan)
    bound = np.zeros((T, Hq, D))
    for b in range(len(qo_indptr) - 1):
        t0, t1 = int(qo_indptr[b]), int(qo_indptr[b + 1])
        idx = np.asarray(kv_indices[kv_indptr[b]:kv_indptr[b + 1]], np.int64)
        n, L = t1 - t0, len(idx)
        if n == 0:
            continue
        seen = np.arange(L)[None, :] <= (L - n + np.arange(n))[:, None]      # [n, L]
        some = seen.any(1)
        o[t0:t1][~some] = 0.0
        if not some.any():
            continue
        seen, rows = seen[some], t0 + np.nonzero(some)[0]
        for h in range(Hq):
            k, v, qh = kc[idx, h // G], vc[idx, h // G], q[rows, h]
            s = np.where(seen, (qh @ k.T) * scale, -np.inf)
            w = np.exp(s - s.max(1, keepdims=True))
            w /= w.sum(1, keepdims=True)
            o[rows, h] = w @ v
            if bound_unit is not None:
                A = w @ np.abs(v)
                ds = D * 2.0 ** -23 * scale * np.where(seen, np.abs(qh) @ np.abs(k).T, 0.0).max(1)[:, None]
                bound[rows, h] = 1.01 * (bound_unit * np.abs(o[rows, h]) + bound_unit * A +
                                         2 * (ds + 2.0 ** -20) * A +
                                         seen.sum(1)[:, None] * (2.0 ** -23 * A + 2.0 ** -31 * np.abs(v).max()))
    return (o, bound) if bound_unit is not None else o


def kv_commit(k_cache, kv_indptr, kv_indices, path, accept_len, N):
    """Copy of k_cache [L, slots, ...] with the accepted rows moved."""
    out = np.array(k_cache, copy=True)
    for b in range(len(accept_len)):
        tree = kv_indices[kv_indptr[b + 1] - N:kv_indptr[b + 1]]
        for i in range(min(int(accept_len[b]), len(path[b]))):
            if path[b][i] < 0:
                break
            out[:, tree[i]] = k_cache[:, tree[path[b][i]]]
    return out
