"""Plain implementations, in 64 bits or with Python loops, of what a serving loop does to its batch around the paged
cache: head norms with positions, gathered attention weights, eviction by them, beam selection and reordering.
numpy on the CPU; no framework code.
"""
from __future__ import annotations

import math

import numpy as np

from . import cache_ops


def qk_norm(x, weight, eps):
    """x [B, QL, H, D] normalised over D, times weight ([D], [H, D] or None), in float64."""
    y = x.astype(np.float64)
    y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps)
    return y if weight is None else y * weight.astype(np.float64)


def qk_norm_rotary(x, weight, eps, inv_freq, pos, interleaved, mscale):
    return cache_ops.rotary(qk_norm(x, weight, eps), inv_freq, pos, interleaved, mscale)


def attn_weights(q, kc, ks, bt, ctx, w, q_lens, sm_scale):
    """(weights afterwards, a bound's worth of them): float64; the second is sum_r p_r A_r, A_r the largest sum of
    |q_d k_d| ks sm_scale over the tokens that row r sees."""
    P, PAGE, HK, D = kc.shape
    G = q.shape[2] // HK
    w, spread = w.astype(np.float64).copy(), np.zeros(w.shape)
    for b, ql in enumerate(q_lens):
        L = min(max(int(ctx[b]), 0), bt.shape[1] * PAGE)
        if L == 0 or ql == 0:
            continue
        pages = bt[b, np.arange(L) // PAGE]
        there = (pages >= 0) & (pages < P)
        pg, sl = np.where(there, pages, 0), np.arange(L) % PAGE
        for h in range(HK):
            k = kc[pg, sl, h].astype(np.float64)
            s = ks[pg, sl, h].astype(np.float64) * sm_scale
            got, size = np.zeros(L), np.zeros(L)
            for i in range(ql):
                seen = there & (np.arange(L) <= L - ql + i)
                if not seen.any():
                    continue
                for g in range(G):
                    row = q[b, i, h * G + g].astype(np.float64)
                    x = np.where(seen, (k @ row) * s, -np.inf)
                    a = (np.where(seen, np.abs(k) @ np.abs(row) * np.abs(s), 0)).max()
                    p = np.exp(x - x[seen].max())
                    p[~seen] = 0
                    p /= p.sum()
                    got += p
                    size += p * a
            w[b, h, max(L - ql, 0):L] = 0
            w[b, h, :L] += got
            spread[b, h, :L] = size
    return w, spread


def evict(bt, ctx, w, caches, budget, recent, sinks, limit, ref=None):
    """(kept, ctx, weights, caches) afterwards; caches [pages, PAGE, H_KV, ...]."""
    ctx, w, caches = ctx.copy(), w.copy(), [c.copy() for c in caches]
    B, HK, _ = w.shape
    P, PAGE = caches[0].shape[:2]
    kept = np.full((B, HK, budget), -1, np.int32)
    for b in range(B):
        L = min(max(int(ctx[b]), 0), bt.shape[1] * PAGE)
        pages = bt[b, :-(-L // PAGE)]
        ok = L > limit and ((pages >= 0) & (pages < P)).all() and (ref is None or (ref[pages] <= 1).all())
        if not ok:
            kept[b, :, :min(L, budget)] = np.arange(min(L, budget))
            continue
        for h in range(HK):
            key = [(-math.inf if math.isnan(x) else float(x)) for x in w[b, h, :L]]
            held = set(range(sinks)) | set(range(L - recent, L))
            others = sorted((t for t in range(L) if t not in held), key=lambda t: (-key[t], t))
            src = sorted(held | set(others[:budget - len(held)]))
            kept[b, h] = src
            w[b, h, :budget] = w[b, h, src].copy()
            t, j = np.array(src), np.arange(budget)
            for c in caches:
                c[bt[b, j // PAGE], j % PAGE, h] = c[bt[b, t // PAGE], t % PAGE, h].copy()
        ctx[b] = budget
    return kept, ctx, w, caches


def beam_select(logits, scores, n, finished=None, eos=None):
    """(scores float64, tokens, parents) of the best n, and of the one behind them its score."""
    B, W, V = logits.shape
    best = np.full((B, n), -np.inf)
    token, parent, behind = np.full((B, n), -1, np.int32), np.full((B, n), -1, np.int32), np.full(B, -np.inf)
    for b in range(B):
        flat = np.full((W, V), -np.inf)
        for w in range(W):
            x, c = logits[b, w].astype(np.float64), float(scores[b, w])
            if finished is not None and finished[b, w]:
                flat[w, eos] = c
                continue
            m = x.max()
            if not np.isfinite(m) or np.isnan(x).any():
                continue
            flat[w] = (x - (m + np.log(np.exp(x - m).sum()))) + c
        with np.errstate(over="ignore"):
            flat = np.where(flat.astype(np.float32) > -np.inf, flat, -np.inf).ravel()  # as it is given out
        order = np.argsort(-flat, kind="stable")
        order = order[flat[order] > -np.inf]
        k = min(n, len(order))
        best[b, :k], token[b, :k], parent[b, :k] = flat[order[:k]], order[:k] % V, b * W + order[:k] // V
        if len(order) > n:
            behind[b] = flat[order[n]]
    return best, token, parent, behind


def reorder(states, parents, group):
    rows = len(parents)
    at = np.array([p if r // group == p // group and p >= 0 else r for r, p in enumerate(parents)], np.int64)
    assert rows % group == 0
    return [s[at] for s in states]
