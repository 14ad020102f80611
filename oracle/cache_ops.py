"""Plain implementations, in 64 bits or with Python loops, of the steps around a paged cache with block
scales: rotary positions, append, attention and page tables.  numpy on the CPU; no framework code.
"""
from __future__ import annotations

import numpy as np

QMAX = {"int8": np.float32(127.0), "fp8": np.float32(448.0)}


def _e4m3_values():
    """The value of every e4m3 code (fn flavour: no infinities, 0x7f and 0xff NaN)."""
    v = np.empty(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        x = (m / 8) * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        v[c] = np.nan if (c & 127) == 127 else (-x if c & 128 else x)
    return v


E4M3 = _e4m3_values()


def decode(codes, fmt):
    """Codes (int8, or uint8 bytes of e4m3) as float64."""
    return codes.astype(np.float64) if fmt == "int8" else E4M3[codes]


def encode(x, fmt):
    """float64 values to the nearest codes, ties to even, clamped to the largest; e4m3 has a code for NaN."""
    m = float(QMAX[fmt])
    if fmt == "int8":
        return np.clip(np.rint(x), -m, m).astype(np.int8)
    mag = E4M3[:127]  # 0 .. 448, rising with the code
    a = np.minimum(np.abs(x), m)
    hi = np.minimum(np.searchsorted(mag, a, side="left"), 126)
    lo = np.maximum(hi - 1, 0)
    dl, dh = a - mag[lo], mag[hi] - a
    code = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    code = np.where(np.isnan(x), 127, code)
    return (code | (np.signbit(x).astype(np.int64) << 7)).astype(np.uint8)


def rotary(x, inv_freq, pos, interleaved, mscale):
    """x [B, QL, H, D] at pos [B, QL], in float64."""
    y = x.astype(np.float64)
    R = 2 * len(inv_freq)
    ang = pos[..., None].astype(np.float64) * np.asarray(inv_freq, np.float64)
    c, s = mscale * np.cos(ang)[:, :, None], mscale * np.sin(ang)[:, :, None]
    i0, i1 = (np.arange(0, R, 2), np.arange(1, R, 2)) if interleaved else (np.arange(R // 2), np.arange(R // 2, R))
    a, b = y[..., i0].copy(), y[..., i1].copy()
    y[..., i0], y[..., i1] = a * c - b * s, b * c + a * s
    return y


def append_block(k_new, v_new, kc, vc, ks, vs, bt, ctx, q_len, fmt, n_seqs=None):
    """The cache after the append: scales and quotients in fp32 as the format defines them, so that codes can be
    compared bit for bit.  Codes are int8, or uint8 bytes of e4m3."""
    kc, vc, ks, vs = (a.copy() for a in (kc, vc, ks, vs))
    P, PAGE, H, _ = kc.shape
    SB = PAGE // ks.shape[1]
    f32 = np.float32
    for b in range(len(ctx) if n_seqs is None else n_seqs):
        if q_len == 0:
            break
        p0 = int(ctx[b]) - q_len
        first = max(p0, 0)
        for lo in range(first // SB * SB, int(ctx[b]), SB):
            if lo // PAGE >= bt.shape[1]:
                break
            pg, hi = int(bt[b, lo // PAGE]), min(lo + SB, int(ctx[b]))
            if not 0 <= pg < P:
                continue
            at, blk, start = lo % PAGE, lo % PAGE // SB, max(first, lo)
            for new, codes, scale in ((k_new, kc, ks), (v_new, vc, vs)):
                for h in range(H):
                    x = new[b, start - p0:hi - p0, h].astype(f32)
                    x = np.clip(np.where(np.isnan(x), f32(0), x), f32(-65504), f32(65504))
                    s = max(np.abs(x).max(), f32(1e-8)) / QMAX[fmt]
                    n_old = start - lo
                    if n_old:
                        was = scale[pg, blk, h]
                        if s > was:
                            old = decode(codes[pg, at:at + n_old, h], fmt).astype(f32) * was
                            codes[pg, at:at + n_old, h] = encode((old / s).astype(np.float64), fmt)
                        s = max(s, was)
                    codes[pg, at + n_old:at + hi - lo, h] = encode((x / f32(s)).astype(np.float64), fmt)
                    scale[pg, blk, h] = s
    return kc, vc, ks, vs


def attention_block(q, kc, vc, ks, vs, bt, ctx, q_len, fmt, n_seqs=None, sm_scale=None):
    """(out, spread) in float64: spread bounds what a relative error of the probabilities does, sum p |v|; and the
    largest sum |q k| of a score.  Rows that see nothing are 0."""
    B, QL, H, D = q.shape
    P, PAGE, HK, _ = kc.shape
    SB, G = PAGE // ks.shape[1], H // HK
    sm = 1 / np.sqrt(D) if sm_scale is None else sm_scale
    out, spread, big = np.zeros(q.shape), np.zeros(q.shape), 0.0
    for b in range(B if n_seqs is None else n_seqs):
        L = min(int(ctx[b]), bt.shape[1] * PAGE)
        t = np.arange(max(L, 0))
        pg = bt[b, t // PAGE].astype(np.int64) if L > 0 else np.zeros(0, np.int64)
        ok = (pg >= 0) & (pg < P)
        t, pg = t[ok], pg[ok]
        for h in range(HK):
            k = decode(kc[pg, t % PAGE, h], fmt) * ks[pg, t % PAGE // SB, h].astype(np.float64)[:, None]
            v = decode(vc[pg, t % PAGE, h], fmt) * vs[pg, t % PAGE // SB, h].astype(np.float64)[:, None]
            for i in range(q_len):
                n = int((t <= L - q_len + i).sum())
                if n == 0:
                    continue
                qq = q[b, i, h * G:(h + 1) * G].astype(np.float64)
                s = qq @ k[:n].T * sm
                p = np.exp(s - s.max(-1, keepdims=True))
                p /= p.sum(-1, keepdims=True)
                out[b, i, h * G:(h + 1) * G] = p @ v[:n]
                spread[b, i, h * G:(h + 1) * G] = p @ np.abs(v[:n])
                big = max(big, float((np.abs(qq) @ np.abs(k[:n]).T).max()) * abs(sm))
    return out, spread, big


# ----------------------------------------------------------------------------------------
# Page tables, one entry at a time
# ----------------------------------------------------------------------------------------
def _cols(n, page, C):
    return 0 if n <= 0 else min(-(-int(n) // page), C)


def _give(ref, wants, put):
    """The lowest free page to each of `wants` in order; how many are missing."""
    short = 0
    for w in wants:
        free = np.flatnonzero(ref <= 0)
        if len(free):
            ref[free[0]] = 1
            put(w, int(free[0]))
        else:
            put(w, -1)
            short += 1
    return short


def reserve(tbl, ref, lens, page):
    tbl, ref = tbl.copy(), ref.copy()
    wants = [(b, c) for b in range(len(tbl)) for c in range(_cols(lens[b], page, tbl.shape[1]))
             if not 0 <= tbl[b, c] < len(ref)]
    return tbl, ref, _give(ref, wants, lambda w, i: tbl.__setitem__(w, i))


def free(tbl, ref, keep, page):
    tbl, ref = tbl.copy(), ref.copy()
    for b in range(len(tbl)):
        for c in range(_cols(keep[b], page, tbl.shape[1]), tbl.shape[1]):
            if 0 <= tbl[b, c] < len(ref):
                ref[tbl[b, c]] -= 1
            tbl[b, c] = -1
    return tbl, ref


def fork(tbl, ref, lens, parent, page):
    """(table, ref, lens, shortage, copies [(from, to)])."""
    B, C = tbl.shape
    P, old, ref = len(ref), tbl, ref.copy()
    new, n2, wants, kept = np.full_like(tbl, -1), np.zeros_like(lens), [], set()
    for b in range(B):
        p = int(parent[b])
        if not 0 <= p < B:
            continue
        n = min(max(int(lens[p]), 0), C * page)
        n2[b] = n
        for c in range(n // page):
            if 0 <= old[p, c] < P:
                new[b, c] = old[p, c]
        if n % page:
            c = n // page
            if 0 <= old[p, c] < P:
                if p in kept:
                    wants.append((b, c, int(old[p, c])))
                else:
                    new[b, c] = old[p, c]
            kept.add(p)
        else:
            kept.add(p)
    for x, by in ((old, -1), (new, 1)):
        for i in x[(x >= 0) & (x < P)]:
            ref[i] += by
    copies = []

    def put(w, i):
        new[w[0], w[1]] = i
        if i >= 0:
            copies.append((w[2], i))
    short = _give(ref, wants, put)
    return new, ref, n2, short, copies


def compact(tbl, ref):
    """(table, ref, map, moves [(from, to)])."""
    tbl, ref = tbl.copy(), ref.copy()
    used = np.flatnonzero(ref > 0)
    n = len(used)
    moves = list(zip(used[used >= n].tolist(), [i for i in range(n) if ref[i] <= 0]))
    to = np.arange(len(ref), dtype=np.int32)
    for a, b in moves:
        ref[b], ref[a], to[a] = ref[a], 0, b
    hit = (tbl >= 0) & (tbl < len(ref))
    tbl[hit] = to[tbl[hit]]
    return tbl, ref, to, moves
