"""The operators of a serving step over a paged FP8 cache in 64 bits, written from their definitions
(include/w4_abi.h), and what a kernel's output may be off by."""
import math

import numpy as np

FP8_MAX = 448.0


def e4m3_values():
    """What each of the 256 codes stands for."""
    v = np.empty(256)
    for b in range(256):
        e, m = (b >> 3) & 15, b & 7
        mag = math.nan if (b & 0x7F) == 0x7F else (8 + m) * 2.0 ** (e - 10) if e else m * 2.0 ** -9
        v[b] = -mag if b & 0x80 else mag
    return v


VALUES = e4m3_values()
_MAGS = VALUES[:0x7F]
_MIDS = (_MAGS[1:] + _MAGS[:-1]) / 2


def encode(x):
    """Nearest E4M3 code, ties to the even one; saturating, 0 for NaN; the sign of a zero is kept."""
    x = np.asarray(x, np.float64)
    a = np.minimum(np.abs(np.where(np.isnan(x), 0.0, x)), FP8_MAX)
    lo = np.searchsorted(_MIDS, a, side="left")   # codes whose lower border lies below a
    tie = (lo < len(_MIDS)) & (a == _MIDS[np.minimum(lo, len(_MIDS) - 1)])
    code = lo + (tie & (lo % 2 == 1))
    return (code | np.where(np.signbit(x) & ~np.isnan(x), 0x80, 0)).astype(np.uint8)


def scale_for(amax):
    """The smallest half that is at least amax / 448."""
    want = amax / FP8_MAX
    h = np.float16(want)
    return h if float(h) >= want else np.nextafter(h, np.float16(np.inf))


# ---- tables ----------------------------------------------------------------------------


def tables(bt, page, npages, tokens, cached, added, free_pages, free_range):
    """-> (bt, lens, cu, slots, positions, result) of w4_paged_tables."""
    bt = bt.copy()
    nseq, R = bt.shape
    lens, cu = np.zeros(nseq, np.int32), np.zeros(nseq + 1, np.int64)
    slots, positions = np.full(tokens, -1, np.int32), np.full(tokens, -1, np.int32)
    pre, taken, status = 0, 0, 0
    left = max(0, int(free_range[1]) - int(free_range[0]))
    for s in range(nseq):
        c, a = int(cached[s]), int(added[s])
        cu[s + 1] = cu[s] + max(a, 0)
        bad = c < 0 or a < 0 or c + a > min(R * page, 2 ** 31 - 1)
        over = a > 0 and cu[s + 1] > tokens
        need = 0 if bad or over else -(-(c + a) // page) - -(-c // page)
        lacks = need > 0 and pre + need > left
        status |= lacks | bad << 1 | over << 2
        lens[s] = max(c, 0) if lacks or bad or over else c + a
        if not (lacks or bad or over):
            for j in range(need):
                bt[s, -(-c // page) + j] = free_pages[free_range[0] + pre + j]
            if need:
                taken = pre + need
            for i in range(a):
                p = c + i
                positions[cu[s] + i] = p
                pg = int(bt[s, p // page])
                if 0 <= pg < npages:
                    slots[cu[s] + i] = pg * page + p % page
        pre += need
    return bt, lens, np.minimum(cu, 2 ** 31 - 1).astype(np.int32), slots, positions, np.array([taken, status], np.int32)


# ---- append ----------------------------------------------------------------------------


def append_side(codes, scales, x, slots):
    """codes [H][npages][page][D] uint8 and scales [H][npages] float16 with x [tokens][H][D] float16 in; also whether
    something was not finite."""
    codes, scales = codes.copy(), scales.copy()
    H, npages, page, D = codes.shape
    t, odd = 0, False
    while t < len(slots):
        slot = int(slots[t])
        if slot < 0 or slot >= npages * page:
            t += 1
            continue
        pg, r0 = divmod(slot, page)
        n = 1
        while t + n < len(slots) and r0 + n < page and slots[t + n] == slot + n:
            n += 1
        rows = x[t:t + n].astype(np.float64)
        for h in range(H):
            r = rows[:, h]
            fine = np.isfinite(r)
            odd |= not fine.all()
            want = scale_for(np.abs(r[fine]).max(initial=0.0))
            if r0 and scales[h, pg] > 0:
                s, k = float(scales[h, pg]), 0
                while s < float(want):
                    s, k = 2 * s, k + 1
                if k:
                    old = codes[h, pg, :r0]
                    again = encode(VALUES[old] * 2.0 ** -k)
                    codes[h, pg, :r0] = np.where(np.isnan(VALUES[old]), old, again)
            else:
                s = float(want)
            with np.errstate(invalid="ignore"):
                codes[h, pg, r0:r0 + n] = encode(r / s) if s else np.where(np.signbit(r) & fine, 0x80, 0)
            scales[h, pg] = np.float16(s)
        t += n
    return codes, scales, odd


# ---- attention --------------------------------------------------------------------------


def attention(q, bt, lens, cu, k, v, page, npages, group, causal, out):
    """q [tokens][Hq][D] float16; k, v: (codes, scales).  -> (out in 64 bits with rows that nothing wrote as they were,
    what a kernel may be off by).

    A kernel adds FP32 products of halves and codes, rounds a weight p sv to FP16 on the way and the result to FP16.
    With A = sum p |v| / sum p: the weights' rounding is 2^-11 A, or 2^-25 of the largest weight for those below
    FP16's normal range; the output's 2^-11 |o| (2^-25 below that range).  A score's FP32 sum of D products is off by
    (D + 4) 2^-24 sum |q k|, its exponent's argument (with x - M and the scales' products) by 2^-21 of its size, which
    moves a p by as much, and quotients by twice that; sums over T positions add T 2^-24."""
    out = out.astype(np.float64).copy()
    tol = np.zeros_like(out)
    T, Hq, D = q.shape
    c = 1.0 / math.sqrt(D)
    q = q.astype(np.float64)
    for s in range(len(lens)):
        q0, n = (int(cu[s]), int(cu[s + 1] - cu[s])) if cu is not None else (s, 1)
        L = max(0, int(lens[s]))
        pg = np.array([bt[s, t // page] if t // page < bt.shape[1] else -1 for t in range(L)], np.int64)
        there = (pg >= 0) & (pg < npages)
        rows = np.where(there, pg, 0) * page + np.arange(L) % page
        pgs = np.where(there, pg, 0)
        for h in range(Hq // group):
            kc, vc = (VALUES[x[0][h].reshape(-1, D)[rows]] for x in (k, v))
            sk, sv = (x[1][h, pgs].astype(np.float64) for x in (k, v))
            for i in range(min(n, T - q0)):
                see = there & ((np.arange(L) <= L - n + i) if causal else True)
                for j in range(group):
                    hq = h * group + j
                    if not see.any():
                        out[q0 + i, hq], tol[q0 + i, hq] = 0.0, 0.0
                        continue
                    kk, vv, a, b = kc[see], vc[see], sk[see], sv[see]
                    x = kk @ q[q0 + i, hq] * a * c
                    rough = np.abs(kk) @ np.abs(q[q0 + i, hq]) * a * c
                    p = np.exp(x - x.max())
                    p /= p.sum()
                    o = (p * b) @ vv
                    A = (p * b) @ np.abs(vv)
                    w = p * b
                    eps = (D + 4) * 2.0 ** -24 * rough.max() + 2.0 ** -21 * (np.abs(x).max() + 48) + len(x) * 2.0 ** -24
                    out[q0 + i, hq] = o
                    tol[q0 + i, hq] = (2.0 ** -11 * (A + np.abs(o)) + 2 * eps * A + 2.0 ** -25 * (1 + w.max() * np.abs(vv).sum(axis=0)))
    return out, tol
