"""A block of experts by its definition in 64 bits (numpy), and how far FP32 arithmetic rounded once may be from it.

u = 2^-24 is half a step of FP32, h = 2^-11 of FP16; 2^-25 is half a step of FP16's subnormals."""
import numpy as np

U, H, SUB = 2.0 ** -24, 2.0 ** -11, 2.0 ** -25

# ---- routing ---------------------------------------------------------------------------------


def route(logits, top_k, sigmoid=False, groups=1, top_groups=1, group_best=1, renorm=True, scale=1.0, bias=None, count=None):
    """logits [T][E] of FP16 or FP32 -> experts, weights, bound of the weights, order, offsets."""
    T, E = logits.shape
    most = float(np.finfo(logits.dtype).max)
    ids = np.full((T, top_k), -1, np.int32)
    w = np.zeros((T, top_k))
    bound = np.zeros((T, top_k))
    per = E // groups
    for t in range(T if count is None else max(0, min(T, count))):
        l = np.minimum(logits[t].astype(np.float64), most)
        there = l > -np.inf
        s = np.zeros(E)
        if there.any():
            if sigmoid:
                with np.errstate(over="ignore"):
                    s[there] = 1.0 / (1.0 + np.exp(-l[there]))
                # exp to a step (2 u), a sum and a quotient
                rel = np.full(E, 5 * U)
            else:
                top = l[there].max()
                x = np.exp(l[there] - top)
                s[there] = x / x.sum()
                # the difference is rounded (u of it, as much of the exponential), exp to a step; the sum of 1024 positive
                # terms, 16 in a lane and six steps across, and what the terms of it are off by
                far = np.minimum(top - np.where(there, l, top), 110.0)
                rel = (far + 3) * U + (far.max() + 3 + 24) * U + 2 * U
        c = l.copy()
        if bias is not None or groups > 1:
            c = s + (0.0 if bias is None else bias.astype(np.float64))
        c = np.where(there & (c > -np.inf), c, -np.inf)
        if groups > 1:
            value = np.full(groups, -np.inf)
            for g in range(groups):
                best = np.sort(c[g * per:(g + 1) * per])[::-1][:group_best]
                best = best[best > -np.inf]
                if len(best):
                    value[g] = best.sum()
            kept = [g for g in sorted(range(groups), key=lambda g: (-value[g], g))[:top_groups] if value[g] > -np.inf]
            c = np.where(np.isin(np.arange(E) // per, kept), c, -np.inf)
        best = [e for e in sorted(range(E), key=lambda e: (-c[e], e))[:top_k] if c[e] > -np.inf]
        ids[t, :len(best)] = best
        v, r = s[best], rel[best] if there.any() else np.zeros(0)
        if renorm and len(best):
            # ratios of scores, from their logarithms: none underflows
            logs = -np.logaddexp(0.0, -l[best]) if sigmoid else l[best]
            v = np.exp(logs - logs.max())
            v /= v.sum()
            # a sigmoid's ratio has a difference of logits in its exponential
            r = r + r.max() + (len(best) + 2 + 2 * np.minimum(logs.max() - logs, 110.0).max()) * U
        w[t, :len(best)] = v * scale
        bound[t, :len(best)] = np.abs(v * scale) * (r + 2 * U) + 2.0 ** -126  # (the smallest normal number may flush)
    flat = ids.reshape(-1)
    order = np.concatenate([np.flatnonzero(flat == e) for e in range(E)] + [np.full((flat < 0).sum(), -1)]).astype(np.int32)
    offsets = np.concatenate([[0], np.cumsum([(flat == e).sum() for e in range(E)])]).astype(np.int32)
    return ids, w, bound, order, offsets


# ---- experts' products -------------------------------------------------------------------------

E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6])


def pack(codes):
    """[rows][n] of 4-bit codes -> [rows][words] of uint32, low first; what stands behind a row's end is 0xF."""
    rows, n = codes.shape
    full = np.full((rows, -(-n // 8) * 8), 15, np.uint32)
    full[:, :n] = codes
    return (full.reshape(rows, -1, 8) << (4 * np.arange(8, dtype=np.uint32))).sum(axis=2, dtype=np.uint64).astype(np.uint32)


class Experts:
    """E matrices of R rows of K: fmt 0 W4 symmetric, 1 with zero-points, 2 MXFP4; `w`: the halves that they stand for."""

    def __init__(self, rng, E, R, K, fmt=0, gs=32):
        self.E, self.R, self.K, self.fmt, self.gs = E, R, K, fmt, 32 if fmt == 2 else gs
        N, G = E * R, -(-K // self.gs)
        self.G = G
        codes = rng.integers(0, 16, (N, K))
        self.q = pack(codes)
        group = np.arange(K) // self.gs
        self.zeros = None
        if fmt == 2:
            self.scales = rng.integers(119, 124, (N, G)).astype(np.uint8)
            value = E2M1[codes] * np.exp2(self.scales.astype(np.float64) - 127)[:, group]
        else:
            self.scales = (rng.uniform(0.5, 1.5, (N, G)) * 0.3 / np.sqrt(K)).astype(np.float16)
            z = np.full((N, G), 8)
            if fmt == 1:
                z = rng.integers(0, 16, (N, G))
                self.zeros = pack(z)
            value = (codes - z[:, group]) * self.scales.astype(np.float64)[:, group]
        self.w = value.astype(np.float16)


def act(kind, x):
    u = x if kind == 1 else 2.0 * np.sqrt(2.0 / np.pi) * (x + 0.044715 * x ** 3)
    with np.errstate(over="ignore"):
        return x / (1.0 + np.exp(-u))


def gemm_experts(m, x, order, offsets, top_k, kind, from_tokens, to_pairs, out):
    """Into a copy of `out` (FP64): the product, and how far FP16 results may be from it."""
    got, bound = out.astype(np.float64), np.zeros(out.shape)
    w = m.w.astype(np.float64).reshape(m.E, m.R, m.K)
    for e in range(m.E):
        for i in range(offsets[e], offsets[e + 1]):
            p = order[i]
            if p < 0 or p >= len(order):
                continue
            row = x[p // top_k if from_tokens else i].astype(np.float64)
            y = w[e] @ row
            off = (m.K + 8) * U * (np.abs(w[e]) @ np.abs(row))  # a sum of K terms in any order
            if kind:
                n = m.R // 2
                a = act(kind, y[:n])
                # the gates' slopes stay below 1.13; their own arithmetic: ten steps, and u of the exponent
                err = (1.13 * off[:n] + np.abs(a) * (12 + np.abs(y[:n])) * 2 * U) * (np.abs(y[n:]) + off[n:]) + np.abs(a) * off[n:]
                y, off = a * y[n:], err
            at = p if to_pairs else i
            got[at], bound[at] = y, off + np.abs(y) * H * (1 + 2 * H) + off * H + SUB
    return got, bound


# ---- norms and the residual stream ---------------------------------------------------------------


def _norm(x, off, weight, bias, centred, eps):
    """x / sqrt(mean x^2 + eps) and its error, from x and the error of x; sums of up to 32768 terms: 32 in a thread, six
    steps across a wave, 16 waves."""
    steps = 32 + 6 + 16 + 4
    if centred:
        mean = x.mean(axis=1, keepdims=True)
        off = off + off.mean(axis=1, keepdims=True) + steps * U * np.abs(x).mean(axis=1, keepdims=True) + U * np.abs(x)
        x = x - mean
        off = off + U * np.abs(x)
    ms = (x * x).mean(axis=1, keepdims=True) + eps
    f = 1.0 / np.sqrt(ms)
    # the mean square is off by steps u and by 2 rms(x) rms(off); half of that, and three roundings, in the factor
    rel = (steps / 2 + 6) * U + np.sqrt((off * off).mean(axis=1, keepdims=True)) * f
    y = x * f
    err = (off * f + np.abs(y) * (rel + U)) * np.abs(weight) + 2 * U * np.abs(y * weight)
    y = y * weight
    if bias is not None:
        y = y + bias
        err = err + U * np.abs(y)
    return y, err


def residual_norm(y, weights, shared, residual, post, post_bias, gate, pre, pre_bias, centred, eps, scale):
    """FP64 r and h and the errors of FP32 arithmetic before the last rounding."""
    T, k, D = y.shape
    b, off = np.zeros((T, D)), np.zeros((T, D))
    for j in range(k):
        w = np.ones(T) if weights is None else weights[:, j].astype(np.float64)
        term = np.where(w[:, None] == 0, 0.0, y[:, j].astype(np.float64)) * w[:, None]
        b += term
        off += (k + 3) * U * np.abs(term)
    if shared is not None:
        b += shared
        off += 2 * U * np.abs(shared.astype(np.float64))
    off += U * np.abs(b)
    if post is not None:
        b, off = _norm(b, off, post.astype(np.float64), None if post_bias is None else post_bias.astype(np.float64), centred, eps)
    if gate is not None:
        b, off = b * gate, off * np.abs(gate) + U * np.abs(b * gate)
    r = residual.astype(np.float64) + scale * b
    off = abs(scale) * (off + 2 * U * np.abs(b)) + U * np.abs(r)
    h = err = None
    if pre is not None:
        h, err = _norm(r, off, pre.astype(np.float64), None if pre_bias is None else pre_bias.astype(np.float64), centred, eps)
    return r, off, h, err


def rounded(value, err, f32=False):
    """The bound of a result that is rounded once."""
    return err + (U if f32 else H) * (np.abs(value) + err) + (2.0 ** -149 if f32 else SUB)
