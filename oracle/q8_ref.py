"""CPU restatements in 64 bits of the 8-bit KV cache and the logit rules — TEST INFRASTRUCTURE
ONLY. Plain numpy from the formulas in include/obn.h, one block, row or id at a time."""
from __future__ import annotations

import math

import numpy as np

BLOCK = 16
MIN_EXP = -126


def rope(x, pos, base):
    """x [heads, d] of one token at position pos, rotated pair by pair."""
    d = x.shape[-1]
    i = np.arange(d // 2, dtype=np.float64)
    ang = pos * np.power(np.float64(base), -2.0 * i / d)
    c, s = np.cos(ang), np.sin(ang)
    y = np.empty(x.shape, np.float64)
    x = x.astype(np.float64)
    y[..., 0::2] = x[..., 0::2] * c - x[..., 1::2] * s
    y[..., 1::2] = x[..., 0::2] * s + x[..., 1::2] * c
    return y


def need_scale(x):
    """The smallest power of two s >= 2^-126 with |x| <= 127 s; 0 for zeros, NaN for others."""
    if not np.all(np.isfinite(x)):
        return math.nan
    a = float(np.max(np.abs(x))) if x.size else 0.0
    if a == 0.0:
        return 0.0
    e = MIN_EXP
    while a > 127.0 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def append(codes, scales, rows, pos):
    """Appends rows [n, Hkv, d] (f64) at positions pos ... to one sequence's codes
    [S_max, Hkv, d] (int) and scales [blocks, Hkv], in place. Returns the unrounded codes of
    the stored rows [S_max, Hkv, d] (NaN elsewhere) for a test of borderline roundings."""
    S_max = codes.shape[0]
    raw = np.full(codes.shape, np.nan)
    n = rows.shape[0]
    lo, hi = max(pos, 0), min(pos + n, S_max)
    for blk in range(lo // BLOCK, -(-hi // BLOCK) if hi > lo else 0):
        a, b = max(lo, blk * BLOCK), min(hi, blk * BLOCK + BLOCK)
        for h in range(codes.shape[1]):
            new = rows[a - pos:b - pos, h]
            had = a > blk * BLOCK
            was = float(scales[blk, h]) if had else 0.0
            need = need_scale(new)
            now = math.nan if math.isnan(was) or math.isnan(need) else max(was, need)
            scales[blk, h] = now
            if not now > 0.0:
                codes[a:b, h] = 0
                continue
            old = codes[blk * BLOCK:a, h].astype(np.float64)
            codes[blk * BLOCK:a, h] = np.rint(old * (was / now))
            raw[a:b, h] = new / now
            codes[a:b, h] = np.rint(raw[a:b, h])
    return raw


def values(codes, scales):
    """codes [S, Hkv, d] with scales [blocks, Hkv] -> f64 values."""
    wide = np.repeat(scales.astype(np.float64), BLOCK, axis=0)[:codes.shape[0]]
    return codes.astype(np.float64) * wide[:, :, None]


def attention(q, k, v, L, scale):
    """q [n, H, d] of the n newest of L positions over values k, v [>= L, Hkv, d] -> (out
    [n, H, d], bound [n, H]): bound is how far an f32 evaluation may be off (see below).

    With u = 2^-24: a score is a sum of products q_i k_i whose magnitudes add up to A; in at
    most 24 accumulation steps of at most 2 u each, of q split to 2^-22, it is off by at most
    48 u A, so a weight is off by that share (and 4 u of the exponential), which moves the
    output by at most twice that times max |v|; sums over up to L keys in f32, a truncating
    step of 2 u per 16 keys and half, add L / 2 u max |v|."""
    n, H, d = q.shape
    G = H // k.shape[1]
    out = np.zeros((n, H, d))
    bound = np.zeros((n, H))
    lim = np.minimum(L, L - n + np.arange(n) + 1)
    rows = np.nonzero(lim > 0)[0]
    if not rows.size:
        return out, bound
    hidden = np.arange(L)[None] >= lim[rows][:, None]
    for h in range(H):
        K, V, Q = k[:L, h // G], v[:L, h // G], q[rows, h].astype(np.float64)
        s = np.where(hidden, -np.inf, Q @ K.T * scale)
        p = np.exp(s - s.max(1, keepdims=True))
        out[rows, h] = p @ V / p.sum(1, keepdims=True)
        A = np.where(hidden, 0.0, np.abs(Q) @ np.abs(K).T).max(1) * abs(scale)
        top = np.maximum.accumulate(np.abs(V).max(1))[lim[rows] - 1]
        bound[rows, h] = top * 2.0 ** -24 * (2 * 48 * A + 64 + lim[rows] / 2)
    return out, bound


def attention_by_products(q, k, v, v_scale, L, scale):
    """attention() with a bound on each output element [n, H, d] that goes by what adds up to it,
    for caches whose value scales [keys, Hkv] lie far apart (a bound by max |v| of all keys would
    hide what the small ones and the total lose).

    With u = 2^-24, p the normalised weights, S = sum p |v| (per element) and P = 127 max p s_v:
    scores are off by 48 u A as above, hence the weights by that share and 4 u, in the sum and
    in the total: 2 (48 A + 4) u S. A weight is held to 2^-27 of the largest product (fixed point
    of 31 bits whose reference is up to 32 times that product; f16 pairs: 2^-30), which is
    L / 8 u P over all keys, and to 2^-23 of itself, 2 u S. f32 sums, flushes and truncating steps
    stay below L / 2 + 32 roundings of S. f32 exponentials are zero below 2^-126 of their
    reference, which is up to 2^4 above the row's largest weight (or the largest total of a part,
    at least that weight): a key below 2^-120 of the largest weight may be missing, and its whole
    share is allowed. Last, results below 2^-126 are multiples of 2^-149."""
    n, H, d = q.shape
    G = H // k.shape[1]
    out = np.zeros((n, H, d))
    bound = np.full((n, H, d), 2.0 ** -148)
    lim = np.minimum(L, L - n + np.arange(n) + 1)
    for t in np.nonzero(lim > 0)[0]:
        for h in range(H):
            K, V, sv = (x[:lim[t], h // G] for x in (k, v, v_scale))
            x = q[t, h].astype(np.float64)
            s = K @ x * scale
            p = np.exp(s - s.max())
            far = np.where(p < 2.0 ** -120, p, 0.0) / p.sum()
            p /= p.sum()
            out[t, h] = p @ V
            bound[t, h] += far @ np.abs(V)
            A = (np.abs(K) @ np.abs(x)).max() * abs(scale)
            S, P = p @ np.abs(V), 127 * (p * sv).max()
            bound[t, h] += 2.0 ** -24 * (2 * 48 * A + 64 + lim[t] / 2) * (S + P)
    return out, bound


def attention_rms(q, k, v, L, scale):
    """attention() with, for each row [n, H], how large the error's root mean square over the row's
    d elements may be: near what f32 arithmetic leaves, so that a weight or query held in one
    f16, or one key too many or too few, shows (a key of average weight is 1 / sqrt(L) of the
    output's root mean square).

    u = 2^-24. A weight is off by ln 2 times the error of its score in base 2, s, whose roundings are
    2 u of the factor, u of the product, 2 u of q's halves, and at most 2 u of what is added up in
    each of 16 truncating tensor core steps: 37 u |s| ln 2 < 26 u |s| in all; and by 4 u of the
    exponential. Errors of keys are independent, as the values are, so their root mean square in
    the output is that of the weights' relative errors (weighted by p^2) times the output's.
    Sums of O are off by a bias of 2.5 u a unit for up to 3 units, by one rounding a flush, part
    or join, and the total by as much: 24 u. Twice that for the spread of a row's 128 elements."""
    n, H, d = q.shape
    G = H // k.shape[1]
    out, tol = np.zeros((n, H, d)), np.zeros((n, H))
    lim = np.minimum(L, L - n + np.arange(n) + 1)
    hidden = np.arange(L)[None] >= lim[:, None]
    for h in range(H):
        K, V, Q = k[:L, h // G], v[:L, h // G], q[:, h].astype(np.float64)
        s = np.where(hidden, -np.inf, Q @ K.T * scale)
        p = np.exp(s - s.max(1, keepdims=True))
        out[:, h] = p @ V / p.sum(1, keepdims=True)
        s = np.where(hidden, 0.0, s) / np.log(2.0)
        rms = np.sqrt((p * p * s * s).sum(1) / (p * p).sum(1))
        tol[:, h] = 2 * 2.0 ** -24 * (26 * rms + 4 + 24) * np.sqrt((out[:, h] ** 2).mean(-1))
    return out, tol


def logits(x, repetition=1.0, frequency=0.0, presence=0.0, history=(), bias=(), mask=None):
    """One row x [V]: history a list of ids, bias a list of (id, value), mask [V] bool."""
    y = x.astype(np.float64)
    V = y.size
    count = {}
    for i in history:
        if 0 <= i < V:
            count[i] = count.get(i, 0) + 1
    for i, c in count.items():
        f = float(repetition) ** c
        y[i] = y[i] / f if y[i] > 0 else y[i] * f
        y[i] -= c * float(frequency) + float(presence)
    for i, b in bias:
        if 0 <= i < V:
            y[i] += float(b)
    if mask is not None:
        y[~mask] = -np.inf
    return y
