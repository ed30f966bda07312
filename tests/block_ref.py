"""The routed-experts operators in 64 bits (numpy), with error bounds for their
kernels derived from the sums they take."""
import numpy as np

import mxfp4hip as M

BLOCK = 128
EPS = 2.0 ** -23
PER_448 = np.float32(1) / np.float32(448)
HALF_ULP = {M.DT_F32: 2.0 ** -24, M.DT_F16: 2.0 ** -11, M.DT_BF16: 2.0 ** -8}
TINY = {M.DT_F32: 1e-38, M.DT_F16: 2.0 ** -25, M.DT_BF16: 1e-38}


def bits_of(v, dtype):
    """f64 values as an array of a device type (bf16: its upper 16 bits, to nearest even)."""
    f = np.asarray(v, np.float32)
    if dtype == M.DT_F32:
        return f
    if dtype == M.DT_F16:
        return f.astype(np.float16)
    u = f.view(np.uint32)
    return ((u + 0x7fff + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def values_of(b, dtype):
    if dtype == M.DT_BF16:
        return (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return b.astype(np.float64)


def np_type(dtype):
    return {M.DT_F32: np.float32, M.DT_F16: np.float16, M.DT_BF16: np.uint16}[dtype]


def e4m3(v):
    """The nearest E4M3 value, ties to even, not past 448."""
    v = np.asarray(v, np.float64)
    exp = np.maximum(np.frexp(v)[1], -5) - 4
    return np.clip(np.ldexp(np.rint(np.ldexp(v, -exp)), exp), -448, 448)


def e4m3_values(codes):
    c = codes.astype(np.int64)
    e, m = (c >> 3) & 15, (c & 7).astype(np.float64)
    v = np.where(e > 0, np.ldexp(1 + m / 8, e - 7), np.ldexp(m / 8, -6))
    v = np.where(c & 127 == 127, np.nan, v)
    return np.where(c > 127, -v, v)


def blocks(n):
    return -(-n // BLOCK)


def act_scales(x):
    """f32 scales [blocks][rows]."""
    f = np.abs(np.asarray(x, np.float32))
    amax = np.stack([f[:, i:i + BLOCK].max(1) for i in range(0, f.shape[1], BLOCK)])
    s = np.maximum(amax * PER_448, np.float32(2.0 ** -126))
    return np.where(amax > 0, s, np.float32(1)).astype(np.float32)


def act_codes(x, s):
    """Code values: those of an f32 division."""
    x = np.asarray(x, np.float32)
    return e4m3((x / np.repeat(s.T, BLOCK, 1)[:, :x.shape[1]]).astype(np.float64))


def spread_w(s, n, k):
    return np.repeat(np.repeat(s, BLOCK, -2)[..., :n, :], BLOCK, -1)[..., :k].astype(np.float64)


def product(a, w, cores=False):
    """C of dequantized operands, and the bound of an f32 sum's error: each of a
    block's 128 products and of the blocks' sums may be rounded (or cut), and
    each block's sum is scaled by a rounded product of two scales.  The FP8 matrix
    cores (cores) align eight neighbouring products to the largest of them and
    cut what lies 2^-13 below its power of two before they add in f32: seven
    products may lose that much."""
    err = (BLOCK + blocks(a.shape[1]) + 4) * EPS * (np.abs(a) @ np.abs(w).T)
    if cores:
        aa, ww = np.abs(a), np.ascontiguousarray(np.abs(w).T)
        for k in range(0, a.shape[1], 8):
            top = aa[:, k, None] * ww[k]
            for j in range(k + 1, min(k + 8, a.shape[1])):
                np.maximum(top, aa[:, j, None] * ww[j], out=top)
            err += 7 * 2.0 ** -13 * top
    return a @ w.T, err


def rounded(c, err, dtype):
    """Bound after rounding to dtype."""
    return err + HALF_ULP[dtype] * (np.abs(c) + err) * 1.01 + TINY[dtype]


def quantized_mid(mid, err):
    """The middle's values as codes and scales, and how far a kernel's may be off
    whose middle is within err: its quotients may fall on the other side of a
    tie, and its scale moves with the largest value."""
    s = act_scales(mid).T.astype(np.float64)
    mx = np.repeat(s, BLOCK, 1)[:, :mid.shape[1]]
    ds = np.stack([err[:, i:i + BLOCK].max(1) for i in range(0, mid.shape[1], BLOCK)], 1)
    rel = np.repeat(ds / (s * 448.0), BLOCK, 1)[:, :mid.shape[1]] + 2 * EPS
    q = mid / mx
    d = err / mx + np.abs(q) * rel
    lo, hi, v = e4m3(q - d), e4m3(q + d), e4m3(q)
    return v * mx, np.maximum(hi - v, v - lo) * mx * (1 + rel) + np.abs(v) * mx * rel


def mlp(x, gate, up, down, cores=False):
    """(y, bound) of dequantized activations and weights."""
    g, eg = product(x, gate, cores)
    u, eu = product(x, up, cores)
    sig = 1 / (1 + np.exp(-g))
    mid = g * sig * u
    # |silu'| < 1.1; the quotient and the two products in f32, and the exponent's argument
    err = 1.1 * eg * np.abs(u) + np.abs(g * sig) * eu + eg * eu + (8 + np.abs(g)) * EPS * np.abs(mid) + 1e-30
    mq, em = quantized_mid(mid, err)
    y, ey = product(mq, down, cores)
    return y, ey * 1.2 + em @ np.abs(down).T


def route(logits, bias, topk, sigmoid, groups, topk_groups, group_top, renorm, scale):
    """(ids, weights, sure): rows are sure where no key or group score that
    decides is within 1e-5 of another unless they are equal."""
    t, e = logits.shape
    ids, weights, sure = np.full((t, topk), -1, np.int32), np.zeros((t, topk)), np.ones(t, bool)
    for r in range(t):
        v = np.minimum(logits[r].astype(np.float64), float(np.finfo(np.float32).max))
        here = v > -np.inf
        if not here.any():
            continue
        if sigmoid:
            p = np.where(here, 1 / (1 + np.exp(-np.where(here, np.maximum(v, -700), 0))), 0)
        else:
            x = np.where(here, np.exp(np.where(here, v, 0) - v[here].max()), 0)
            p = x / x.sum()
        p = np.where(p < 2.0 ** -150, 0, p)  # scores are f32: below its least value they are zero
        key = np.where(here, p + (0 if bias is None else bias.astype(np.float64)), -np.inf)
        key = np.where(np.isnan(key), -np.inf, key)
        def close(ranked):
            d = np.abs(np.diff(ranked[ranked > -np.inf]))
            return bool(((d > 0) & (d < 1e-5)).any())
        if groups > 1:
            size = e // groups
            best = -np.sort(-key.reshape(groups, size), 1)
            score = best[:, 0].copy()
            if group_top == 2 and size > 1:
                score = np.where(best[:, 1] > -np.inf, score + np.where(best[:, 1] > -np.inf, best[:, 1], 0), score)
            order = np.argsort(-score, kind="stable")
            sure[r] &= not close(score[order])
            for g in order[topk_groups:]:
                key[g * size:(g + 1) * size] = -np.inf
        order = np.argsort(-key, kind="stable")
        sure[r] &= not close(key[order][:topk + 1])
        order = [i for i in order[:topk] if key[i] > -np.inf]
        w = p[order]
        if renorm:
            w = w / w.sum() if w.sum() > 0 else 0 * w
        ids[r, :len(order)] = order
        weights[r, :len(order)] = w * scale
    return ids, weights, sure


def dispatch(ids, experts):
    """counts, rows, and the slots in expert order."""
    flat = ids.reshape(-1)
    slots = [i for e in range(experts) for i in np.nonzero(flat == e)[0]]
    rows = np.full(flat.size, -1, np.int32)
    rows[slots] = np.arange(len(slots))
    counts = np.array([(flat == e).sum() for e in range(experts)], np.int32)
    return counts, rows.reshape(ids.shape), np.array(slots, np.int64)
