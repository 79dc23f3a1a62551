"""Plain 64-bit implementations of the norm, routing and integer-product entry
points (numpy, from the formulas of include/apus_hip.h), and the device-buffer
plumbing of their tests."""
import numpy as np

I8_FLOOR = 2.0 ** -100


def bf16_bits(v):
    """fp32 values -> BF16 bits, ties to even (no NaN)."""
    u = np.ascontiguousarray(v, np.float32).view(np.uint32).astype(np.uint64)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def from_bf16(b):
    return (np.asarray(b, np.uint16).astype(np.uint32) << 16).view(np.float32)


def round_bf16(v):
    v = np.ascontiguousarray(v, np.float32)
    return np.where(np.isnan(v), v, from_bf16(bf16_bits(np.where(np.isnan(v), 0, v))))


def norm_truth(r, gamma, eps):
    """y in 64 bits of rows r [M, K] (already the stored sum)"""
    r = r.astype(np.float64)
    with np.errstate(invalid="ignore", divide="ignore"):
        v = 1.0 / np.sqrt((r * r).sum(1, keepdims=True) / r.shape[1] + np.float64(np.float32(eps)))
        return r * gamma.astype(np.float64) * v


def quant_i8(b):
    """(codes, scales) of BF16-valued rows b [M, K], finite"""
    a = np.maximum(np.abs(b).max(1).astype(np.float64), I8_FLOOR)
    inv = (127.0 / a).astype(np.float32)
    q = np.clip(np.rint(b.astype(np.float32) * inv[:, None]), -127, 127)
    return q.astype(np.int8), (a / 127.0).astype(np.float32)


def quant_e4m3(oracle, b):
    """(codes, scales) of BF16-valued rows by the oracle's act quant"""
    out = [oracle.act_quant_row(np.ascontiguousarray(row, np.float32)) for row in b]
    return np.stack([c for c, _ in out]), np.stack([s for _, s in out])


def product(a, sa, w, sw):
    """fp32 outputs with the documented roundings"""
    acc = a.astype(np.float64) @ w.astype(np.float64).T          # integers below 2^53: exact
    return (acc.astype(np.float32) * sa.astype(np.float32)[:, None]) * sw.astype(np.float32)[None, :]


def scores(kind, z):
    """p in 64 bits; masked logits (-inf, NaN) 0; +inf the largest fp32"""
    z = np.where(np.isnan(z), -np.inf, np.minimum(z, np.finfo(np.float32).max)).astype(np.float64)
    with np.errstate(over="ignore", invalid="ignore", divide="ignore"):
        if kind == "sigmoid":
            p = 1.0 / (1.0 + np.exp(-z))
        elif kind == "softmax":
            m = z.max(1, keepdims=True)
            e = np.where(np.isinf(m), 0.0, np.exp(z - np.where(np.isinf(m), 0.0, m)))
            t = e.sum(1, keepdims=True)
            p = np.where(t > 0, e / np.where(t > 0, t, 1.0), 0.0)
        else:
            p = np.sqrt(np.maximum(z, 0.0) + np.log1p(np.exp(-np.abs(z))))
    return np.where(np.isinf(z), 0.0, p), ~np.isinf(z)


def route(kind, z, bias, topk, groups, keep, top, renorm, scale):
    """(idx, wgt, p, gap): gap [s] = the smallest relative distance between different
    neighbours in the order that decides the row"""
    s, E = z.shape
    p, live = scores(kind, z)
    sel = p.copy()
    if bias is not None:
        live = live & ~(np.isnan(bias) | (bias == -np.inf))[None, :]
        with np.errstate(invalid="ignore"):
            sel = p + bias.astype(np.float64)[None, :]
    idx = np.empty((s, topk), np.int32)
    gap = np.full(s, np.inf)

    def order(v, ok, ids):
        return sorted(ids, key=lambda e: (0 if ok[e] else 1, -v[e] if ok[e] else 0, e))

    def near(v):
        v = np.asarray(v, np.float64)
        v = v[np.isfinite(v)]
        d, big = np.abs(np.diff(v)), np.maximum(np.abs(v[1:]), np.abs(v[:-1]))
        return (d[d > 0] / big[d > 0]).min() if (d > 0).any() else np.inf

    for t in range(s):
        ids = range(E)
        if groups > 1:
            per = E // groups
            best, any_ = np.full(groups, -np.inf), np.zeros(groups, bool)
            for g in range(groups):
                v = sorted((sel[t, e] for e in range(g * per, g * per + per) if live[t, e]), reverse=True)[:top]
                if v:
                    best[g], any_[g] = sum(v), True
            og = sorted(range(groups), key=lambda g: (0 if any_[g] else 1, -best[g] if any_[g] else 0, g))
            gap[t] = min(gap[t], near([best[g] for g in og[:keep + 1] if any_[g]]))
            ids = [e for g in og[:keep] for e in range(g * per, g * per + per)]
        o = order(sel[t], live[t], ids)
        idx[t] = o[:topk]
        gap[t] = min(gap[t], near([sel[t, e] for e in o[:topk + 1] if live[t, e]]))
    rows = np.arange(s)[:, None]
    w = np.where(live[rows, idx], p[rows, idx], 0.0)
    if renorm:
        t = w.sum(1, keepdims=True)
        w = np.where(t > 0, w / np.where(t > 0, t, 1.0), 0.0)
    return idx, w * np.float64(np.float32(scale)), p, gap
