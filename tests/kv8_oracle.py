"""The cache in 8 bits (include/tha_hybrid.h, tha_kv8_t) in float64 numpy, from its definition: codes, scales, kept rows, and the attention over them."""
import numpy as np

MOST = {"int8": 127.0, "e4m3": 448.0}


def levels(fmt):
    """The numbers that the codes 0, 1, .. stand for, in ascending order."""
    if fmt == "int8":
        return np.arange(128.0)
    return np.array([m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7) for e in range(16) for m in range(8)][:127])


def nearest(y, fmt):
    """The format's number nearest to y; of two the one with the even code."""
    v = levels(fmt)
    edge = (v[1:] + v[:-1]) / 2
    a = np.minimum(np.abs(y), v[-1])
    i = np.searchsorted(edge, a)                      # borders below a
    on = (i < len(edge)) & (edge[np.minimum(i, len(edge) - 1)] == a)
    return np.copysign(v[i + (on & (i % 2 == 1))], y)


def quantise(x, fmt):
    """x fp32 [position, channel] -> (numbers of the codes, scale)"""
    x = np.asarray(x, np.float32)
    fine = np.where(np.isfinite(x), np.abs(x), 0)
    top = float(fine.max(initial=0.0))
    s = np.float32(0) if top == 0 else max(np.float32(np.float64(top) / MOST[fmt]), np.float32(2.0 ** -126))
    if s == 0:
        q = np.zeros(x.shape)
    else:
        q = nearest(np.where(np.isfinite(x), x, 0).astype(np.float64) / np.float64(s), fmt)
    q = np.where(np.isnan(x), 0.0, q)
    return np.where(np.isinf(x), np.copysign(MOST[fmt] if s > 0 else 0.0, x), q) + 0.0, s


def numbers(codes, fmt):
    """uint8 codes -> the numbers they stand for (-0 as 0)"""
    codes = np.asarray(codes).view(np.uint8)
    if fmt == "int8":
        return codes.view(np.int8).astype(np.float64)
    v = np.append(levels("e4m3"), np.nan)
    return np.where(codes & 128, -1.0, 1.0) * v[codes & 127] + 0.0


def sees(a, t, p):
    """Whether a query at p sees key t; a: dict with window, keep_first, chunk."""
    ok = t <= p
    if a.get("chunk"):
        ok = ok & (t >= p // a["chunk"] * a["chunk"])
    if a.get("window"):
        ok = ok & ((p - t < a["window"]) | (t < a.get("keep_first", 0)))
    return ok


def attend(a, q, K, V, p0, absent=None):
    """q [n, heads, dim], K [T, kv heads, dim], V [T, kv heads, vdim] in float64, rows at p0 .. -> [n, heads, vdim].  absent [T]: keys of blocks that do not exist."""
    n, heads, _ = q.shape
    group = heads // K.shape[1]
    t, p = np.arange(K.shape[0])[None], np.arange(p0, p0 + n)[:, None]
    vis = sees(a, t, p)
    if absent is not None:
        vis = vis & ~absent[None]
    out = np.zeros((n, heads, V.shape[2]))
    for h in range(heads):
        s = q[:, h] @ K[:, h // group].T * a["scale"]
        if a.get("head_scale") is not None:
            s = s * a["head_scale"][h]
        if a.get("softcap"):
            s = a["softcap"] * np.tanh(s / a["softcap"])
        if a.get("rel") is not None:
            s = s + a["rel"][h][np.clip(p - t, 0, a["rel"].shape[1] - 1)]
        s = np.where(vis, s, -np.inf)
        sink = a["sink"][h] if a.get("sink") is not None else -np.inf
        m = np.maximum(s.max(1), sink)
        m = np.where(np.isfinite(m), m, 0.0)
        w = np.exp(s - m[:, None])
        total = w.sum(1) + np.exp(sink - m)
        out[:, h] = np.where(vis.any(1)[:, None], w @ V[:, h // group] / np.where(total > 0, total, 1)[:, None], 0.0)
        if a.get("gate") is not None:
            out[:, h] /= 1 + np.exp(-a["gate"][:, h])[:, None]
    return out
