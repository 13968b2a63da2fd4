"""Matrices in microscaled numbers in numpy and 64 bits, from their definition: what the kernels are held to."""
import numpy as np

BLOCK, TILE = 32, 128
MOST = {"e2m1": 6.0, "e4m3": 448.0}


def levels(fmt):
    """The format's numbers from 0 up, in the order of their codes."""
    if fmt == "e2m1":
        return np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
    return np.array([m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7) for e in range(16) for m in range(8)][:127])


def nearest(y, fmt):
    """The code (without its sign) nearest to |y|: at a border the even one."""
    v = levels(fmt)
    edge = (v[1:] + v[:-1]) / 2
    a = np.abs(y)
    i = np.searchsorted(edge, a)                          # borders below a
    at = np.minimum(i, len(edge) - 1)
    return i + ((i < len(edge)) & (edge[at] == a) & (i % 2 == 1))


def quantise(x, fmt):
    """x [rows, cols] in 64 bits -> (values [rows, cols], scale bytes [rows, blocks], codes [rows, cols])"""
    x = np.asarray(x, np.float64)
    rows, cols = x.shape
    y = np.pad(x, ((0, 0), (0, -cols % BLOCK))).reshape(rows, -1, BLOCK)
    bad = ~np.isfinite(y).all(-1)
    y = np.where(bad[..., None], 0.0, y)
    top = np.abs(y).max(-1)
    byte = np.zeros(top.shape, np.int64)
    for _ in range(255):                                  # the smallest power at which nothing exceeds the format's largest number
        byte += top > MOST[fmt] * np.exp2(byte - 127.0)
    scale = np.exp2(byte - 127.0)[..., None]
    code = nearest(y / scale, fmt)
    v = np.copysign(levels(fmt)[code], y) * scale
    v[bad] = np.nan
    byte[bad] = 255
    code = code | (np.signbit(y) << (3 if fmt == "e2m1" else 7))
    code[bad] = 0
    flat = lambda t: t.reshape(rows, -1)[:, :cols]  # noqa: E731
    return flat(v), byte, flat(code)


def scales_of(m):
    """Scale bytes [rows, blocks] of a matrix (an Mx), by the place that the layout gives each."""
    s = m.scales.cpu().numpy().reshape(-1)
    across = -(-m.cols // TILE)
    r, b = np.arange(m.rows)[:, None], np.arange(4 * across)[None]
    return s[((r // 128) * across + b // 4) * 512 + (r % 32) * 16 + (r // 32 % 4) * 4 + b % 4].astype(np.int64)


def codes_of(m):
    """Codes [rows, padded] of a matrix."""
    import torch
    c = m.codes.view(torch.uint8).cpu().numpy()
    return c.astype(np.int64) if m.format == "e4m3" else np.stack([c & 15, c >> 4], -1).reshape(m.rows, -1).astype(np.int64)


def values(m):
    """What a matrix stands for, in 64 bits."""
    c, s = codes_of(m), scales_of(m)
    sign = 8 if m.format == "e2m1" else 128
    v = np.append(levels(m.format), np.nan) if m.format == "e4m3" else levels(m.format)
    v = v[c % sign] * np.where(c >= sign, -1.0, 1.0)
    f = np.where(s == 255, np.nan, np.exp2(s - 127.0))
    return (v * np.repeat(f, BLOCK, 1))[:, :m.cols]


def half_step(y, fmt):
    """Half the distance of the format's numbers around |y| (y over its scale)."""
    e = np.floor(np.log2(np.maximum(np.abs(y), 1e-300)))
    return np.exp2(np.maximum(e, 0 if fmt == "e2m1" else -6) - (2 if fmt == "e2m1" else 4))


def act(name, g, u, limit, alpha):
    with np.errstate(over="ignore"):
        return _act(name, g, u, limit, alpha)


def _act(name, g, u, limit, alpha):
    if name == "relu2":
        return np.maximum(u, 0) ** 2
    if name == "xielu":
        p, q = np.log1p(np.exp(limit)), 0.5 + np.log1p(np.exp(alpha))
        return np.where(u > 0, p * u * u + 0.5 * u, q * (np.expm1(np.minimum(u, 0)) - u) + 0.5 * u)
    if name == "silu":
        return g / (1 + np.exp(-g)) * u
    if name == "gelu":
        return 0.5 * g * (1 + np.tanh(np.sqrt(2 / np.pi) * (g + 0.044715 * g ** 3))) * u
    g = np.minimum(g, limit)
    return g / (1 + np.exp(-alpha * g)) * (np.clip(u, -limit, limit) + 1)
