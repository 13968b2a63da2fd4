"""Matrices in microscaled numbers: quantising, reading back, the norm that ends in them, products and a feed-forward's input products, against 64 bits (mx_oracle.py)."""
import numpy as np
import pytest
import torch

import mx_oracle as O
from pkgload import load_pkg

M = load_pkg("mx")
pytestmark = pytest.mark.gpu
FORMATS = ["e2m1", "e4m3"]
DTYPES = [torch.float32, torch.bfloat16]


def numbers(rows, cols, seed, spread=3.0):
    """Values over several binades, with zeros, whole blocks of them, and values on the borders between codes"""
    g = np.random.default_rng(seed)
    x = g.standard_normal((rows, cols)) * np.exp2(g.uniform(-spread, spread, (rows, cols)))
    x[g.random((rows, cols)) < 0.05] = 0.0
    on_border = g.random((rows, cols)) < 0.2
    x[on_border] = (g.integers(-24, 25, (rows, cols)) / 4.0)[on_border]
    if cols >= 64:
        x[:, 32:64][g.random(rows) < 0.3] = 0.0
    return x


def upload(x, dtype=torch.float32, wide=0, offset=0):
    """x on the device, as columns of a wider array"""
    t = torch.from_numpy(np.ascontiguousarray(x, np.float32)).cuda().to(dtype)
    if not wide and not offset:
        return t
    room = torch.full((x.shape[0], x.shape[1] + wide + offset), 7.0, dtype=dtype, device="cuda")
    room[:, offset:offset + x.shape[1]] = t
    return room[:, offset:offset + x.shape[1]]


def same_matrix(m, x):
    """Codes and scales of m are those of x in 64 bits; padding holds codes of 0 and scales that are numbers."""
    v, byte, code = O.quantise(x, m.format)
    got, s = O.codes_of(m), O.scales_of(m)
    assert np.array_equal(s[:, :byte.shape[1]], byte)
    assert np.array_equal(got[:, :m.cols], code)
    assert not got[:, m.cols:].any() and (s[:, byte.shape[1]:] == 0).all()
    return v


# ---- quantising and reading back --------------------------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols,wide,offset", [(1, 1, 0, 0), (1, 768, 0, 0), (3, 31, 1, 0), (5, 33, 0, 3), (130, 256, 8, 0), (37, 257, 7, 1), (200, 1000, 0, 0), (129, 383, 1, 0),
                                                   (2, 5000, 24, 8)])
def test_quantise(fmt, dtype, rows, cols, wide, offset):
    x = upload(numbers(rows, cols, rows + cols), dtype, wide, offset)
    m = M.quantise(x, fmt)
    v = same_matrix(m, x.double().cpu().numpy())
    for out in DTYPES:
        assert torch.equal(m.read(out).double().cpu(), torch.from_numpy(v))      # few bits under a power of two: exact in either
    room = torch.full((rows, cols + 5), 9.0, device="cuda")
    m.read(out=room[:, 2:2 + cols])
    assert torch.equal(room[:, 2:2 + cols].double().cpu(), torch.from_numpy(v)) and (room[:, :2] == 9).all() and (room[:, 2 + cols:] == 9).all()


@pytest.mark.parametrize("fmt", FORMATS)
def test_every_binade_and_border(fmt):
    """Scales from the smallest power to the largest numbers of fp32; values just at, below and above the border of a scale and of codes"""
    most = O.MOST[fmt]
    rows = []
    for e in list(range(-149, 128, 3)) + [-127, -126, -125, 126, 127]:
        top = np.float32(np.ldexp(1.0, e))
        rows.append(np.float32(np.linspace(-1, 1, 32)) * top)
    edge = (O.levels(fmt)[1:] + O.levels(fmt)[:-1]) / 2
    for e in (-100, 0, 60):
        for s in (np.nextafter(np.float32(most), np.float32(0)), np.float32(most), np.nextafter(np.float32(most), np.float32(1e9))):
            r = np.zeros(32, np.float32)
            r[0] = s
            near = np.float32(np.random.default_rng(e + 200).choice(edge, 10))
            r[1:11], r[11:21], r[21:31] = near, np.nextafter(near, np.float32(0)), -np.nextafter(near, np.float32(1e9))
            rows.append(np.ldexp(r, e).astype(np.float32))
    x = np.stack(rows)
    for dtype in DTYPES:                                     # one block a row, and all in a row
        for t in (torch.from_numpy(x).cuda().to(dtype), torch.from_numpy(x).cuda().to(dtype).view(1, -1)):
            m = M.quantise(t, fmt)
            v = torch.from_numpy(same_matrix(m, t.double().cpu().numpy()))
            assert torch.equal(m.read().double().cpu(), v.float().double())
            assert torch.equal(m.read(torch.bfloat16).double().cpu(), v.float().bfloat16().double())


@pytest.mark.parametrize("fmt", FORMATS)
def test_blocks_that_hold_no_number(fmt):
    """A NaN or an infinity makes its block NaN and no other"""
    x = numbers(5, 160, 3)
    x[0, 5], x[1, 40], x[2, 159], x[3, 96] = np.nan, np.inf, -np.inf, np.nan
    m = M.quantise(upload(x), fmt)
    v = same_matrix(m, x)
    got = m.read().double().cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(v)) and np.isnan(got).sum() == 4 * 32
    assert np.array_equal(got[~np.isnan(got)], v[~np.isnan(v)])


@pytest.mark.parametrize("fmt", FORMATS)
def test_rows_of_a_checkpoint(fmt):
    """Row-major codes and scales, as files have them"""
    x = numbers(70, 161, 8)
    _, byte, code = O.quantise(x, fmt)
    if fmt == "e2m1":
        c = np.pad(code, ((0, 0), (0, 1)), constant_values=9).astype(np.uint8)     # the last half byte is nobody's
        codes = torch.from_numpy(c[:, 0::2] | (c[:, 1::2] << 4)).cuda()
    else:
        codes = torch.from_numpy(code.astype(np.uint8)).cuda().view(torch.float8_e4m3fn)
    m = M.Mx.of_rows(codes, torch.from_numpy(byte.astype(np.uint8)).cuda(), 161)
    same_matrix(m, x)


# ---- the norm ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols,wide,offset", [(1, 4096, 0, 0), (3, 1, 0, 0), (7, 33, 1, 1), (130, 288, 8, 0), (5, 1001, 0, 0), (2, 2049, 3, 2), (3, 14336, 0, 0), (2, 20001, 0, 0), (2, 32768, 0, 0), (3, 40001, 2, 0),
                                                   (400, 300, 0, 0), (400, 4104, 1, 0), (700, 8192, 8, 0), (600, 4096, 0, 0), (1300, 1000, 16, 8), (650, 11008, 0, 0),
                                                   (601, 40, 0, 0), (900, 12, 4, 0)])
def test_add_norm(fmt, dtype, rows, cols, wide, offset):
    x, left, w = numbers(rows, cols, 1), numbers(rows, cols, 2), numbers(1, cols, 3)[0]
    x, w = (torch.from_numpy(t.astype(np.float32)).cuda() for t in (x, w))
    l = upload(left, dtype, wide, offset)
    s = (x + l.float()).double().cpu().numpy()                                       # the sum as stored
    y = s / np.sqrt((s * s).mean(-1, keepdims=True) + 1e-5) * (0.25 + w.double().cpu().numpy())
    to = torch.empty_like(x)
    kept = x.clone()
    m = M.add_norm(x, l, w, eps=1e-5, w_offset=0.25, format=fmt, x_out=to)
    assert torch.equal(to.double().cpu(), torch.from_numpy(s)) and torch.equal(x, kept)
    same_matrix(m, y)
    m = M.add_norm(x, l, w, eps=1e-5, w_offset=0.25, format=fmt)                     # in place
    assert torch.equal(x, to)
    same_matrix(m, y)
    m = M.add_norm(x, None, w, eps=1e-5, w_offset=0.25, format=fmt)                  # nothing joins
    assert torch.equal(x, to)
    same_matrix(m, y)


@pytest.mark.parametrize("rows", [3, 700])
@pytest.mark.parametrize("power", [-90, -60, -20, 40, 70, 100])
def test_add_norm_at_the_ends_of_fp32(power, rows):
    """Rows whose squares are no numbers of fp32, some of them between others"""
    x = numbers(rows, 1000, 5)
    x[::2] = np.ldexp(x[::2], power)
    x = x.astype(np.float32)
    w = numbers(1, 1000, 6)[0].astype(np.float32)
    s = x.astype(np.float64)
    y = s / np.sqrt((s * s).mean(-1, keepdims=True) + float(np.float32(1e-30))) * w.astype(np.float64)
    same_matrix(M.add_norm(torch.from_numpy(x).cuda(), None, torch.from_numpy(w).cuda(), eps=1e-30), y)


@pytest.mark.parametrize("rows", [3, 900])
def test_add_norm_of_zeros_and_of_no_numbers(rows):
    x = torch.zeros(rows, 100, device="cuda")
    x[1::3, 7], x[2::3, 9] = float("nan"), float("inf")
    w = torch.ones(100, device="cuda")
    got = M.add_norm(x, None, w, eps=1e-5).read().cpu()
    assert (got[0::3] == 0).all() and got[1::3].isnan().all()
    assert got[2::3, :32].isnan().all() and (got[2::3, 32:] == 0).all()              # inf * 0 in its block, 0 / inf in the others


# ---- products ---------------------------------------------------------------------------------------------------------------
def matrices(rows, n, k, fmt, seed, count=1):
    """Rows in `fmt` and matrices in 4 bits, made on the host, so that a product is tested by itself; scale bytes of rows that are not there are 255"""
    g = np.random.default_rng(seed)
    made = []
    for r, f in [(rows, fmt)] + [(n, "e2m1")] * count:
        x = g.standard_normal((r, k)) * np.exp2(g.integers(-3, 4, (r, 1)))
        _, byte, code = O.quantise(x, f)
        c = torch.from_numpy(np.pad(code, ((0, 0), (0, k % 2 if f == "e2m1" else 0))).astype(np.uint8))
        codes = c[:, 0::2] | (c[:, 1::2] << 4) if f == "e2m1" else c.view(torch.float8_e4m3fn)
        m = M.Mx.of_rows(codes.cuda(), torch.from_numpy(byte.astype(np.uint8)).cuda(), k)
        tiles = m.scales.view(-1, m.scales.numel() // 512 // -(-r // 128), 32, 4, 4)
        for lane in range(128):
            if (r - 1) // 128 * 128 + lane >= r:
                tiles[-1, :, lane % 32, lane // 32] = 255
        made.append(m)
    return made


def sum_bound(a, w):
    """How far fp32 sums of exact products may be off: an instruction adds 32 values or more at a time to the sum, each addition (and each value's alignment) off by less than a unit of the
    24th bit of what is added up so far, at most sum |a| |w|."""
    total = np.abs(a) @ np.abs(w).T
    return (a.shape[1] / 32 + 33) * 2.0 ** -23 * total


SIZES = [(1, 1, 1), (1, 128, 128), (2, 33, 32), (3, 127, 31), (15, 129, 33), (16, 256, 256), (17, 300, 129), (33, 64, 384), (64, 260, 500), (65, 128, 640), (128, 129, 1000), (129, 31, 257),
         (200, 200, 1152), (300, 513, 96), (7, 1000, 4100), (513, 640, 2048), (1000, 777, 300),
         # pairs: fewer items than pairs; the last round whole, in quarters, in halves; activation rows behind whole tiles of every width
         (1100, 2600, 160), (1030, 5000, 96), (1024, 6400, 130), (2100, 4900, 64), (900, 3900, 288), (256, 20000, 33)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows,n,k", SIZES)
def test_linear(fmt, rows, n, k):
    a, w = matrices(rows, n, k, fmt, rows + n + k)
    va, vw = O.values(a), O.values(w)
    want, tol = va @ vw.T, sum_bound(va, vw)
    got = M.linear(a, w).double().cpu().numpy()
    assert (np.abs(got - want) <= tol).all(), np.abs(got - want).max()
    room = torch.full((rows, n + 9), 5.0, dtype=torch.bfloat16, device="cuda")
    M.linear(a, w, out=room[:, 4:4 + n])
    got = room[:, 4:4 + n].double().cpu().numpy()
    assert (np.abs(got - want) <= tol + (np.abs(want) + tol) * 2.0 ** -8).all()      # and one rounding to bf16
    assert (room[:, :4] == 5).all() and (room[:, 4 + n:] == 5).all()
    M.check_error()


ACTS = [("silu", 0.0, 0.0), ("gelu", 0.0, 0.0), ("clamped", 3.0, 1.702), ("relu2", 0.0, 0.0), ("xielu", 0.3, -0.2)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("out_fmt", FORMATS)
@pytest.mark.parametrize("act,limit,alpha", ACTS)
@pytest.mark.parametrize("rows,n,k", [(1, 1, 1), (2, 33, 100), (16, 128, 256), (40, 300, 384), (100, 257, 1000), (129, 513, 640), (300, 1000, 513),
                                      (700, 2100, 160), (513, 4900, 96), (300, 9300, 130), (128, 19000, 64)])
def test_linear_act(fmt, out_fmt, act, limit, alpha, rows, n, k):
    gated = act not in M.UNGATED
    a, *ws = matrices(rows, n, k, fmt, rows + n + k, 2 if gated else 1)
    va = O.values(a)
    p = [va @ O.values(w).T for w in ws]
    y = O.act(act, p[0], p[-1], limit, alpha)
    m = M.linear_act(a, ws[0] if gated else None, ws[-1], act=act, format=out_fmt, limit=limit, alpha=alpha)
    M.check_error()
    cancels = 2.0 ** -23 * np.abs(p[0] * p[-1]) if act == "gelu" else 2.0 ** -21 * np.abs(p[-1]) if act == "xielu" else 2.0 ** -126 * np.abs(p[0]) * (1 + np.abs(p[-1]))
    near(m, y, cancels, [O.act(act, p[0] + s * sum_bound(va, O.values(ws[0])), p[-1] + t * sum_bound(va, O.values(ws[-1])), limit, alpha) for s in (-1, 1) for t in (-1, 1)])


@pytest.mark.parametrize("act", ["silu", "gelu", "clamped"])
@pytest.mark.parametrize("power", [20, 45, 55])
@pytest.mark.parametrize("rows,n", [(3, 300), (600, 9300)])
def test_large_gates(act, power, rows, n):
    """Gates whose cube, in gelu, is no number of fp32, and whose sigmoid is 1 or 0"""
    a, gate, up = matrices(rows, n, 64, "e4m3", power, 2)
    gate.scales.add_(torch.where(gate.scales < 255, torch.tensor(power, dtype=torch.uint8, device="cuda"), torch.tensor(0, dtype=torch.uint8, device="cuda")))
    va, vg, vu = O.values(a), O.values(gate), O.values(up)
    g, u = va @ vg.T, va @ vu.T
    m = M.linear_act(a, gate, up, act=act, limit=5.0, alpha=1.5)
    M.check_error()
    y = O.act(act, g, u, 5.0, 1.5)
    assert np.isfinite(y).all() and np.isfinite(O.values(m)).all()
    cancels = 2.0 ** -23 * np.abs(g * u) if act == "gelu" else 2.0 ** -126 * np.abs(g) * (1 + np.abs(u))
    near(m, y, cancels, [O.act(act, g + s * sum_bound(va, vg), u + t * sum_bound(va, vu), 5.0, 1.5) for s in (-1, 1) for t in (-1, 1)])


def near(m, y, cancels, around):
    """m's values are within half a step of y, as far as y itself is known: `around` holds it at the ends of its products' bounds; the activation in fp32 is good to 2^-20 of it, and to
    `cancels` where it is a difference: gelu's 1 + tanh is off by a unit of tanh near 1 and a rounding, 2^-23 + 2^-24 in all and 0.5 g u times that; xielu's e^u - 1 - u by a unit of e^u - 1 and a
    rounding, 2^-23 + 2^-24 of |u| at most, times a factor below 2, and so much again for 0.5 u and the sum;
    a sigmoid below 2^-128, whose e^-g is no number of fp32, is 0, and one below 2^-126 keeps fewer bits: off by 2^-126 of g (1 + u) at most."""
    off = np.max([np.abs(t - y) for t in around], 0) + np.abs(y) * 2.0 ** -20 + cancels
    s, rows, cols = O.scales_of(m), m.rows, m.cols
    blocks = lambda t: np.pad(t, ((0, 0), (0, -cols % 32))).reshape(rows, -1, 32).max(-1)  # noqa: E731
    lo, hi = blocks(np.abs(y) - off).clip(0), blocks(np.abs(y) + off)
    most = O.MOST[m.format] * np.exp2(s[:, :lo.shape[1]] - 127.0)
    assert (lo <= most).all() and ((hi > most / 2) | (s[:, :lo.shape[1]] == 0)).all()      # the smallest power that holds the block
    assert (s[:, lo.shape[1]:] == 0).all() and not O.codes_of(m)[:, cols:].any()
    f = np.repeat(np.exp2(s - 127.0), 32, 1)[:, :cols]
    worst = np.abs(O.values(m) - y) - off - f * O.half_step((np.abs(y) + off) / f, m.format)
    assert (worst <= 1e-12 * np.abs(y)).all(), worst.max()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows,n", [(20, 200), (100, 200), (1100, 2600)])
def test_nan_rows_stay_in_their_rows(fmt, rows, n):
    a, w = matrices(rows, n, 300, fmt, 4)
    a.scales.view(-1)[(0 * 32 + 3) * 16 + 0] = 255           # row 3, block 0
    w.scales.view(-1)[(1 * 3 + 2) * 512 + (5 % 32) * 16 + 1] = 255    # row 133, block 9
    got = M.linear(a, w).cpu()
    bad = torch.zeros(rows, n, dtype=torch.bool)
    bad[3], bad[:, 133] = True, True
    assert torch.equal(got.isnan(), bad)
    got = M.linear_act(a, w, w).read().cpu()                 # a block of the result is NaN as a whole
    bad[:, 128:160] = True
    assert torch.equal(got.isnan(), bad)


def test_no_rows():
    w = M.quantise(torch.randn(64, 96, device="cuda"))
    a = M.quantise(torch.randn(0, 96, device="cuda"), "e4m3")
    assert a.read().shape == (0, 96) and M.linear(a, w).shape == (0, 64) and M.linear_act(a, w, w).rows == 0
    assert M.add_norm(torch.randn(0, 96, device="cuda"), None, torch.ones(96, device="cuda"), eps=1e-5).rows == 0


# ---- as a layer uses them -----------------------------------------------------------------------------------------------------
def layer(rows, width, ff, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    return {"x": rand(rows, width), "att": rand(rows, width).bfloat16(), "norm": 1 + 0.1 * rand(width), "wo": M.quantise(rand(width, width) / width ** 0.5),
            "gate": M.quantise(rand(ff, width) / width ** 0.5), "up": M.quantise(rand(ff, width) / width ** 0.5), "down": M.quantise(rand(width, ff) / ff ** 0.5)}


def run_layer(s, fmt="e4m3"):
    """attention's result -> output product -> residual and norm -> feed-forward -> residual"""
    x = s["x"].clone()
    y = M.linear(M.quantise(s["att"], fmt), s["wo"], dtype=torch.bfloat16)
    a = M.add_norm(x, y, s["norm"], eps=1e-5, format=fmt)
    h = M.linear_act(a, s["gate"], s["up"], format=fmt)
    z = M.linear(h, s["down"])
    last = M.add_norm(x, z, s["norm"], eps=1e-5, format=fmt)
    return y, a.read(), h.read(), z, x, last.read()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows,width,ff", [(1, 288, 768), (17, 512, 1100), (260, 768, 2048), (1100, 512, 2600)])
def test_a_layer(fmt, rows, width, ff):
    """Every call's result against 64 bits on what the call ahead of it left"""
    s = layer(rows, width, ff, rows)
    y, a, h, z, x, last = (t.double().cpu().numpy() for t in run_layer(s, fmt))
    att, _, _ = O.quantise(s["att"].double().cpu().numpy(), fmt)
    wo, gate, up, down = (O.values(s[k]) for k in ("wo", "gate", "up", "down"))
    assert (np.abs(y - att @ wo.T) <= sum_bound(att, wo) + (np.abs(att @ wo.T) + sum_bound(att, wo)) * 2.0 ** -8).all()
    first = (s["x"].double().cpu().numpy() + y).astype(np.float32).astype(np.float64)
    norm = lambda t: t / np.sqrt((t * t).mean(-1, keepdims=True) + 1e-5) * s["norm"].double().cpu().numpy()  # noqa: E731
    assert np.array_equal(a, O.quantise(norm(first), fmt)[0])
    assert (np.abs(z - h @ down.T) <= sum_bound(h, down)).all()
    assert np.array_equal(x, (first + z).astype(np.float32).astype(np.float64)) and np.array_equal(last, O.quantise(norm(x), fmt)[0])
    g, u = a @ gate.T, a @ up.T
    want = O.act("silu", g, u, 0, 0)
    # a value is off by half a step at most, 2^-4 (8 bits) or 1/4 (4 bits) of it or as much of the smallest normal number under its block's scale, which is below 2 / M of the block's largest
    top = np.repeat(np.pad(np.abs(want), ((0, 0), (0, -ff % 32))).reshape(rows, -1, 32).max(-1), 32, 1)[:, :ff]
    half, least = (2.0 ** -4, 2.0 ** -6 / 448) if fmt == "e4m3" else (0.25, 1 / 6)
    assert (np.abs(h - want) <= 1.01 * half * np.maximum(np.abs(want), 2 * least * top) + 1e-5 * top).all()


def test_captured_layers_share_nothing():
    """Two captured layers on streams of their own, replayed at once and again with other inputs, as the same calls one by one"""
    cases = [layer(5, 512, 1100, 1), layer(700, 512, 2600, 2)]
    graphs, outs = [], []
    for s in cases:
        run_layer(s)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run_layer(s))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for turn in range(3):
        for s in cases:
            s["att"].copy_(torch.randn_like(s["att"], dtype=torch.float32))
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for s, o in zip(cases, outs):
            for got, want in zip(o, run_layer(s)):
                assert torch.equal(got, want)
    M.check_error()


def test_first_calls_of_a_process_captured():
    """What the library keeps for a device is made inside the capture"""
    import subprocess
    import sys
    code = ("import sys; sys.path.insert(0, 'tests')\nimport torch\nfrom pkgload import load_pkg\nM = load_pkg('mx')\n"
            "x = torch.randn(700, 4096, device='cuda'); w = torch.ones(4096, device='cuda'); k = torch.randn(2600, 4096, device='cuda')\ntorch.cuda.synchronize()\n"
            "g = torch.cuda.CUDAGraph()\nwith torch.cuda.graph(g):\n    q = M.quantise(k); a = M.add_norm(x, None, w, eps=1e-5); y = M.linear(a, q); h = M.linear_act(a, q, q)\n"
            "g.replay(); torch.cuda.synchronize()\nassert torch.equal(y, M.linear(M.add_norm(x, None, w, eps=1e-5), M.quantise(k)))\n"
            "assert torch.equal(h.read(), M.linear_act(a, q, q).read())\nM.check_error(); print('fine')\n")
    import os
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "fine" in r.stdout, r.stderr[-2000:]


def test_threads_and_streams():
    """Four threads on streams of their own make calls of different forms at once"""
    import threading
    cases = [layer(*c) for c in ((1, 512, 1100, 1), (33, 512, 1100, 2), (300, 768, 2048, 3), (900, 512, 2600, 4))]
    want = [run_layer(s) for s in cases]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(5):
                got = run_layer(cases[i])
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                    bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(cases))]
    for t in threads:
        t.start()
    for t in threads:
        t.join(120)
    assert not bad and not any(t.is_alive() for t in threads)
    M.check_error()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows,cols", [(1, 1), (33, 130), (129, 513), (700, 4096)])
def test_nothing_else_is_written(fmt, rows, cols):
    """Memory around a matrix, and the scale bytes of rows behind its last one, stay as they were"""
    size = M.Mx.empty(rows, cols, fmt)
    nc, ns = size.codes.numel(), size.scales.numel()
    room = torch.full((512 + nc + 1024 + ns + 512,), 0xA5, dtype=torch.uint8, device="cuda")
    a, b = 512, (512 + nc + 1023) // 512 * 512
    codes = room[a:a + nc].view(rows, -1)
    m = M.Mx(codes if fmt == "e2m1" else codes.view(torch.float8_e4m3fn), room[b:b + ns], rows, cols)
    x = torch.randn(rows, cols, device="cuda")
    one, up = M.quantise(torch.randn(rows, 64, device="cuda"), "e4m3"), M.quantise(torch.randn(cols, 64, device="cuda"))

    def around():
        t = room.clone()
        t[a:a + nc] = 0xA5
        s = t[b:b + ns].view(-1, ns // 512 // -(-rows // 128), 32, 4, 4)
        for r in range(rows - (rows - 1) // 128 * 128):
            s[-1, :, r % 32, r // 32] = 0xA5
        s[:-1] = 0xA5
        return bool((t == 0xA5).all())

    for call in (lambda: M.quantise(x, out=m), lambda: M.add_norm(x, None, torch.ones(cols, device="cuda"), eps=1e-5, out=m), lambda: M.linear_act(one, None, up, act="relu2", out=m),
                 lambda: M.linear_act(one, up, up, out=m)):
        room.fill_(0xA5)
        call()
        assert around()
        assert not O.codes_of(m)[:, cols:].any() and (O.scales_of(m)[:, -(-cols // 32):] == 0).all()


def test_long_rows():
    """Offsets beyond 32 bits: a matrix of more than 2^31 codes, and results of more than 2^31 elements"""
    rows, cols = 70000, 33000
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    x[-1], x[0, :5], x[35000, 7] = torch.randn(cols, device="cuda").bfloat16(), 2.0, -3.0
    for fmt in FORMATS:
        m = M.quantise(x, fmt)
        back = m.read(torch.bfloat16)
        want = O.quantise(x[[0, 35000, rows - 1]].double().cpu().numpy(), fmt)[0]
        assert np.array_equal(back[[0, 35000, rows - 1]].double().cpu().numpy(), want)
        assert int((back != 0).sum()) == int((torch.from_numpy(want) != 0).sum())
        del m, back
    del x
    a, w = matrices(70000, 31000, 32, "e4m3", 1)
    got = M.linear(a, w, dtype=torch.bfloat16)
    pick = [0, 1, 34999, 69998, 69999]
    va, vw = O.values(a)[pick], O.values(w)
    want = va @ vw.T
    assert (np.abs(got[pick].double().cpu().numpy() - want) <= sum_bound(va, vw) + (np.abs(want) + sum_bound(va, vw)) * 2.0 ** -8).all()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("act,limit,alpha", ACTS)
@pytest.mark.parametrize("where", ["rows", "gate", "up"])
@pytest.mark.parametrize("rows,n,k", [(20, 200, 300), (20, 200, 4100), (1100, 2600, 300)])
def test_nan_passes_every_activation(fmt, act, limit, alpha, where, rows, n, k):
    """One block, clusters, pairs: what is no number in the rows or in a matrix is none in the result, and changes nothing else"""
    gated = act not in M.UNGATED
    if where == "gate" and not gated:
        where = "up"
    a, *ws = matrices(rows, n, k, fmt, 4, 2 if gated else 1)
    call = lambda: M.linear_act(a, ws[0] if gated else None, ws[-1], act=act, limit=limit, alpha=alpha).read().cpu()  # noqa: E731
    clean = call()
    bad = torch.zeros(rows, n, dtype=torch.bool)
    if where == "rows":
        a.scales.view(-1)[(0 * 32 + 3) * 16 + 0] = 255       # row 3, block 0
        bad[3] = True
    else:
        w, across = ws[0 if where == "gate" else -1], -(-k // 128)
        w.scales.view(-1)[(1 * across + 2) * 512 + (5 % 32) * 16 + 1] = 255    # row 133, block 9
        bad[:, 128:160] = True                               # a block of the result is NaN as a whole
    got = call()
    assert not clean.isnan().any() and torch.equal(got.isnan(), bad) and torch.equal(got[~bad], clean[~bad])
    M.check_error()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("power,weight,w_offset", [(95, -50, 0.0), (90, -40, 0.0), (95, -60, 0.0), (70, -70, 0.0), (-60, 80, 0.0), (-40, 120, 0.0), (20, -120, 0.0), (0, 122, 2.0 ** 127),
                                                   (30, 0, 1.0)])
@pytest.mark.parametrize("rows,cols", [(3, 300), (700, 1000), (600, 4096), (310, 11008), (2, 40001)])
def test_add_norm_with_weights_far_from_one(fmt, power, weight, w_offset, rows, cols):
    """Roots times weights that are no numbers of fp32, or have few bits there, where the norm is an ordinary one: a block a row, the ring, wide rows.  Some weights, with their offset, are 0."""
    x = numbers(rows, cols, 5)
    x[::2] = np.ldexp(x[::2], power)
    if w_offset == 2.0 ** 127:
        x[:, 0], x[:, 1:] = 2.0 ** 40, x[:, 1:] * 2.0 ** -30      # the norm of most is small
    x = x.astype(np.float32)
    w = np.ldexp(numbers(1, cols, 6)[0], weight).astype(np.float32)
    w[::7] = -w_offset
    s = x.astype(np.float64)
    y = s / np.sqrt((s * s).mean(-1, keepdims=True) + float(np.float32(1e-30))) * (w_offset + w.astype(np.float64))
    y[np.abs(y) >= 2.0 ** 128] = np.inf
    same_matrix(M.add_norm(torch.from_numpy(x).cuda(), None, torch.from_numpy(w).cuda(), eps=1e-30, w_offset=w_offset, format=fmt), y)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows,cols", [(3, 300), (700, 1000), (600, 4096)])
def test_add_norm_with_weights_beyond_fp32(fmt, rows, cols):
    """A weight and its offset whose sum is no number of fp32, on small values: numbers; on large ones: infinite, the block NaN"""
    x = np.full((rows, cols), 2.0 ** -40, np.float32)
    x[:, 0], x[1, 33:] = 2.0 ** 20, 2.0 ** 20
    w = np.full(cols, 3e38, np.float32)
    w_offset = float(np.float32(3e38))
    s = x.astype(np.float64)
    y = s / np.sqrt((s * s).mean(-1, keepdims=True) + float(np.float32(1e-5))) * (w_offset + w.astype(np.float64))
    y[np.abs(y) >= 2.0 ** 128] = np.inf
    assert np.isinf(y[0, 0]) and np.isfinite(y[0, 32:]).all() and (y[0, 32:] != 0).all() and np.isinf(y[1, 40])
    same_matrix(M.add_norm(torch.from_numpy(x).cuda(), None, torch.from_numpy(w).cuda(), eps=1e-5, w_offset=w_offset, format=fmt), y)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("power,weight", [(55, -80), (58, -70), (40, -100), (-30, -60)])
@pytest.mark.parametrize("rows,cols", [(3, 300), (700, 1000), (600, 4096)])
def test_add_norm_with_small_weights_among_others(fmt, power, weight, rows, cols):
    """Weights of whole blocks, and of single columns in others, far below those beside them; blocks of zeros of either sign"""
    x = np.ldexp(numbers(rows, cols, 7), power).astype(np.float32)
    x[:, 96:128] = np.copysign(0.0, np.random.default_rng(8).standard_normal((rows, 32)))
    w = numbers(1, cols, 9)[0]
    w[32:64], w[64:96:2], w[128::3] = np.ldexp(w[32:64], weight), np.ldexp(w[64:96:2], weight), np.ldexp(w[128::3], weight)
    w = w.astype(np.float32)
    s = x.astype(np.float64)
    y = s / np.sqrt((s * s).mean(-1, keepdims=True) + float(np.float32(1e-30))) * w.astype(np.float64)
    same_matrix(M.add_norm(torch.from_numpy(x).cuda(), None, torch.from_numpy(w).cuda(), eps=1e-30, format=fmt), y)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(3, 301), (700, 1000), (600, 4100), (310, 11012), (2, 40001)])
def test_add_norm_with_an_offset_below_zero(fmt, dtype, rows, cols):
    """What pads a row has codes of 0, not those of -0; zeros among the values keep their sign"""
    x, left, w = numbers(rows, cols, 1), numbers(rows, cols, 2), numbers(1, cols, 3)[0]
    x[:, 64:96], left[:, 64:96] = -0.0, -0.0
    x, w = (torch.from_numpy(t.astype(np.float32)).cuda() for t in (x, w))
    l = upload(left, dtype)
    s = (x + l.float()).double().cpu().numpy()
    y = s / np.sqrt((s * s).mean(-1, keepdims=True) + 1e-5) * (-8.5 + w.double().cpu().numpy())
    same_matrix(M.add_norm(x, l, w, eps=1e-5, w_offset=-8.5, format=fmt), y)


# ---- pairs of blocks at the edges of their items; sums -------------------------------------------------------------------------
# Matrices of 61 tiles of 128 rows, so that tiles of 64 activation rows would be more than the SMs have places for.  An item is 256 weight rows x 256 activation rows (128 with a gate): what is left
# of the activation rows is rounded up to 32 and touches one tile of 128 scales or two; 20 and 128 rows in the last item leave its second block without any; 384 columns are three tiles
# of 128 values, an odd number, of which 4-bit stages take two.
LEFT, EDGE_N, EDGE_K = [1, 31, 32, 33, 127, 128, 129], [7700, 7808], 384


@pytest.fixture(scope="module")
def edge():
    made = {}

    def of(n, fmt):
        if (n, fmt) not in made:
            a, gate, up = matrices(256 + 129, n, EDGE_K, fmt, n, 2)
            made[n, fmt] = (a, gate, up, O.values(a), O.values(gate), O.values(up))
        return made[n, fmt]
    return of


def first_rows(a, rows):
    """The first rows of a matrix, in memory of their own, scale bytes behind them 255"""
    m = M.Mx.empty(rows, a.cols, a.format)
    m.codes.view(torch.uint8).copy_(a.codes.view(torch.uint8)[:rows])
    m.scales.copy_(a.scales.view(-1)[:m.scales.numel()])
    tiles = m.scales.view(-1, m.scales.numel() // 512 // -(-rows // 128), 32, 4, 4)
    for lane in range(128):
        if (rows - 1) // 128 * 128 + lane >= rows:
            tiles[-1, :, lane % 32, lane // 32] = 255
    return m


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("n", EDGE_N)
@pytest.mark.parametrize("left", LEFT)
def test_pairs_at_the_edges_of_their_items(fmt, n, left, edge):
    a, gate, up, va, vg, vu = edge(n, fmt)
    rows = 256 + left
    got = M.linear(first_rows(a, rows), up).double().cpu().numpy()
    assert (np.abs(got - va[:rows] @ vu.T) <= sum_bound(va[:rows], vu)).all()
    rows = 128 + left
    m = M.linear_act(first_rows(a, rows), gate, up)
    g, u, bg, bu = va[:rows] @ vg.T, va[:rows] @ vu.T, sum_bound(va[:rows], vg), sum_bound(va[:rows], vu)
    near(m, O.act("silu", g, u, 0, 0), 2.0 ** -126 * np.abs(g) * (1 + np.abs(u)), [O.act("silu", g + s * bg, u + t * bu, 0, 0) for s in (-1, 1) for t in (-1, 1)])
    M.check_error()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows,n,k", [(1, 128, 1000), (20, 260, 4100), (70, 300, 5900), (1100, 2600, 5900)])
@pytest.mark.parametrize("sign", ["one", "both"])
def test_sums_of_whole_numbers_are_exact(fmt, rows, n, k, sign):
    """Products are whole numbers, and |a| |w| adds up to less than 2^24: every sum on the way, in any order, is a number of fp32, and an accumulator with fewer bits would show.  8-bit rows
    are up to 448 under a scale of 1, 4-bit rows up to 6 under a scale of 128 or of 1: in 5900 columns of one sign 2^22 to 2^24, odd sums among them."""
    g = np.random.default_rng(k + rows)
    whole = np.array([1, 2, 3, 4, 6])
    w = np.where(g.random((n, k)) < 0.6, 6, g.choice(whole, (n, k)))
    w[g.random((n, k)) < 0.1] = 0
    if fmt == "e4m3":
        wide = np.array([v for v in O.levels(fmt) if v >= 1 and v == int(v)]).astype(int)
        a = np.where(g.random((rows, k)) < 0.8, g.choice(wide[wide >= 256], (rows, k)), g.choice(wide, (rows, k)))
    else:
        a = g.choice(whole, (rows, k)) * np.where(np.repeat(g.random((rows, -(-k // 32))) < 0.7, 32, 1)[:, :k], 128, 1)
    if sign == "both":
        a, w = a * g.choice([-1, 1], (rows, k)), w * g.choice([-1, 1], (n, k))
    total = np.abs(a).astype(float) @ np.abs(w).astype(float).T
    assert total.max() < 2 ** 24 and (k < 5900 or total.max() > 2 ** 22)
    x, y = torch.from_numpy(a.astype(np.float32)).cuda(), torch.from_numpy(w.astype(np.float32)).cuda()
    ma, mw = M.quantise(x, fmt), M.quantise(y)
    assert torch.equal(ma.read(), x) and torch.equal(mw.read(), y)                   # no code is rounded
    want = a.astype(float) @ w.astype(float).T                                       # exact: all below 2^53
    assert (want % 2 != 0).any()
    assert np.array_equal(M.linear(ma, mw).double().cpu().numpy(), want)
    M.check_error()
