"""Matrices in microscaled numbers: what makes them, the norm that ends in them, and the products over them, on calls that a decoder layer makes.

A row is cut into blocks of 32 values.  A block has one scale, a power of two 2^(c - 127) kept as the byte c, the smallest at which no value of it exceeds the format's largest
number (6 for e2m1, 448 for e4m3); a value's code is the format's number nearest to x / scale, ties to even.  Rows are padded with zeros to a multiple of 128 values; two
codes of e2m1 share a byte, the first in the low half.  Scales lie in tiles of 128 rows and 4 blocks: [row tile][column tile][row % 32][row / 32 % 4][block % 4].

  quant       a matrix is quantised, and read back as the values that its codes stand for
  add_norm    a sublayer's result joins the residual stream, whose root-mean-square norm is quantised: the next product's input
  linear      the product of quantised rows with a matrix in 4 bits
  linear_act  the two input products of a gated feed-forward, its activation, and the result quantised: the input of the product that follows

With `own` the calls go to the framework (hip_llama.cpp_b200/mx.py); without it they are plain torch.
"""
import importlib
import importlib.util
import math
import os
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
BLOCK, TILE = 32, 128
# the largest number of a format as fraction and exponent (frexp), its smallest normal exponent, and its bits of mantissa
TOP = {"e2m1": (0.75, 3), "e4m3": (0.875, 9)}
LEAST = {"e2m1": 0, "e4m3": -6}
MANT = {"e2m1": 1, "e4m3": 3}
EPS = 1e-5


def _package(sub):
    """A module of the package, whose folder name is not an identifier."""
    name, folder = "hip_llama_cpp_b200", os.path.join(ROOT, "hip_llama.cpp_b200")
    if name not in sys.modules:
        spec = importlib.util.spec_from_file_location(name, os.path.join(folder, "__init__.py"), submodule_search_locations=[folder])
        mod = importlib.util.module_from_spec(spec)
        sys.modules[name] = mod
        spec.loader.exec_module(mod)
    return importlib.import_module(name + "." + sub)


# ---- cases ----------------------------------------------------------------------------------------------------------------
def _case(name, kind, rows, cols, n=0, **more):
    """rows x cols: the call's rows; n: the matrix's rows, for linear_act those of each of the two; format: the rows' (linear_act: the result's too); dtype: what is plain."""
    return dict(name=name, kind=kind, rows=rows, cols=cols, n=n, **more)


def listed():
    return [
        # one decoded token's attention result of the small model
        _case("quant 1 row small", "quant", 1, 768, format="e4m3", dtype="f32", wide=0),
        # a matrix of the large model on its way into 4 bits
        _case("quant weights 7B", "quant", 11008, 4096, format="e2m1", dtype="bf16", wide=0),
        # prompt rows of an odd width, columns of a wider product
        _case("quant ragged columns", "quant", 1333, 1365, format="e2m1", dtype="f32", wide=75),
        # between two sublayers of the large model: one decoded token, and a prompt
        _case("add_norm 1 row 7B", "add_norm", 1, 4096, format="e4m3", dtype="bf16"),
        _case("add_norm prompt 7B", "add_norm", 2048, 4096, format="e4m3", dtype="f32"),
        # one decoded token through the attention's output product of the large model
        _case("linear 1 row 7B", "linear", 1, 4096, 4096, format="e4m3", dtype="f32"),
        # a full batch of decoded tokens through the down product
        _case("linear 64 rows down 7B", "linear", 64, 11008, 4096, format="e4m3", dtype="bf16"),
        # a prompt through the stacked q, k, v product
        _case("linear prompt qkv 7B", "linear", 2048, 4096, 12288, format="e4m3", dtype="f32"),
        # prompts of ragged length with rows in 4 bits, too
        _case("linear prompts 4 bit", "linear", 3333, 4096, 11008, format="e2m1", dtype="bf16"),
        # the small model's feed-forward for one token
        _case("linear_act 1 row small", "linear_act", 1, 768, 2048, format="e4m3", dtype="bf16"),
        # the large model's feed-forward: a batch of decoded tokens, and a prompt
        _case("linear_act 16 rows 7B", "linear_act", 16, 4096, 11008, format="e4m3", dtype="bf16"),
        _case("linear_act prompt 7B", "linear_act", 2048, 4096, 11008, format="e4m3", dtype="bf16"),
    ]


def _log_between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["quant", "add_norm", "linear", "linear", "linear", "linear_act", "linear_act"])
    c = dict(kind=kind, format=rng.choice(["e4m3", "e4m3", "e2m1"]), dtype=rng.choice(["f32", "bf16"]), n=0)
    rows = rng.choice([1, _log_between(rng, 2, 64), _log_between(rng, 2, 4096)])
    # widths of layers are round, those of slices and of small models are not
    width = lambda hi: 64 * _log_between(rng, 2, hi // 64) if rng.random() < 0.6 else _log_between(rng, 33, hi)  # noqa: E731
    if kind in ("quant", "add_norm"):
        c.update(rows=rows if rng.random() < 0.6 else _log_between(rng, 2, 12000), cols=width(14336))
        while c["rows"] * c["cols"] > 4.5e7 / (4 if kind == "add_norm" else 1):
            c["rows"] = c["rows"] * 3 // 4
        if kind == "quant":
            c["wide"] = rng.choice([0, 0, 8, rng.randint(1, 500)])
        return c
    c.update(rows=rows, cols=width(14336), n=width(16384))
    most = 3e11 / (2 if kind == "linear_act" else 1)
    while 2.0 * c["rows"] * c["cols"] * c["n"] > most:
        c["rows"] = c["rows"] * 3 // 4
    while c["cols"] * c["n"] > (3.0e7 if kind == "linear_act" else 6.0e7):
        c["n"] = c["n"] * 3 // 4
    if kind == "linear_act":
        c["dtype"] = "bf16"
    return c


def _padded(cols):
    return -(-cols // TILE) * TILE


def _held(rows, cols, fmt):
    """Bytes of a matrix: codes and scales"""
    return rows * cols * (4 if fmt == "e2m1" else 8) / 8 + rows * -(-cols // BLOCK)


def work(case):
    r, c, n, fmt = case["rows"], case["cols"], case["n"], case["format"]
    size = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "quant":
        return {"bytes": r * c * (size + 2) + _held(r, c, fmt), "flops": 2 * r * c}
    if case["kind"] == "add_norm":
        return {"bytes": r * c * (8 + size + 2) + 4 * c + _held(r, c, fmt), "flops": 6 * r * c}
    if case["kind"] == "linear":
        return {"bytes": _held(r, c, fmt) + _held(n, c, "e2m1") + r * n * size, "flops": 2 * r * c * n}
    return {"bytes": _held(r, c, fmt) + 2 * _held(n, c, "e2m1") + _held(r, n, fmt) + 2 * r * n, "flops": 4 * r * c * n}


# ---- numbers and layout ---------------------------------------------------------------------------------------------------
def _nearest(y, fmt):
    """The format's number nearest to y, ties to even: a multiple of the step of |y|'s binade.  y in 64 bits, at most the format's largest."""
    e = torch.frexp(y.abs())[1] - 1
    step = torch.ldexp(torch.ones_like(y), e.clamp_min(LEAST[fmt]) - MANT[fmt])
    return torch.round(y / step) * step


def _quantise(x, fmt):
    """x [rows, cols] -> (numbers of the format [rows, padded], scale bytes [rows, blocks]); in 64 bits, where the norm's values keep what decides at a border"""
    y = torch.nn.functional.pad(x.double(), (0, _padded(x.shape[1]) - x.shape[1])).unflatten(1, (-1, BLOCK))
    top = y.abs().amax(-1)
    frac, exp = torch.frexp(top)
    m, e = TOP[fmt]
    exp = exp - e + (frac > m)
    byte = torch.where(top > 0, (exp + 127).clamp_min(0), torch.zeros_like(exp))
    return _nearest(torch.ldexp(y, (127 - byte)[..., None]), fmt).flatten(1), byte


def _codes(v, fmt):
    """Numbers of the format as bytes"""
    if fmt == "e4m3":
        return v.float().to(torch.float8_e4m3fn)
    a = v.abs()
    c = torch.where(a < 2, 2 * a, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8) | (torch.signbit(v).to(torch.uint8) << 3)
    return c[:, 0::2] | (c[:, 1::2] << 4)


def _tiles(byte):
    """Scale bytes [rows, blocks] in the order that the framework keeps them in; what pads the last row tile holds 0"""
    rows = byte.shape[0]
    return torch.nn.functional.pad(byte, (0, 0, 0, -rows % TILE)).to(torch.uint8).view(-1, 4, 32, byte.shape[1] // 4, 4).permute(0, 3, 2, 1, 4).contiguous()


def _made(x, fmt):
    v, byte = _quantise(x, fmt)
    return {"codes": _codes(v, fmt), "scales": _tiles(byte), "rows": x.shape[0], "cols": x.shape[1], "format": fmt}


def _numbers(m, dtype):
    """The codes of a matrix as numbers [rows, padded]"""
    if m["format"] == "e4m3":
        return m["codes"].to(dtype)
    c = torch.stack([m["codes"] & 15, m["codes"] >> 4], -1).flatten(1).int()
    return torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=dtype, device=c.device)[c]


def _values(m, dtype):
    """What a matrix stands for, [rows, cols]"""
    byte = m["scales"].permute(0, 3, 2, 1, 4).flatten(0, 2).flatten(1)[:m["rows"]].int()
    x = _numbers(m, dtype).unflatten(1, (-1, BLOCK))
    return torch.ldexp(x, (byte - 127)[..., None]).flatten(1)[:, :m["cols"]]


# ---- inputs ---------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    r, c, n, fmt, kind = case["rows"], case["cols"], case["n"], case["format"], case["kind"]
    rand = lambda *shape: torch.randn(*shape, device=dev, generator=g)  # noqa: E731
    channels = torch.exp(0.7 * rand(c))                      # a few channels of real rows are several times larger than the others
    s = {"case": case}
    if kind == "quant":
        x = rand(r, c + case["wide"]) * torch.nn.functional.pad(channels, (0, case["wide"]), value=1.0)
        s["x"] = x.to(TYPES[case["dtype"]])[:, :c]           # columns of a wider product
    elif kind == "add_norm":
        s["x"] = rand(r, c) * channels
        s["left"] = (0.3 * rand(r, c)).to(TYPES[case["dtype"]])
        s["weight"] = torch.exp(0.3 * rand(c))
    else:
        s["a"] = _made(rand(r, c) * channels, fmt)
        for name in ("w",) if kind == "linear" else ("gate", "up"):
            s[name] = _made(rand(n, c) * torch.exp(0.4 * rand(n, 1)) / c ** 0.5, "e2m1")
    return s


# ---- plain forms ----------------------------------------------------------------------------------------------------------
def _read_back(x, fmt, dtype=torch.float32):
    """What the codes of x stand for, without the codes themselves"""
    v, byte = _quantise(x, fmt)
    return torch.ldexp(v.unflatten(1, (-1, BLOCK)), (byte - 127)[..., None]).flatten(1)[:, :x.shape[1]].to(dtype)


def _plain(s):
    case = s["case"]
    if case["kind"] == "quant":
        return _read_back(s["x"], case["format"], torch.bfloat16)
    if case["kind"] == "add_norm":
        x = s["x"] + s["left"].float()                       # the residual stream is kept in 32 bits
        y = x.double()                                       # 64 bits: values next to a border between two codes
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + EPS) * s["weight"].double()
        return {"x": x, "y": _read_back(y, case["format"], torch.bfloat16)}
    a = _values(s["a"], torch.float32)
    if case["kind"] == "linear":
        return (a @ _values(s["w"], torch.float32).T).to(TYPES[case["dtype"]])
    gate, up = a @ _values(s["gate"], torch.float32).T, a @ _values(s["up"], torch.float32).T
    return _read_back(gate / (1 + torch.exp(-gate)) * up, case["format"], torch.bfloat16)


# ---- the framework's calls ------------------------------------------------------------------------------------------------
def _own(s):
    mx, case = _package("mx"), s["case"]
    if case["kind"] == "quant":
        return mx.quantise(s["x"], case["format"]).read(torch.bfloat16)
    if case["kind"] == "add_norm":
        if "sum" not in s:
            s["sum"] = torch.empty_like(s["x"])              # a layer's residual stream in front of and behind the addition
        y = mx.add_norm(s["x"], s["left"], s["weight"], eps=EPS, format=case["format"], x_out=s["sum"])
        return {"x": s["sum"], "y": y.read(torch.bfloat16)}
    if "bound" not in s:                                     # the handles that a program keeps of its matrices
        s["bound"] = {k: mx.Mx(s[k]["codes"], s[k]["scales"], s[k]["rows"], s[k]["cols"]) for k in ("a", "w", "gate", "up") if k in s}
    b = s["bound"]
    if case["kind"] == "linear":
        return mx.linear(b["a"], b["w"], dtype=TYPES[case["dtype"]])
    return mx.linear_act(b["a"], b["gate"], b["up"], act="silu", format=case["format"]).read(torch.bfloat16)


def run(state):
    return _own(state) if own else _plain(state)


# ---- from the definitions, in 64 bits -------------------------------------------------------------------------------------
def _levels(fmt):
    """The format's numbers from 0 up, and the borders between them"""
    if fmt == "e2m1":
        v = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
    else:
        v = torch.tensor([(m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)) for e in range(16) for m in range(8)][:127], dtype=torch.float64)
    return v.cuda(), ((v[1:] + v[:-1]) / 2).cuda()


def _stands_for(x, fmt):
    """x in 64 bits -> the values of its codes: every scale is found by trying the powers of two from a low one up"""
    rows, cols = x.shape
    v, edge = _levels(fmt)
    pad = torch.zeros(rows, -cols % BLOCK, dtype=torch.float64, device=x.device)
    y = torch.cat([x.double(), pad], 1).view(rows, -1, BLOCK)
    top = y.abs().max(-1).values
    power = (torch.floor(torch.log2(torch.where(top > 0, top, 1.0))) - 12).clamp(min=-127)
    for _ in range(16):
        power = torch.where(top > v[-1] * torch.pow(2.0, power), power + 1, power)
    power = torch.where(top > 0, power, -127.0)
    y = y * torch.pow(2.0, -power)[..., None]
    i = torch.searchsorted(edge, y.abs().contiguous())       # borders below |y|; a border itself belongs to the even neighbour
    i = i + ((i < len(edge)) & (edge[i.clamp(max=len(edge) - 1)] == y.abs()) & (i % 2 == 1)).long()
    return (torch.copysign(v[i], y) * torch.pow(2.0, power)[..., None]).reshape(rows, -1)[:, :cols]


def _stored(m):
    """The values of a made matrix in 64 bits, by the place that the layout gives each byte"""
    rows, cols = m["rows"], m["cols"]
    r, k = torch.arange(rows, device="cuda")[:, None], torch.arange(cols, device="cuda")[None]
    b = k // BLOCK
    across = _padded(cols) // TILE
    at = ((r // 128) * across + b // 4) * 512 + (r % 32) * 16 + (r // 32 % 4) * 4 + b % 4
    scale = torch.pow(2.0, m["scales"].flatten()[at].double() - 127)
    if m["format"] == "e4m3":
        return m["codes"][:, :cols].double() * scale
    c = (m["codes"].long()[:, k[0] // 2] >> (4 * (k % 2))) & 15
    v, _ = _levels("e2m1")
    return torch.where(c >= 8, -v[c % 8], v[c % 8]) * scale


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "quant":
        return _stands_for(s["x"].double(), case["format"])
    if case["kind"] == "add_norm":
        x = (s["x"].double() + s["left"].double()).float().double()      # as the residual stream holds it
        y = x * torch.rsqrt(torch.mean(torch.square(x), 1) + EPS)[:, None] * s["weight"].double()[None]
        return {"x": x, "y": _stands_for(y, case["format"])}
    a = _stored(s["a"])
    if case["kind"] == "linear":
        return torch.einsum("rk,nk->rn", a, _stored(s["w"]))
    gate, up = (torch.einsum("rk,nk->rn", a, _stored(s[m])) for m in ("gate", "up"))
    return _stands_for(torch.nn.functional.silu(gate) * up, case["format"])
