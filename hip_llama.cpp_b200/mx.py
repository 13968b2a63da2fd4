"""Python binding of the matrices in microscaled numbers (tha_mx_t and tha_hyb_mx_* in include/tha_hybrid.h): 4 and 8 bits a value under a power of two for each 32.

    w = quantise(weight)                                         # [n, k] fp32 or bf16 -> 4 bits (e2m1)
    a = add_norm(x, attention, norm, eps=1e-5)                   # x += attention; its norm in 8 bits (e4m3)
    h = linear_act(a, gate, up)                                  # silu(a gate^T) * (a up^T) in 8 bits
    y = linear(h, down, dtype=torch.bfloat16)                    # [rows, n]
    w.read(torch.float32)                                        # the values that the codes stand for

Calls go to the current stream of the tensors' device, which has to be the current device, and do not wait for it; results are allocated by torch on that stream.  Nothing is kept between calls.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import cabi

I, F, P, L = C.c_int, C.c_float, C.c_void_p, C.c_longlong
DTYPES = {torch.bfloat16: 0, torch.float32: 1}                  # THA_DT_*
FORMATS = {"e2m1": 0, "e4m3": 1}                                # THA_MX_*
CODES = {torch.uint8: "e2m1", torch.float8_e4m3fn: "e4m3"}      # what holds them
ACTS = {"clamped": 0, "relu2": 1, "gelu": 2, "xielu": 3, "silu": 4}    # THA_ACT_*
UNGATED = ("relu2", "xielu")
WITH_NUMBERS = ("clamped", "xielu")                             # that take limit and alpha
BLOCK, TILE, MOST = 32, 128, 1 << 30


class MxStruct(C.Structure):
    _fields_ = [("codes", P), ("scales", P), ("rows", I), ("cols", I), ("format", I)]


MxStruct.__name__ = "tha_mx_t"
STRUCTS = (MxStruct,)

# the current device, and the number of its current stream; the public calls look around and make an object first, 1 and 3.3 us
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)
_lib = _c = None


def _load():
    """The library's calls, their arguments' types set."""
    global _lib, _c
    _lib = cabi.lib()
    c, M = _lib.c, C.POINTER(MxStruct)
    c.tha_hyb_mx_quant.argtypes = [P, I, P, L, M]
    c.tha_hyb_mx_read.argtypes = [P, I, M, P, L]
    c.tha_hyb_mx_add_norm.argtypes = [P, I, P, P, L, P, P, F, F, M]
    c.tha_hyb_mx_linear.argtypes = [P, I, P, L, M, M]
    c.tha_hyb_mx_linear_act.argtypes = [P, I, M, M, M, F, F, M]
    for name in ("tha_hyb_mx_codes_bytes", "tha_hyb_mx_scales_bytes"):
        getattr(c, name).restype = C.c_size_t
    c.tha_hyb_mx_codes_bytes.argtypes, c.tha_hyb_mx_scales_bytes.argtypes = [I, I, I], [I, I]
    _c = c
    return c


def lib():
    if _c is None:
        _load()
    return _lib


def padded(cols: int) -> int:
    """The columns that a row of codes has room for."""
    return -(-cols // TILE) * TILE


def tiles(scales):
    """Scale bytes [rows, blocks of 32] in the order in which a matrix keeps them, [row tiles, column tiles, 32, 4, 4]."""
    rows, blocks = scales.shape
    s = torch.nn.functional.pad(scales, (0, -blocks % 4, 0, -rows % TILE))
    return s.view(-1, 4, 32, s.shape[1] // 4, 4).permute(0, 3, 2, 1, 4).contiguous()


class Mx:
    """A matrix of rows x cols microscaled numbers.  codes: uint8 [rows, padded(cols) / 2] (e2m1, two a byte, the first in the low half) or float8_e4m3fn [rows, padded(cols)], what is padding 0;
    scales: uint8 in the order of `tiles`, 255: NaN."""

    _codes = _scales = None                                     # until they are asked for, where a call made room

    def __init__(self, codes, scales, rows: int, cols: int):
        if codes.dtype not in CODES:
            raise ValueError(f"codes are uint8 (e2m1, two a byte) or float8_e4m3fn, not {codes.dtype}")
        if not 0 <= rows <= MOST or not 1 <= cols <= MOST:
            raise ValueError(f"a matrix has rows and at least one column, got {rows} x {cols}")
        format = CODES[codes.dtype]
        width, count = padded(cols) // (2 if format == "e2m1" else 1), -(-rows // TILE) * padded(cols) * TILE // BLOCK
        if codes.shape != (rows, width) or not codes.is_contiguous() or codes.data_ptr() % 32:
            raise ValueError(f"codes: contiguous [{rows}, {width}] on a 32-byte boundary is needed, got {tuple(codes.shape)}, strides {codes.stride()}")
        if scales.dtype != torch.uint8 or not scales.is_contiguous() or scales.numel() != count or scales.device != codes.device or scales.data_ptr() % 16:
            raise ValueError(f"scales: {count} contiguous bytes on {codes.device} and a 16-byte boundary are needed, got {tuple(scales.shape)} {scales.dtype} on {scales.device}")
        self._codes, self._scales = codes, scales
        self.rows, self.cols, self.format, self.device = rows, cols, format, codes.device
        self.c = MxStruct(codes.data_ptr(), scales.data_ptr(), rows, cols, FORMATS[format])

    @classmethod
    def empty(cls, rows: int, cols: int, format: str = "e2m1", device="cuda"):
        """Room for a matrix: what a call fills.  Codes and scales are one piece of memory; the tensors over them are made when they are asked for."""
        kind = FORMATS.get(format)
        if kind is None or not 0 <= rows <= MOST or not 1 <= cols <= MOST:
            raise ValueError(f"a matrix of rows and at least one column in e2m1 or e4m3, not {rows} x {cols} in {format!r}")
        wide = (cols + 127) & -128
        scales = (rows * (wide if kind else wide >> 1) + 511) & -512
        m = cls.__new__(cls)
        m._room = room = torch.empty(scales + ((rows + 127) & -128) * (wide >> 5), dtype=torch.uint8, device=device)
        at = room.data_ptr()
        m.rows, m.cols, m.format, m.device = rows, cols, format, room.device
        m.c = MxStruct(at, at + scales, rows, cols, kind)
        return m

    @property
    def codes(self):
        if self._codes is None:
            width = padded(self.cols) // (2 if self.format == "e2m1" else 1)
            t = self._room[:self.rows * width].view(self.rows, width)
            self._codes = t if self.format == "e2m1" else t.view(torch.float8_e4m3fn)
        return self._codes

    @property
    def scales(self):
        if self._scales is None:
            self._scales = self._room[self._room.numel() - -(-self.rows // TILE) * padded(self.cols) * TILE // BLOCK:]
        return self._scales

    @classmethod
    def of_rows(cls, codes, scales, cols: int):
        """From codes and scale bytes row by row, as checkpoints have them: codes uint8 [rows, cols / 2 rounded up] or float8_e4m3fn [rows, cols], scales uint8 [rows, cols / 32 rounded up]."""
        kind = CODES.get(codes.dtype)
        width = -(-cols // 2) if kind == "e2m1" else cols
        if kind is None or codes.dim() != 2 or codes.shape[1] != width or scales.dtype != torch.uint8 or scales.shape != (codes.shape[0], -(-cols // BLOCK)):
            raise ValueError(f"codes [rows, {width}] and scales uint8 [rows, {-(-cols // BLOCK)}] are needed, got {tuple(codes.shape)} {codes.dtype}, {tuple(scales.shape)} {scales.dtype}")
        c = codes.view(torch.uint8)
        if kind == "e2m1" and cols % 2:
            c = torch.cat([c[:, :-1], c[:, -1:] & 15], 1)        # the last byte's other half is padding
        c = torch.nn.functional.pad(c, (0, padded(cols) // (2 if kind == "e2m1" else 1) - width)).contiguous()
        return cls(c if kind == "e2m1" else c.view(torch.float8_e4m3fn), tiles(scales), codes.shape[0], cols)

    def read(self, dtype=torch.float32, out=None):
        """The values that the codes stand for (tha_hyb_mx_read), [rows, cols]."""
        out, kind, ld = _result(out, self.rows, self.cols, dtype, self.device)
        status = (_c or _load()).tha_hyb_mx_read(_stream(self.device), kind, self.c, out.data_ptr(), ld)
        if status:
            _lib.check(status, "tha_hyb_mx_read")
        return out


# What a call costs on the host decides small sizes (7 to 8 us of which the launch is 2): arguments are looked at once, in few steps.
def _pitch(name, t, rows, cols, device):
    """The row pitch of t [rows, cols], whose columns are neighbours."""
    s = t.stride()
    if t.shape != (rows, cols) or t.dtype not in DTYPES or t.device != device or (rows and cols > 1 and s[1] != 1) or (rows > 1 and s[0] < cols):
        raise ValueError(f"{name}: [{rows}, {cols}] float32 or bfloat16 with neighbouring columns on {device} is needed, got {tuple(t.shape)} {t.dtype} on {t.device}, strides {s}")
    return s[0] if rows > 1 else cols


def _floats(name, t, shape, device):
    if t.shape != shape or t.dtype != torch.float32 or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name}: contiguous float32 {list(shape)} on {device} is needed, got {tuple(t.shape)} {t.dtype} on {t.device}, strides {t.stride()}")


def _result(out, rows, cols, dtype, device):
    """(`out` or room for it, its THA_DT_*, its pitch)"""
    if out is not None:
        return out, DTYPES.get(out.dtype), _pitch("out", out, rows, cols, device)
    kind = DTYPES.get(dtype)
    if kind is None:
        raise ValueError(f"results are float32 or bfloat16, not {dtype}")
    return torch.empty(rows, cols, dtype=dtype, device=device), kind, cols


def _matrix(m, rows, cols, format, device):
    """`m`, which has to have this size"""
    if (m.rows, m.cols, m.device) != (rows, cols, device):
        raise ValueError(f"out: {rows} x {cols} on {device} is needed, got {m.rows} x {m.cols} on {m.device}")
    if format not in FORMATS:
        raise ValueError(f"a format is e2m1 or e4m3, not {format!r}")
    return m


def _stream(device):
    """The current stream of a device that has to be the current one."""
    index = device.index
    if index is None or _current_device() != index:
        raise ValueError(f"the tensors are on {device}, the current device is cuda:{torch.cuda.current_device() if torch.cuda.is_available() else None}")
    return _raw_stream(index)


def check_error(device="cuda") -> None:
    """Waits for the current stream of a device; raises if a kernel on it gave up on a barrier since the last such question (the results of that call are NaN where it was)."""
    with torch.cuda.device(device):                             # whose kernels the library is asked about
        torch.cuda.current_stream().synchronize()
        gave_up = (_c or _load()).tha_gemm_check_error()
    if gave_up:
        raise cabi.ThaError("a kernel gave up on a barrier of its own")


def quantise(x, format: str = "e2m1", out: Mx | None = None) -> Mx:
    """x [rows, cols], fp32 or bf16, rows any pitch apart, as microscaled numbers (tha_hyb_mx_quant).  out: room for them, in its own format."""
    shape, device = x.shape, x.device
    if len(shape) != 2:
        raise ValueError(f"x: [rows, columns] is needed, got {tuple(shape)}")
    rows, cols = shape
    ldx = _pitch("x", x, rows, cols, device)
    out = Mx.empty(rows, cols, format, device) if out is None else _matrix(out, rows, cols, format, device)
    status = (_c or _load()).tha_hyb_mx_quant(_stream(device), DTYPES[x.dtype], x.data_ptr(), ldx, out.c)
    if status:
        _lib.check(status, "tha_hyb_mx_quant")
    return out


def add_norm(x, left, weight, *, eps: float, w_offset: float = 0.0, format: str = "e4m3", x_out=None, out: Mx | None = None) -> Mx:
    """x + left (fp32 [rows, cols] and fp32 or bf16 of any pitch; left None: x alone) into x_out (None: x itself); its root-mean-square norm, weighted with w_offset + weight,
    as microscaled numbers (tha_hyb_mx_add_norm)."""
    shape, device = x.shape, x.device
    if len(shape) != 2:
        raise ValueError(f"x: [rows, columns] is needed, got {tuple(shape)}")
    rows, cols = shape
    _floats("x", x, shape, device)
    if x_out is None:
        x_out = x
    else:
        _floats("x_out", x_out, shape, device)
    _floats("weight", weight, shape[1:], device)
    kind, at, ldl = 1, None, 0
    if left is not None:
        ldl, kind, at = _pitch("left", left, rows, cols, device), DTYPES[left.dtype], left.data_ptr()
    out = Mx.empty(rows, cols, format, device) if out is None else _matrix(out, rows, cols, format, device)
    status = (_c or _load()).tha_hyb_mx_add_norm(_stream(device), kind, x.data_ptr(), at, ldl, x_out.data_ptr(), weight.data_ptr(), w_offset, eps, out.c)
    if status:
        _lib.check(status, "tha_hyb_mx_add_norm")
    return out


def linear(a: Mx, w: Mx, dtype=torch.float32, out=None):
    """a [rows, k] times w [n, k] transposed (tha_hyb_mx_linear): [rows, n], fp32 or bf16.  w is e2m1."""
    device = a.device
    if device != w.device:
        raise ValueError(f"the rows are on {device}, the matrix is on {w.device}")
    out, kind, ld = _result(out, a.rows, w.rows, dtype, device)
    status = (_c or _load()).tha_hyb_mx_linear(_stream(device), kind, out.data_ptr(), ld, a.c, w.c)
    if status:
        _lib.check(status, "tha_hyb_mx_linear")
    return out


def linear_act(a: Mx, gate: Mx | None, up: Mx, act: str = "silu", format: str = "e4m3", limit: float | None = None, alpha: float | None = None,
               out: Mx | None = None) -> Mx:
    """A feed-forward's input products and activation (tha_hyb_mx_linear_act): act(a gate^T, a up^T) [rows, n] as microscaled numbers.  act: silu, gelu, clamped (limit, alpha), or without a gate
    (None) relu2, xielu (its two stored numbers as limit, alpha)."""
    device, kind = a.device, ACTS.get(act)
    if kind is None:
        raise ValueError(f"act is one of {', '.join(ACTS)}, not {act!r}")
    if (gate is None) != (act in UNGATED):
        raise ValueError(f"{act} {'has no gate' if act in UNGATED else 'needs a gate'}")
    if limit is None or alpha is None:
        if act in WITH_NUMBERS:
            raise ValueError(f"{act} needs limit and alpha")
        limit = alpha = 0.0
    if up.device != device or (gate is not None and gate.device != device):
        raise ValueError(f"the rows are on {device}, a matrix is not")
    out = Mx.empty(a.rows, up.rows, format, device) if out is None else _matrix(out, a.rows, up.rows, format, device)
    status = (_c or _load()).tha_hyb_mx_linear_act(_stream(device), kind, a.c, None if gate is None else gate.c, up.c, limit, alpha, out.c)
    if status:
        _lib.check(status, "tha_hyb_mx_linear_act")
    return out
