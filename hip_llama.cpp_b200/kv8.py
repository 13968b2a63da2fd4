"""Python binding of the key/value cache in 8 bits (tha_kv8_t and tha_hyb_kv8_* in include/tha_hybrid.h).

    cache = Kv8Cache.empty(blocks=512, layers=2, kv_heads=8, block_size=16, dim=128, slots=4, table_stride=64)
    cache.table.copy_(...)                                       # [slots, table_stride] block ids, the caller's to hand out
    rows = Rows.of([(0, 0, 300), (2, 17, 1)])                    # slot 0: positions 0 .. 299, slot 2: position 17
    cache.write(rows, k, v, layer=0)                             # k [301, 8 * 128]: rows or columns of a wider product
    out = cache.attend(Attention(32, 8, 128, scale=128 ** -0.5), rows, q, layer=0)   # [301, 32 * 128]
    k, v = cache.read(rows, layer=0)                             # the values that the codes stand for

Calls go to the current stream of the cache's device, which has to be the current device.  Nothing synchronises.  Results and scratch are allocated by torch on
that stream, so that calls on several streams, and captured ones, share nothing; a cache is written by one stream at a time.
"""
from __future__ import annotations

import ctypes as C

import numpy as np
import torch

from . import cabi

I, F, P, L = C.c_int, C.c_float, C.c_void_p, C.c_longlong
DTYPES = {torch.bfloat16: 0, torch.float32: 1}                  # THA_DT_*
FORMATS = {torch.int8: 0, torch.float8_e4m3fn: 1}               # THA_KV8_*


def _struct(name, fields):
    return type(name, (C.Structure,), {"_fields_": [(n, t) for names, t in fields for n in names.split()]})


RowsStruct = _struct("tha_rows_t", [("n_rows n_seqs", I), ("token pos row_seq seq_first seq_slot", P), ("max_seq_rows max_pos", I)])
AttnStruct = _struct("tha_attn_t", [("heads kv_heads dim vdim rot unit_rms", I), ("eps scale", F), ("chunk cache_layer o_q o_k o_v", I), ("w_o", P),
                                    ("values_in_keys window keep_first", I), ("sink head_scale", P), ("rot_layout head_gate o_g fp32_scores v_share out_f32", I),
                                    ("q_temp_coef", F), ("q_temp_every kv_shared diff", I), ("diff_lambda diff_mult", F), ("conv_taps", I), ("conv_w", P),
                                    ("conv_state_off", L), ("conv_b", P), ("v_is_k", I), ("q_norm k_norm", P), ("softcap", F), ("b_o", P), ("head_norm", I),
                                    ("rel", P), ("rel_n v_mix v_mix_layer", I), ("v_mix_lambda", F)])
Kv8Struct = _struct("tha_kv8_t", [("k_pool v_pool k_scale v_scale k_open v_open table", P),
                                  ("table_stride block_size n_blocks n_cache_layers kv_heads dim vdim format", I)])
STRUCTS = (RowsStruct, AttnStruct, Kv8Struct)

_lib = None


def lib():
    global _lib
    if _lib is None:
        _lib = cabi.lib()
        c, R, K, A = _lib.c, C.POINTER(RowsStruct), C.POINTER(Kv8Struct), C.POINTER(AttnStruct)
        c.tha_hyb_kv8_write.argtypes = [P, I, R, K, I, P, L, P, L]
        c.tha_hyb_kv8_read.argtypes = [P, I, R, K, I, P, L, P, L]
        c.tha_hyb_kv8_attn.argtypes = [P, I, A, R, K, P, P, P, C.c_size_t, P, L]
        c.tha_hyb_kv8_attn_scratch.argtypes = [I, A, R, K]
        c.tha_hyb_kv8_attn_scratch.restype = C.c_size_t
    return _lib


def _ints(name, t, count):
    if t.dtype != torch.int32 or not t.is_contiguous() or t.numel() < count:
        raise ValueError(f"{name}: {count} contiguous int32 values are needed, got {tuple(t.shape)} {t.dtype}")


def _floats(name, t, count, device):
    if t.dtype != torch.float32 or not t.is_contiguous() or t.numel() < count or t.device != device:
        raise ValueError(f"{name}: {count} contiguous float32 values on {device} are needed, got {tuple(t.shape)} {t.dtype} on {t.device}")


class Rows:
    """The rows of a step (tha_rows_t): device arrays of every row's position and sequence, every sequence's first row and slot."""

    slots = None                                                # what Rows.of knows of the slots: (lowest, highest, whether all sequences with rows to write differ)

    def __init__(self, pos, row_seq, seq_first, seq_slot, max_seq_rows: int, max_pos: int):
        n, s = pos.numel(), seq_slot.numel()
        for name, t, count in (("pos", pos, n), ("row_seq", row_seq, n), ("seq_first", seq_first, s + 1), ("seq_slot", seq_slot, s)):
            _ints(name, t, count)
            if t.device != pos.device:
                raise ValueError(f"{name} is on {t.device}, pos on {pos.device}")
        self.n, self.device = n, pos.device
        self._keep = (pos, row_seq, seq_first, seq_slot)
        self.c = RowsStruct(n, s, None, pos.data_ptr(), row_seq.data_ptr(), seq_first.data_ptr(), seq_slot.data_ptr(), max_seq_rows, max_pos)
        self.ref = C.byref(self.c)

    @classmethod
    def of(cls, portions, device="cuda"):
        """portions: [(slot, first position, rows)], at least one row each; (slot, -1, 1): an idle slot."""
        if not portions or any(n < 1 or (p < 0 and n > 1) for _, p, n in portions):
            raise ValueError("a portion has at least one row, and one row where its position is negative")
        pos = np.concatenate([p + np.arange(n) for _, p, n in portions])
        first = np.cumsum([0] + [n for _, _, n in portions])
        seq = np.repeat(np.arange(len(portions)), np.diff(first))
        put = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(device)  # noqa: E731
        rows = cls(put(pos), put(seq), put(first), put([s for s, _, _ in portions]), max(n for _, _, n in portions), int(pos.max()))
        live, every = [s for s, p, _ in portions if p >= 0], [s for s, _, _ in portions]
        rows.slots = (min(every), max(every), len(set(live)) == len(live))
        return rows


class Attention:
    """The attention of a layer as far as a call over a cache goes (tha_attn_t, whose comments say what each argument does).  sink, head_scale: [heads], rel: [heads, n],
    fp32 on the device.  head_gate: sigmoid of column gate_column + h of `proj` scales head h's result."""

    def __init__(self, heads: int, kv_heads: int, dim: int, vdim: int | None = None, *, scale: float, chunk: int = 0, window: int = 0, keep_first: int = 0, sink=None,
                 head_scale=None, softcap: float = 0.0, rel=None, head_gate: bool = False, gate_column: int = 0):
        for name, t, count in (("sink", sink, heads), ("head_scale", head_scale, heads)):
            if t is not None:
                _floats(name, t, count, t.device)
        if rel is not None:
            _floats("rel", rel, heads, rel.device)
            if rel.dim() != 2 or rel.shape[0] != heads or rel.shape[1] < 1:
                raise ValueError(f"rel: [heads, distances] is needed, got {tuple(rel.shape)}")
        self._keep = (sink, head_scale, rel)
        self.device = next((t.device for t in self._keep if t is not None), None)
        if any(t is not None and t.device != self.device for t in self._keep):
            raise ValueError("sink, head_scale and rel are on different devices")
        at = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        self.c = AttnStruct(heads=heads, kv_heads=kv_heads, dim=dim, vdim=dim if vdim is None else vdim, rot=-1, scale=scale, chunk=chunk, window=window,
                            keep_first=keep_first, sink=at(sink), head_scale=at(head_scale), softcap=softcap, rel=at(rel),
                            rel_n=0 if rel is None else rel.shape[1], head_gate=int(head_gate), o_g=gate_column)
        self.ref = C.byref(self.c)


class Kv8Cache:
    """Pools of codes [blocks, layers, kv heads, block size, channels] (int8 or float8_e4m3fn), their scales [blocks, layers, kv heads], the fp32 rows of every slot's last
    block [slots, layers, kv heads, block size, channels] and the block table [slots, blocks per slot] int32.  k_open, v_open None: a cache that is only read."""

    def __init__(self, k_pool, v_pool, k_scale, v_scale, k_open, v_open, table):
        if k_pool.dtype not in FORMATS or v_pool.dtype != k_pool.dtype:
            raise ValueError(f"pools of int8 or float8_e4m3fn are needed, got {k_pool.dtype} and {v_pool.dtype}")
        if k_pool.dim() != 5 or v_pool.dim() != 5 or k_pool.shape[:4] != v_pool.shape[:4] or not k_pool.is_contiguous() or not v_pool.is_contiguous():
            raise ValueError("pools are contiguous [blocks, layers, kv heads, block size, channels], K and V alike but for the channels")
        if (k_open is None) != (v_open is None):
            raise ValueError("k_open and v_open come together")
        blocks, layers, heads, size, dim = k_pool.shape
        vdim, dev = v_pool.shape[4], k_pool.device
        if table.dim() != 2:
            raise ValueError("the table is [slots, blocks per slot]")
        _ints("table", table, table.numel())
        for name, t in (("v_pool", v_pool), ("table", table)):
            if t.device != dev:
                raise ValueError(f"{name} is on {t.device}, k_pool on {dev}")
        for name, t, count in (("k_scale", k_scale, blocks * layers * heads), ("v_scale", v_scale, blocks * layers * heads),
                               ("k_open", k_open, table.shape[0] * layers * heads * size * dim), ("v_open", v_open, table.shape[0] * layers * heads * size * vdim)):
            if t is not None:
                _floats(name, t, count, dev)
        self.k_pool, self.v_pool, self.k_scale, self.v_scale, self.k_open, self.v_open, self.table = k_pool, v_pool, k_scale, v_scale, k_open, v_open, table
        self.device, self.kw, self.vw = dev, heads * dim, heads * vdim
        at = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        self.c = Kv8Struct(at(k_pool), at(v_pool), at(k_scale), at(v_scale), at(k_open), at(v_open), at(table), table.shape[1], size, blocks, layers, heads, dim, vdim,
                           FORMATS[k_pool.dtype])
        self.ref, self.lib = C.byref(self.c), lib()

    @classmethod
    def empty(cls, *, blocks: int, layers: int, kv_heads: int, block_size: int, dim: int, vdim: int | None = None, slots: int, table_stride: int,
              dtype=torch.int8, device="cuda"):
        vdim = dim if vdim is None else vdim
        codes = lambda w: torch.zeros(blocks, layers, kv_heads, block_size, w, dtype=torch.int8, device=device).view(dtype)  # noqa: E731
        scale = lambda: torch.zeros(blocks, layers, kv_heads, device=device)  # noqa: E731
        rows = lambda w: torch.zeros(slots, layers, kv_heads, block_size, w, device=device)  # noqa: E731
        return cls(codes(dim), codes(vdim), scale(), scale(), rows(dim), rows(vdim), torch.zeros(slots, table_stride, dtype=torch.int32, device=device))

    def _stream(self, rows):
        if rows.device != self.device:
            raise ValueError(f"the rows are described on {rows.device}, the cache is on {self.device}")
        if rows.slots is not None and (rows.slots[0] < 0 or rows.slots[1] >= self.table.shape[0]):
            raise ValueError(f"slots {rows.slots[0]} .. {rows.slots[1]} of a cache of {self.table.shape[0]}")
        if torch.cuda.current_device() != self.device.index:
            raise ValueError(f"the cache is on {self.device}, the current device is cuda:{torch.cuda.current_device()}")
        return torch.cuda.current_stream().cuda_stream

    def _rows(self, name, t, n, width, dtypes):
        if t.device != self.device or t.dtype not in dtypes or t.dim() != 2 or t.shape[0] != n or t.shape[1] != width or (n and t.stride(1) != 1) or (n > 1 and t.stride(0) < width):
            raise ValueError(f"{name}: [{n}, {width}] on {self.device} of {' or '.join(str(d) for d in dtypes)} with neighbouring columns is needed, "
                             f"got {tuple(t.shape)} {t.dtype} on {t.device}, strides {t.stride()}")
        return t.data_ptr(), t.stride(0) if n > 1 else max(width, t.stride(0))

    def write(self, rows: Rows, k, v, layer: int = 0) -> None:
        """Rows enter the cache (tha_hyb_kv8_write): k [rows, kv heads * dim], v [rows, kv heads * vdim] in fp32 or bf16, rows any pitch apart."""
        stream = self._stream(rows)
        if rows.slots is not None and not rows.slots[2]:
            raise ValueError("a step writes at most one portion of a slot")
        kp, ldk = self._rows("k", k, rows.n, self.kw, DTYPES)
        vp, ldv = self._rows("v", v, rows.n, self.vw, (k.dtype,))
        self.lib.check(self.lib.c.tha_hyb_kv8_write(stream, DTYPES[k.dtype], rows.ref, self.ref, layer, kp, ldk, vp, ldv), "tha_hyb_kv8_write")

    def read(self, rows: Rows, layer: int = 0, dtype=torch.float32, k_out=None, v_out=None):
        """The values of cached rows (tha_hyb_kv8_read) as (k, v); into k_out, v_out where given."""
        stream = self._stream(rows)
        if k_out is None:
            k_out = torch.empty(rows.n, self.kw, dtype=dtype, device=self.device)
        if v_out is None:
            v_out = torch.empty(rows.n, self.vw, dtype=dtype, device=self.device)
        kp, ldk = self._rows("k_out", k_out, rows.n, self.kw, DTYPES)
        vp, ldv = self._rows("v_out", v_out, rows.n, self.vw, (k_out.dtype,))
        self.lib.check(self.lib.c.tha_hyb_kv8_read(stream, DTYPES[k_out.dtype], rows.ref, self.ref, layer, kp, ldk, vp, ldv), "tha_hyb_kv8_read")
        return k_out, v_out

    def attend(self, attn: Attention, rows: Rows, q, layer: int = 0, dtype=torch.float32, out=None, proj=None):
        """Attention of every row over its visible keys (tha_hyb_kv8_attn): q fp32 [rows, heads * dim] -> [rows, heads * vdim] of `dtype`.  proj: what head_gate reads."""
        stream = self._stream(rows)
        a = attn.c
        if attn.device is not None and attn.device != self.device:
            raise ValueError(f"the attention's tensors are on {attn.device}, the cache is on {self.device}")
        if layer != a.cache_layer:
            a.cache_layer = layer
        self._rows("q", q, rows.n, a.heads * a.dim, (torch.float32,))
        if not q.is_contiguous():
            raise ValueError("q has rows without gaps")
        if out is None:
            out = torch.empty(rows.n, a.heads * a.vdim, dtype=dtype, device=self.device)
        else:
            self._rows("out", out, rows.n, a.heads * a.vdim, DTYPES)
            if not out.is_contiguous():
                raise ValueError("out has rows without gaps")
        gate, ldg = None, 0
        if a.head_gate:
            if proj is None or proj.dim() != 2 or a.o_g < 0 or a.o_g + a.heads > proj.shape[1]:
                raise ValueError("head_gate reads its columns from proj [rows, columns]")
            gate, ldg = self._rows("proj", proj, rows.n, proj.shape[1], (torch.float32,))
        c = self.lib.c
        need = c.tha_hyb_kv8_attn_scratch(DTYPES[out.dtype], attn.ref, rows.ref, self.ref)
        scratch = torch.empty(need, dtype=torch.float32, device=self.device) if need else None
        self.lib.check(c.tha_hyb_kv8_attn(stream, DTYPES[out.dtype], attn.ref, rows.ref, self.ref, q.data_ptr(), out.data_ptr(), scratch.data_ptr() if need else None, need,
                                          gate, ldg), "tha_hyb_kv8_attn")
        return out
