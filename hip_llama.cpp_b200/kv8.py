"""Python binding of the key/value cache in 8 bits (tha_kv8_t and tha_hyb_kv8_* in include/tha_hybrid.h).

    cache = Kv8Cache.empty(blocks=512, layers=2, kv_heads=8, block_size=16, dim=128, slots=4, table_stride=64)
    cache.table.copy_(...)                                       # [slots, table_stride] block ids, the caller's to hand out
    rows = Rows.of([(0, 0, 300), (2, 17, 1)])                    # slot 0: positions 0 .. 299, slot 2: position 17
    cache.write(rows, k, v, layer=0)                             # k [301, 8 * 128]: rows or columns of a wider product
    out = cache.attend(Attention(32, 8, 128, scale=128 ** -0.5), rows, q, layer=0)   # [301, 32 * 128]
    k, v = cache.read(rows, layer=0)                             # the values that the codes stand for

Calls go to the current stream of the cache's device, which has to be the current device, and do not wait for it; Rows.of copies from pageable host memory, check_error waits.  Results and
scratch are allocated by torch on that stream, so that calls on several streams, from several threads, and captured ones, share nothing; a cache is written by one stream at a time.
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
                                  ("table_stride block_size n_blocks n_cache_layers kv_heads dim vdim format", I), ("open_end", P)])
STRUCTS = (RowsStruct, AttnStruct, Kv8Struct)

# the number of the current stream of a device; the public call makes an object around it first, 3.3 us
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)
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
    fp32 on the device.  head_gate: sigmoid of column gate_column + h of `proj` scales head h's result.  fp32_scores: q and the
    softmax weights keep 22 bits in long portions with bf16 results too, as they do everywhere else."""

    def __init__(self, heads: int, kv_heads: int, dim: int, vdim: int | None = None, *, scale: float, chunk: int = 0, window: int = 0, keep_first: int = 0, sink=None,
                 head_scale=None, softcap: float = 0.0, rel=None, head_gate: bool = False, gate_column: int = 0, fp32_scores: bool = False):
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
        vdim = dim if vdim is None else vdim
        at = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        self.c = AttnStruct(heads=heads, kv_heads=kv_heads, dim=dim, vdim=vdim, rot=-1, scale=scale, chunk=chunk, window=window, keep_first=keep_first, sink=at(sink),
                            head_scale=at(head_scale), softcap=softcap, rel=at(rel), rel_n=0 if rel is None else rel.shape[1], head_gate=int(head_gate), o_g=gate_column,
                            fp32_scores=int(fp32_scores))
        self.ref = C.byref(self.c)
        self.heads, self.q_width, self.out_width, self.gate = heads, heads * dim, heads * vdim, gate_column if head_gate else None
        self._of = {}

    def of(self, layer: int):
        """The struct `c` with this cache layer in it: one for each layer, written before anyone sees it, because other threads may be in calls with theirs."""
        now, (was, at) = bytes(self.c), self._of.get(layer, (None, None))
        if was != now:
            c = AttnStruct.from_buffer_copy(self.c)
            c.cache_layer, at = layer, C.byref(c)               # a reference keeps its struct
            self._of[layer] = now, at
        return at


class Kv8Cache:
    """Pools of codes [blocks, layers, kv heads, block size, channels] (int8 or float8_e4m3fn), their scales [blocks, layers, kv heads], the fp32 rows of every slot's last
    block [slots, layers, kv heads, block size, channels] and the block table [slots, blocks per slot] int32.  k_open, v_open None: a cache that is only read.
    open_end [slots, layers, kv heads, 2] int32, at first -1: with it a slot may be written again from any position, across a border of blocks too; `empty` makes one.  It says behind which
    position the rows of k_open, v_open end: a host that fills those sets it, or -1."""

    def __init__(self, k_pool, v_pool, k_scale, v_scale, k_open, v_open, table, open_end=None):
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
        if open_end is not None:
            _ints("open_end", open_end, 2 * table.shape[0] * layers * heads)
            if open_end.device != dev:
                raise ValueError(f"open_end is on {open_end.device}, k_pool on {dev}")
        self.k_pool, self.v_pool, self.k_scale, self.v_scale, self.k_open, self.v_open, self.table = k_pool, v_pool, k_scale, v_scale, k_open, v_open, table
        self.open_end = open_end
        self.device, self.kw, self.vw = dev, heads * dim, heads * vdim
        at = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        self.c = Kv8Struct(at(k_pool), at(v_pool), at(k_scale), at(v_scale), at(k_open), at(v_open), at(table), table.shape[1], size, blocks, layers, heads, dim, vdim,
                           FORMATS[k_pool.dtype], at(open_end))
        self.ref, self.lib, self.slots = C.byref(self.c), lib(), table.shape[0]
        self.calls = self.lib.c

    @classmethod
    def empty(cls, *, blocks: int, layers: int, kv_heads: int, block_size: int, dim: int, vdim: int | None = None, slots: int, table_stride: int,
              dtype=torch.int8, device="cuda"):
        vdim = dim if vdim is None else vdim
        codes = lambda w: torch.zeros(blocks, layers, kv_heads, block_size, w, dtype=torch.int8, device=device).view(dtype)  # noqa: E731
        scale = lambda: torch.zeros(blocks, layers, kv_heads, device=device)  # noqa: E731
        rows = lambda w: torch.zeros(slots, layers, kv_heads, block_size, w, device=device)  # noqa: E731
        return cls(codes(dim), codes(vdim), scale(), scale(), rows(dim), rows(vdim), torch.zeros(slots, table_stride, dtype=torch.int32, device=device),
                   torch.full((slots, layers, kv_heads, 2), -1, dtype=torch.int32, device=device))

    def _stream(self, rows):
        if rows.device != self.device:
            raise ValueError(f"the rows are described on {rows.device}, the cache is on {self.device}")
        if rows.slots is not None and (rows.slots[0] < 0 or rows.slots[1] >= self.slots):
            raise ValueError(f"slots {rows.slots[0]} .. {rows.slots[1]} of a cache of {self.slots}")
        if torch.cuda.current_device() != self.device.index:
            raise ValueError(f"the cache is on {self.device}, the current device is cuda:{torch.cuda.current_device()}")
        return _raw_stream(self.device.index)

    def _pitch(self, name, t, n, width, dtypes):
        """The row pitch of t [n, width], whose columns are neighbours."""
        s = t.stride()
        if t.shape != (n, width) or t.dtype not in dtypes or t.device != self.device or (n and s[1] != 1) or (n > 1 and s[0] < width):
            raise ValueError(f"{name}: [{n}, {width}] on {self.device} of {' or '.join(str(d) for d in dtypes)} with neighbouring columns is needed, "
                             f"got {tuple(t.shape)} {t.dtype} on {t.device}, strides {s}")
        return s[0] if n > 1 else max(width, s[0])

    def check_error(self) -> None:
        """Waits for the current stream; raises if a kernel on the device gave up on a barrier since the last such question (attend's rows concerned are NaN then)."""
        if self.device.type == "cuda":
            torch.cuda.current_stream(self.device).synchronize()
        if self.calls.tha_gemm_check_error():
            raise cabi.ThaError("a kernel gave up on a barrier of its own")

    def _check(self, status, name):
        if status:
            self.lib.check(status, name)

    def write(self, rows: Rows, k, v, layer: int = 0) -> None:
        """Rows enter the cache (tha_hyb_kv8_write): k [rows, kv heads * dim], v [rows, kv heads * vdim] in fp32 or bf16, rows any pitch apart."""
        stream = self._stream(rows)
        if rows.slots is not None and not rows.slots[2]:
            raise ValueError("a step writes at most one portion of a slot")
        kind = k.dtype
        ldk, ldv = self._pitch("k", k, rows.n, self.kw, DTYPES), self._pitch("v", v, rows.n, self.vw, (kind,))
        self._check(self.calls.tha_hyb_kv8_write(stream, DTYPES[kind], rows.ref, self.ref, layer, k.data_ptr(), ldk, v.data_ptr(), ldv), "tha_hyb_kv8_write")

    def read(self, rows: Rows, layer: int = 0, dtype=torch.float32, k_out=None, v_out=None):
        """The values of cached rows (tha_hyb_kv8_read) as (k, v); into k_out, v_out where given."""
        stream, n, ldk, ldv = self._stream(rows), rows.n, self.kw, self.vw
        if k_out is not None:
            ldk, dtype = self._pitch("k_out", k_out, n, ldk, DTYPES), k_out.dtype
        if v_out is not None:
            dtype = dtype if k_out is not None else v_out.dtype
            ldv = self._pitch("v_out", v_out, n, ldv, (dtype,))
        if dtype not in DTYPES:
            raise ValueError(f"values are read as float32 or bfloat16, not {dtype}")
        if k_out is None:
            k_out = torch.empty((n, ldk), dtype=dtype, device=self.device)
        if v_out is None:
            v_out = torch.empty((n, ldv), dtype=dtype, device=self.device)
        self._check(self.calls.tha_hyb_kv8_read(stream, DTYPES[dtype], rows.ref, self.ref, layer, k_out.data_ptr(), ldk, v_out.data_ptr(), ldv), "tha_hyb_kv8_read")
        return k_out, v_out

    def attend(self, attn: Attention, rows: Rows, q, layer: int = 0, dtype=torch.float32, out=None, proj=None):
        """Attention of every row over its visible keys (tha_hyb_kv8_attn): q fp32 [rows, heads * dim] -> [rows, heads * vdim] of `dtype`.  proj: what head_gate reads."""
        stream, n = self._stream(rows), rows.n
        if attn.device is not None and attn.device != self.device:
            raise ValueError(f"the attention's tensors are on {attn.device}, the cache is on {self.device}")
        of = attn.of(layer)
        if q.shape != (n, attn.q_width) or q.dtype != torch.float32 or q.device != self.device or not q.is_contiguous():
            raise ValueError(f"q: contiguous float32 [{n}, {attn.q_width}] on {self.device} is needed, got {tuple(q.shape)} {q.dtype} on {q.device}, strides {q.stride()}")
        if out is None:
            if dtype not in DTYPES:
                raise ValueError(f"results are float32 or bfloat16, not {dtype}")
            out = torch.empty((n, attn.out_width), dtype=dtype, device=self.device)
        elif out.shape != (n, attn.out_width) or out.dtype not in DTYPES or out.device != self.device or not out.is_contiguous():
            raise ValueError(f"out: contiguous [{n}, {attn.out_width}] float32 or bfloat16 on {self.device} is needed, got {tuple(out.shape)} {out.dtype} on {out.device}")
        gate, ldg = None, 0
        if attn.gate is not None:
            if proj is None or proj.dim() != 2 or attn.gate < 0 or attn.gate + attn.heads > proj.shape[1]:
                raise ValueError("head_gate reads its columns from proj [rows, columns]")
            gate, ldg = proj.data_ptr(), self._pitch("proj", proj, n, proj.shape[1], (torch.float32,))
        kind, room = DTYPES[out.dtype], None
        need = self.calls.tha_hyb_kv8_attn_scratch(kind, of, rows.ref, self.ref)
        if need:
            scratch = torch.empty(need, dtype=torch.float32, device=self.device)
            room = scratch.data_ptr()
        self._check(self.calls.tha_hyb_kv8_attn(stream, kind, of, rows.ref, self.ref, q.data_ptr(), out.data_ptr(), room, need, gate, ldg), "tha_hyb_kv8_attn")
        return out
