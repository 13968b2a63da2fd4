"""What the calls over microscaled numbers refuse, and the layout that their binding makes: no GPU."""
import ctypes as C
import os
import re
import subprocess

import numpy as np
import pytest
import torch

import mx_oracle as O
from pkgload import load_pkg

M = load_pkg("mx")
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ROOM = torch.zeros(1 << 16, dtype=torch.uint8)
BASE = (ROOM.data_ptr() + 511) // 512 * 512


def struct(rows=4, cols=96, format="e4m3", codes=0, scales=1024, **more):
    s = M.MxStruct(BASE + codes, BASE + scales, rows, cols, M.FORMATS.get(format, 7))
    for k, v in more.items():
        setattr(s, k, v)
    return s


def refused(name, *args):
    lib = M.lib()
    assert getattr(lib.c, name)(None, *args) == 2, name
    text = lib.c.tha_last_error().decode()
    assert name in text
    return text


def test_struct_matches_the_header(tmp_path):
    (tmp_path / "a.c").write_text('#include <stdio.h>\n#include "tha_hybrid.h"\nint main(void) { printf("%zu %zu %zu %zu %zu %zu\\n", sizeof(tha_mx_t), offsetof(tha_mx_t, codes), '
                                  'offsetof(tha_mx_t, scales), offsetof(tha_mx_t, rows), offsetof(tha_mx_t, cols), offsetof(tha_mx_t, format)); return 0; }')
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), "-o", str(tmp_path / "a"), str(tmp_path / "a.c")])
    S = M.MxStruct
    assert [int(x) for x in subprocess.check_output([str(tmp_path / "a")]).split()] == [C.sizeof(S), S.codes.offset, S.scales.offset, S.rows.offset, S.cols.offset, S.format.offset]


@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 128), (128, 129), (129, 1000), (1000, 32)])
@pytest.mark.parametrize("fmt", ["e2m1", "e4m3"])
def test_sizes_and_layout(rows, cols, fmt):
    m, c = M.Mx.empty(rows, cols, fmt, "cpu"), M.lib().c
    assert c.tha_hyb_mx_codes_bytes(M.FORMATS[fmt], rows, cols) == m.codes.numel() and c.tha_hyb_mx_scales_bytes(rows, cols) == m.scales.numel()
    assert m.c.codes == m.codes.data_ptr() and m.c.scales == m.scales.data_ptr() and m.codes.data_ptr() % 32 == 0 and m.scales.data_ptr() % 16 == 0
    x = np.random.default_rng(rows).standard_normal((rows, cols))
    v, byte, code = O.quantise(x, fmt)
    codes = torch.from_numpy(np.pad(code, ((0, 0), (0, cols % 2 if fmt == "e2m1" else 0))).astype(np.uint8))
    codes = codes[:, 0::2] | (codes[:, 1::2] << 4) if fmt == "e2m1" else codes.view(torch.float8_e4m3fn)
    m = M.Mx.of_rows(codes, torch.from_numpy(byte.astype(np.uint8)), cols)
    assert np.array_equal(O.values(m), v) and np.array_equal(O.scales_of(m)[:, :byte.shape[1]], byte) and not O.codes_of(m)[:, cols:].any()


def test_sizes_of_no_matrix():
    c = M.lib().c
    for f, r, k in ((2, 1, 1), (0, 0, 1), (0, 1, 0), (1, -1, 5), (1, 5, -1), (0, 1, 0x7fffffff)):
        assert c.tha_hyb_mx_codes_bytes(f, r, k) == 0
    assert c.tha_hyb_mx_scales_bytes(0, 5) == c.tha_hyb_mx_scales_bytes(5, 0) == 0


BAD = [dict(format="e5m2"), dict(cols=0), dict(cols=-3), dict(rows=-1), dict(codes=16), dict(scales=1032), dict(codes=-BASE), dict(scales=-BASE), dict(cols=(1 << 30) + 1), dict(rows=(1 << 30) + 1)]


@pytest.mark.parametrize("bad", BAD)
def test_matrices_that_are_none(bad):
    m, good, w = C.byref(struct(**bad)), C.byref(struct()), C.byref(struct(format="e2m1"))
    refused("tha_hyb_mx_quant", 1, BASE, 4096, m)
    refused("tha_hyb_mx_read", 1, m, BASE, 4096)
    refused("tha_hyb_mx_add_norm", 1, BASE, BASE, 4096, BASE, BASE, 0.0, 1e-5, m)
    refused("tha_hyb_mx_linear", 1, BASE, 4096, m, w)
    refused("tha_hyb_mx_linear", 1, BASE, 4096, good, m)
    refused("tha_hyb_mx_linear_act", 4, m, w, w, 0.0, 0.0, good)
    refused("tha_hyb_mx_linear_act", 4, good, m, w, 0.0, 0.0, good)
    refused("tha_hyb_mx_linear_act", 4, good, w, m, 0.0, 0.0, good)
    refused("tha_hyb_mx_linear_act", 4, good, w, w, 0.0, 0.0, m)


def test_arguments_that_do_not_fit():
    a, w, wide = C.byref(struct()), C.byref(struct(format="e2m1", rows=200)), C.byref(struct(format="e2m1", rows=200, cols=97))
    y = C.byref(struct(rows=4, cols=200))
    assert "NULL" in refused("tha_hyb_mx_quant", 1, None, 96, a) and "pitch" in refused("tha_hyb_mx_quant", 1, BASE, 95, a) and "dtype" in refused("tha_hyb_mx_quant", 2, BASE, 96, a)
    assert "NULL" in refused("tha_hyb_mx_read", 1, a, None, 96) and "pitch" in refused("tha_hyb_mx_read", 0, a, BASE, 95) and "dtype" in refused("tha_hyb_mx_read", -1, a, BASE, 96)
    for x, left, ldl, out, g in ((None, BASE, 96, BASE, BASE), (BASE, BASE, 96, None, BASE), (BASE, BASE, 96, BASE, None), (BASE, BASE, 95, BASE, BASE)):
        refused("tha_hyb_mx_add_norm", 1, x, left, ldl, out, g, 0.0, 1e-5, a)
    refused("tha_hyb_mx_add_norm", 3, BASE, BASE, 96, BASE, BASE, 0.0, 1e-5, a)
    assert "columns" in refused("tha_hyb_mx_linear", 1, BASE, 4096, a, wide) and "E2M1" in refused("tha_hyb_mx_linear", 1, BASE, 4096, a, a)
    assert "NULL" in refused("tha_hyb_mx_linear", 1, None, 4096, a, w) and "pitch" in refused("tha_hyb_mx_linear", 1, BASE, 199, a, w) and "dtype" in refused("tha_hyb_mx_linear", 5, BASE, 200, a, w)
    refused("tha_hyb_mx_linear", 1, BASE, 4096, None, w)
    assert "gate" in refused("tha_hyb_mx_linear_act", 4, a, None, w, 0.0, 0.0, y) and "gate" in refused("tha_hyb_mx_linear_act", 1, a, w, w, 0.0, 0.0, y)
    assert "activation" in refused("tha_hyb_mx_linear_act", 5, a, w, w, 0.0, 0.0, y) and "activation" in refused("tha_hyb_mx_linear_act", -1, a, w, w, 0.0, 0.0, y)
    assert "rows" in refused("tha_hyb_mx_linear_act", 4, a, C.byref(struct(format="e2m1", rows=199)), w, 0.0, 0.0, y)
    for r, c in ((5, 200), (4, 199)):
        refused("tha_hyb_mx_linear_act", 4, a, w, w, 0.0, 0.0, C.byref(struct(rows=r, cols=c)))


def test_the_binding_refuses():
    x = torch.zeros(4, 96)
    w = M.Mx.empty(200, 96, device="cpu")
    a = M.Mx.empty(4, 96, "e4m3", "cpu")
    bad = [lambda: M.quantise(x, "e5m2"), lambda: M.quantise(x[0]), lambda: M.quantise(x.half()), lambda: M.quantise(x.T), lambda: M.quantise(x, out=M.Mx.empty(4, 95, device="cpu")),
           lambda: a.read(torch.float16), lambda: a.read(out=torch.zeros(4, 95)), lambda: a.read(out=torch.zeros(96, 4).T),
           lambda: M.add_norm(x.bfloat16(), x, x[0], eps=1e-5), lambda: M.add_norm(x, x[:3], x[0], eps=1e-5), lambda: M.add_norm(x, x, x[0, :95], eps=1e-5),
           lambda: M.add_norm(x, x, x[0].double(), eps=1e-5), lambda: M.add_norm(torch.zeros(4, 99)[:, :96], x, x[0], eps=1e-5), lambda: M.add_norm(x, x, x[0], eps=1e-5, x_out=torch.zeros(3, 96)),
           lambda: M.linear(a, w, dtype=torch.int8), lambda: M.linear(a, w, out=torch.zeros(4, 199)),
           lambda: M.linear_act(a, None, w), lambda: M.linear_act(a, w, w, act="relu2"), lambda: M.linear_act(a, w, w, act="tanh"), lambda: M.linear_act(a, w, w, format="int8"),
           lambda: M.linear_act(a, w, w, out=M.Mx.empty(4, 199, "e4m3", "cpu")),
           lambda: M.Mx(torch.zeros(4, 128, dtype=torch.int8), a.scales, 4, 96), lambda: M.Mx(a.codes, a.scales[:-1], 4, 96), lambda: M.Mx(a.codes, a.scales, 4, 129),
           lambda: M.Mx(a.codes, a.scales, 5, 96), lambda: M.Mx(a.codes, a.scales, 4, 0), lambda: M.Mx(a.codes.T, a.scales, 128, 4),
           lambda: M.Mx.of_rows(a.codes, torch.zeros(4, 3, dtype=torch.uint8), 96), lambda: M.Mx.empty(4, 96, "int8", "cpu")]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was taken")


def test_devices(monkeypatch):
    x, w = torch.zeros(4, 96), torch.ones(96)
    m = M.Mx.empty(4, 96, "e4m3", "cpu")
    for call in (lambda: M.quantise(x), lambda: M.add_norm(x, None, w, eps=1e-5), lambda: m.read(), lambda: M.linear(m, M.Mx.empty(5, 96, device="cpu"))):
        with pytest.raises(ValueError, match="current device"):
            call()
    monkeypatch.setattr(M, "_current_device", lambda: 1)
    with pytest.raises(ValueError, match="current device"):
        M._stream(torch.device("cuda", 0))
    monkeypatch.setattr(M, "_raw_stream", lambda index: 100 + index)
    assert M._stream(torch.device("cuda", 1)) == 101


def test_room_is_one_piece():
    """The tensors over a matrix that a call made lie where the call wrote"""
    for rows, cols, fmt in ((3, 70, "e2m1"), (130, 300, "e4m3"), (0, 5, "e2m1")):
        m = M.Mx.empty(rows, cols, fmt, "cpu")
        again = M.Mx(m.codes, m.scales, rows, cols)
        assert rows == 0 or (again.c.codes, again.c.scales) == (m.c.codes, m.c.scales)
        assert again.format == fmt and m.codes is m.codes and m.scales is m.scales


def source(name, kernel):
    text = re.sub(r"//[^\n]*", "", open(os.path.join(os.path.dirname(M.__file__), "csrc", name)).read())
    text = text[text.index(kernel + "("):]
    return text[:text.index("\n}\n")]


def test_a_norm_whose_wait_gives_up_leaves_no_number():
    """No wait of the ring runs out in a sound pipeline, so this is read from its source: a thread that has given up waits and reads no more and has NaN for its values, which go into the row's sum,
    and so into root and codes, and into x_out; nothing more is asked for, and what is under way lands ahead of the block's end."""
    k = source("mx_rows.cu", "mx_add_norm_ring_kernel")
    rows = k[k.index("bool ok = true;"):]
    order = [rows.index(t) for t in ("ok = ok && tc_mbar_wait(&full[s]", "const float none = ok ? 0.f : __uint_as_float(0x7fc00000u);", "ok ? cols - col : 0, true, v[i], none);", "total = fma(", "__syncthreads();",
                                     "if (threadIdx.x == 0 && ok && row", "ask(s", "mr_store(x_out", "mr_norm_codes<FMT>", "if (threadIdx.x == 0 && abort_flag) {", "tc_drain(full, stages, asked);")]
    assert order == sorted(order) and rows.count("tc_mbar_wait") == rows.count("mr_store(x_out") == len(re.findall(r"\bask\(", rows)) == len(re.findall(r"\bok = ", rows)) - 1 == 1
    load = source("mx_rows.cu", "void mr_load")
    assert "float none = 0.f" in load and "v[i] = i < n ? p[i] : none;" in load


def test_lanes_without_a_weight_row_stay_with_their_warp():
    """Lanes may leave a store of results one by one; between it and whatever takes a warp as one (tcgen05.ld, barrier.cluster) stands a __syncwarp.  Read from the source, as lanes that leave early
    usually meet again."""
    stores = 0
    for kernel in ("mx_gemm_kernel", "mx_gemm_pair_kernel"):
        k = source("mx_gemm.cu", kernel)
        assert "mg_store_blocks" not in k
        for m in re.finditer(r"mg_store<READ>\([^;]*;", k):
            assert re.match(r"\s*__syncwarp\(\);", k[m.end():]), k[m.start():m.end() + 80]
            stores += 1
    assert stores == 3


def test_the_error_of_another_device(monkeypatch):
    """check_error asks about the device that it is given, current or not, and leaves the current one as it was"""
    import contextlib
    current, asked, waited = [0], [], []

    @contextlib.contextmanager
    def device(d):
        before, current[0] = current[0], torch.device(d).index if torch.device(d).index is not None else current[0]
        yield
        current[0] = before

    class Stream:
        def __init__(self, d):
            self.d = current[0] if d is None else torch.device(d).index

        def synchronize(self):
            waited.append(self.d)

    class Calls:
        def tha_gemm_check_error(self):
            asked.append(current[0])
            return current[0]

    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda d=None: Stream(d))
    monkeypatch.setattr(M, "_c", Calls())
    M.check_error("cuda:0")
    with pytest.raises(M.cabi.ThaError):
        M.check_error("cuda:1")
    M.check_error()
    assert asked == waited == [0, 1, 0] and current == [0]


def test_activations_that_take_numbers_are_given_them():
    """clamped without a limit would clamp at 0"""
    a, w = M.Mx.empty(4, 96, "e4m3", "cpu"), M.Mx.empty(200, 96, device="cpu")
    for act, gate in (("clamped", w), ("xielu", None)):
        for numbers in ({}, {"limit": 7.0}, {"alpha": 1.702}):
            with pytest.raises(ValueError, match="limit and alpha"):
                M.linear_act(a, gate, w, act=act, **numbers)
        with pytest.raises(ValueError, match="current device"):         # taken, but for where it is
            M.linear_act(a, gate, w, act=act, limit=7.0, alpha=1.702)
    for act, gate in (("silu", w), ("gelu", w), ("relu2", None)):
        with pytest.raises(ValueError, match="current device"):
            M.linear_act(a, gate, w, act=act)


def test_more_results_than_a_call_counts():
    """Refused under the call's own name, ahead of anything that is asked of a device"""
    rows, w = C.byref(struct(rows=1 << 30)), C.byref(struct(format="e2m1", rows=1 << 30))
    assert "too many" in refused("tha_hyb_mx_linear", 1, BASE, 1 << 30, rows, w)
    y = C.byref(struct(rows=1 << 30, cols=1 << 30))
    assert "too many" in refused("tha_hyb_mx_linear_act", 4, rows, w, w, 0.0, 0.0, y) and "too many" in refused("tha_hyb_mx_linear_act", 1, rows, None, w, 0.0, 0.0, y)


def test_eps_below_zero():
    a = C.byref(struct())
    for eps in (-1e-5, float("nan"), -float("inf")):
        assert "eps" in refused("tha_hyb_mx_add_norm", 1, BASE, BASE, 96, BASE, BASE, 0.0, eps, a)
