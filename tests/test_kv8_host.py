"""The cache in 8 bits without a GPU: the binding's structs against the header, the oracle's roundings against torch's, and what the calls refuse (before any launch)."""
import ctypes as C
import os
import re
import subprocess

import numpy as np
import pytest
import torch

import kv8_oracle as O
from pkgload import load_pkg

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
K = load_pkg("kv8")
A = 1 << 20                                                       # an aligned address that no refused call looks at


def test_structs_match_the_header(tmp_path):
    src, want = ['#include <stdio.h>', '#include "tha_hybrid.h"', "int main(void) {"], []
    for s in K.STRUCTS:
        src.append('printf("%%zu\\n", sizeof(%s));' % s.__name__)
        want.append(C.sizeof(s))
        for f, _ in s._fields_:
            src.append('printf("%%zu\\n", offsetof(%s, %s));' % (s.__name__, f))
            want.append(getattr(s, f).offset)
    (tmp_path / "a.c").write_text("\n".join(src + ["return 0; }"]))
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), "-o", str(tmp_path / "a"), str(tmp_path / "a.c")])
    assert [int(x) for x in subprocess.check_output([str(tmp_path / "a")]).split()] == want


def test_every_declared_call_is_exported():
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "tha_hybrid.h")).read(), flags=re.S)
    names = set(re.findall(r"\b(tha_hyb_kv8_[a-z0-9_]+)\s*\(", text))
    assert names == {"tha_hyb_kv8_write", "tha_hyb_kv8_read", "tha_hyb_kv8_attn", "tha_hyb_kv8_attn_scratch"}
    assert all(hasattr(K.lib().c, n) for n in names)


def test_the_oracle_rounds_as_the_formats_do():
    y = np.concatenate([np.linspace(-448, 448, 20001), O.levels("e4m3"), -O.levels("e4m3"), (O.levels("e4m3")[1:] + O.levels("e4m3")[:-1]) / 2])
    got = torch.from_numpy(y).float().to(torch.float8_e4m3fn).float().numpy()
    assert np.array_equal(O.nearest(y.astype(np.float32).astype(np.float64), "e4m3"), got.astype(np.float64))
    y = np.concatenate([np.linspace(-127, 127, 5001), np.arange(-126.5, 127, 1)])
    assert np.array_equal(O.nearest(y, "int8"), np.rint(y))
    codes = np.arange(256, dtype=np.uint8)
    assert np.array_equal(O.numbers(codes, "int8"), codes.view(np.int8).astype(np.float64))
    of = torch.from_numpy(codes).view(torch.float8_e4m3fn).float().numpy().astype(np.float64)
    assert np.array_equal(O.numbers(codes, "e4m3"), of, equal_nan=True)


def rows(**more):
    return K.RowsStruct(**{**dict(n_rows=3, n_seqs=2, pos=A, row_seq=A, seq_first=A, seq_slot=A, max_seq_rows=2, max_pos=40), **more})


def cache(**more):
    return K.Kv8Struct(**{**dict(k_pool=A, v_pool=A, k_scale=A, v_scale=A, k_open=A, v_open=A, table=A, table_stride=4, block_size=16, n_blocks=9, n_cache_layers=2,
                                 kv_heads=2, dim=64, vdim=64, format=0), **more})


def attn(**more):
    return K.AttnStruct(**{**dict(heads=4, kv_heads=2, dim=64, vdim=64, scale=0.125), **more})


REFUSED_ROWS = [dict(pos=None), dict(row_seq=None), dict(seq_first=None), dict(seq_slot=None), dict(n_seqs=0), dict(n_seqs=4), dict(max_seq_rows=0), dict(max_seq_rows=4),
                dict(max_pos=64)]
REFUSED_CACHE = [dict(k_pool=None), dict(v_pool=None), dict(k_scale=None), dict(v_scale=None), dict(table=None), dict(format=2), dict(format=-1), dict(block_size=8),
                 dict(block_size=48), dict(block_size=256), dict(dim=0), dict(dim=24), dict(dim=144), dict(vdim=8), dict(vdim=136), dict(kv_heads=0), dict(kv_heads=65536),
                 dict(n_cache_layers=0), dict(n_cache_layers=1), dict(n_blocks=0), dict(table_stride=0), dict(table_stride=2), dict(k_pool=A + 8), dict(v_pool=A + 1)]


def status(call, *args):
    got = call(*args)
    return got, K.lib().c.tha_last_error().decode()


def calls(r, c, layer=1, dtype=1):
    """(name, status, text) of the three calls with these descriptions."""
    f = K.lib().c
    return [("write",) + status(f.tha_hyb_kv8_write, None, dtype, r, c, layer, A, 128, A, 128),
            ("read",) + status(f.tha_hyb_kv8_read, None, dtype, r, c, layer, A, 128, A, 128),
            ("attn",) + status(f.tha_hyb_kv8_attn, None, dtype, attn(cache_layer=layer, kv_heads=c.kv_heads, heads=2 * c.kv_heads, dim=c.dim, vdim=c.vdim), r, c, A, A, None, 0,
                               None, 0)]


@pytest.mark.parametrize("bad", REFUSED_ROWS, ids=str)
def test_rows_that_are_refused(bad):
    for name, got, text in calls(rows(**bad), cache()):
        assert got == 2 and "tha_hyb_kv8_" + name in text


@pytest.mark.parametrize("bad", REFUSED_CACHE, ids=str)
def test_caches_that_are_refused(bad):
    for name, got, text in calls(rows(), cache(**bad)):
        assert got == 2 and "tha_hyb_kv8_" + name in text


def test_layers_and_types_that_are_refused():
    for r, c, layer, dtype in ((rows(), cache(), 2, 1), (rows(), cache(), -1, 1), (rows(), cache(), 0, 2), (rows(), cache(), 0, -1)):
        assert all(got == 2 for _, got, _ in calls(r, c, layer, dtype))


def test_operands_that_are_refused():
    f, r, c = K.lib().c, rows(), cache()
    for k, ldk, v, ldv in ((None, 128, A, 128), (A, 128, None, 128), (A, 127, A, 128), (A, 128, A, 64)):
        assert f.tha_hyb_kv8_write(None, 1, r, c, 0, k, ldk, v, ldv) == 2
    for more in (dict(k_open=None), dict(v_open=None), dict(k_open=A + 4), dict(v_open=A + 8)):
        assert f.tha_hyb_kv8_write(None, 1, r, cache(**more), 0, A, 128, A, 128) == 2
    for k, ldk, v, ldv in ((A, 127, A, 128), (A, 128, A, 100), (A, 1, None, 0)):
        assert f.tha_hyb_kv8_read(None, 1, r, c, 0, k, ldk, v, ldv) == 2
    for q, out, scratch in ((None, A, None), (A, None, None), (A + 4, A, None), (A, A, A + 8)):
        assert f.tha_hyb_kv8_attn(None, 1, attn(), r, c, q, out, scratch, 1 << 20, None, 0) == 2


@pytest.mark.parametrize("bad,code", [(dict(heads=3), 2), (dict(heads=0), 2), (dict(kv_heads=4), 2), (dict(dim=32), 2), (dict(vdim=32), 2), (dict(window=-1), 2),
                                      (dict(keep_first=-1), 2), (dict(chunk=-1), 2), (dict(rel=A), 2), (dict(cache_layer=2), 2), (dict(values_in_keys=1), 7),
                                      (dict(v_share=2), 7), (dict(diff=1), 7)], ids=str)
def test_attention_that_is_refused(bad, code):
    f = K.lib().c
    assert f.tha_hyb_kv8_attn(None, 1, attn(**bad), rows(), cache(), A, A, None, 0, None, 0) == code
    assert f.tha_hyb_kv8_attn_scratch(1, attn(**bad), rows(), cache()) == 0


def test_a_step_of_prompts_is_not_cut_for_the_short_portions_it_might_hold():
    """Room for the visible keys as fp16 and nothing for partial results: a step of prompts would pass all of its rows once more."""
    big = dict(kv_heads=32, dim=128, vdim=128)
    r, c = rows(n_rows=2825, max_seq_rows=2048, max_pos=2047), cache(**big, table_stride=128, n_blocks=257)
    a = attn(heads=32, **big)
    parts = 2 * (2048 // 32 + 2)                                  # of 32 keys, K and V, fp16; one more percent for their scales
    need = 4 * K.lib().c.tha_hyb_kv8_attn_scratch(1, a, r, c)
    assert 2 * 2048 * 32 * 2 * 128 * 2 <= need <= parts * 32 * 32 * 2 * 128 * 2 * 1.01


def test_no_rows_are_no_work():
    f, r = K.lib().c, rows(n_rows=0)
    assert f.tha_hyb_kv8_write(None, 1, r, cache(), 0, A, 128, A, 128) == 0
    assert f.tha_hyb_kv8_read(None, 1, r, cache(), 0, A, 128, A, 128) == 0
    assert f.tha_hyb_kv8_attn(None, 1, attn(), r, cache(), A, A, None, 0, None, 0) == 0
    assert f.tha_hyb_kv8_read(None, 1, rows(), cache(), 0, None, 0, None, 0) == 0


def small(device="cpu", **more):
    return K.Kv8Cache.empty(**{**dict(blocks=4, layers=1, kv_heads=2, block_size=16, dim=32, slots=2, table_stride=2, device=device), **more})


def test_the_binding_refuses_what_the_library_cannot_see():
    z = torch.zeros
    pool, scale, rows_, table = z(4, 1, 2, 16, 32, dtype=torch.int8), z(4, 1, 2), z(2, 1, 2, 16, 32), z(2, 2, dtype=torch.int32)
    good = [pool, pool.clone(), scale, scale.clone(), rows_, rows_.clone(), table]
    K.Kv8Cache(*good)
    K.Kv8Cache(*good[:4], None, None, table)
    for i, bad in ((0, pool.float()), (1, pool.view(torch.float8_e4m3fn)), (1, pool[:3]), (0, pool.transpose(2, 3)), (2, scale[:3]), (3, scale.double()), (4, None),
                   (4, rows_[:1]), (5, rows_.half()), (6, table.long()), (6, table[0]), (6, z(2, 4, dtype=torch.int32)[:, ::2])):
        with pytest.raises(ValueError):
            K.Kv8Cache(*good[:i], bad, *good[i + 1:])
    with pytest.raises(ValueError):
        K.Rows.of([], "cpu")
    for portion in ((0, 0, 0), (0, -1, 2)):
        with pytest.raises(ValueError):
            K.Rows.of([portion], "cpu")
    ints = z(3, dtype=torch.int32)
    with pytest.raises(ValueError):
        K.Rows(ints, ints[:2], ints, ints[:2], 2, 0)
    with pytest.raises(ValueError):
        K.Rows(ints, ints, ints[:2], ints[:2], 2, 0)
    with pytest.raises(ValueError):
        K.Attention(4, 2, 32, scale=1.0, sink=z(3))
    with pytest.raises(ValueError):
        K.Attention(4, 2, 32, scale=1.0, rel=z(2, 8))
    r = K.Rows.of([(0, 0, 3), (1, 5, 1), (1, -1, 1)], "cpu")
    assert r.n == 5 and r.c.max_seq_rows == 3 and r.c.max_pos == 5 and r.slots == (0, 1, True)
    assert not K.Rows.of([(0, 0, 3), (0, 5, 1)], "cpu").slots[2]


@pytest.mark.parametrize("beside", [0, 1, 15, 31, 63, 127])
@pytest.mark.parametrize("most,rows_", [(2047, 1024), (4095, 1024), (8191, 512)])
@pytest.mark.parametrize("dtype", [0, 1])
def test_a_prompt_beside_decoded_rows_keeps_its_form(beside, most, rows_, dtype):
    """Room for the visible keys as fp16 goes by the sequences that may be long, not by all of the step's: with that for all, 31 rows at up to 2048 were too much, and none was asked for."""
    big = dict(kv_heads=32, dim=128, vdim=128)
    c = cache(**big, table_stride=512, n_blocks=9000)
    r = rows(n_rows=rows_ + beside, n_seqs=1 + beside, max_seq_rows=rows_, max_pos=most)
    need = 4 * K.lib().c.tha_hyb_kv8_attn_scratch(dtype, attn(heads=32, **big), r, c)
    one = 2 * (most + 1) * 32 * 2 * 128                           # of the prompt's context in fp16
    assert one <= need < (1 << 30) + (64 << 20)
    # Portions of up to 29 rows are short ones: four blocks of eight of them take 4 * 32 * 0.72 us / 444 / 32 = 6.5 ns a key, staged ones at least 32 * 0.145 ns, and 32 * 1.0 us / 148 / 64
    # for their tiles, 8.0 ns.  Portions of 30 rows or more are at most so many of the step.
    assert need <= max(1, min(1 + beside, (rows_ + beside) // 30)) * one * 1.1 + (64 << 20)


def test_portions_that_find_no_room_are_the_shorter_ones():
    """With more sequences that may be long than find room, the long ones keep the form; a context that finds no room alone does not have it."""
    big = dict(kv_heads=32, dim=128, vdim=128)
    for most, n_seqs, n_rows, there in ((32767, 40, 4000, True), (32767, 1, 2048, True), (131071, 1, 2048, False)):
        r = rows(n_rows=n_rows, n_seqs=n_seqs, max_seq_rows=2048, max_pos=most)
        need = 4 * K.lib().c.tha_hyb_kv8_attn_scratch(0, attn(heads=32, **big), r, cache(**big, table_stride=8192, n_blocks=9000))
        assert (need >= 2 * most * 32 * 2 * 128) == there and need < (1 << 30) + (128 << 20)


FASTER = [  # heads, kv heads, channels, fp32 results, sequences, first position, rows; us as short portions, us as long ones
    (16, 4, 128, 0, 1, 0, 256, 23.6, 19.5), (32, 32, 128, 0, 4, 0, 64, 29.7, 17.4), (32, 8, 128, 0, 16, 0, 16, 27.6, 17.4), (12, 12, 64, 0, 16, 0, 64, 27.6, 17.4), (64, 8, 64, 0, 1, 0, 128, 22.5, 15.4),
    (32, 32, 128, 1, 4, 0, 64, 29.7, 21.5), (32, 8, 128, 1, 1, 1000, 64, 27.6, 48.1), (16, 4, 128, 1, 1, 1000, 128, 29.7, 48.1), (8, 1, 128, 1, 1, 16000, 32, 44.0, 60.4),
    (8, 1, 128, 1, 16, 16000, 128, 1422.3, 312.4), (32, 32, 128, 0, 1, 4000, 128, 140.2, 60.4), (16, 4, 128, 0, 1, 4000, 64, 46.1, 33.8)]


@pytest.mark.parametrize("case", FASTER, ids=str)
def test_portions_take_the_form_that_was_measured_to_be_faster(case):
    """... by a quarter or more.  Staged keys are most of the scratch that the form of long ones asks for."""
    heads, kv_heads, dim, dtype, seqs, p, n, short, long = case
    assert max(short, long) >= 1.2 * min(short, long)
    shape = dict(kv_heads=kv_heads, dim=dim, vdim=dim)
    r = rows(n_rows=seqs * n, n_seqs=seqs, max_seq_rows=n, max_pos=p + n - 1)
    floats = K.lib().c.tha_hyb_kv8_attn_scratch(dtype, attn(heads=heads, **shape), r, cache(**shape, table_stride=2048, n_blocks=40000))
    assert (floats >= seqs * (p + n) * kv_heads * dim) == (long < short)
