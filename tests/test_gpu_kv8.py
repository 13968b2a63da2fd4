"""The cache in 8 bits (csrc/kv8_rows.cu, csrc/kv8_attn.cu) against its definition in float64 (kv8_oracle.py).

Tolerances.  Codes, scales and kept rows are equal to the bit.  Values read back: code * scale rounded once (2^-24 of the value in fp32), bf16 once more (2^-8).
Attention in fp32, relative to the norm of the result, for q and keys of order one, scale dim^-1/2: a score is a sum of up to 128 products with sum |q k| scale of about 0.64 * 128^1/2 =
7, off by 2^-22 of that (q in two fp16) and 2^-23 (fp32 sums), 2.5e-6 if all errors agree; its rounding beside the maximum and the factor 2^15, |x| < 32, adds 2^-24 * 32 = 1.9e-6; the
weight 2^-22 (ex2) + 2^-22 (two fp16), the sums 2^-22: 0.7e-6.  Together 5.1e-6, and 6e-6 is asked for.  (Sums of the tensor cores are cut off, not rounded: 128 of them in a row, each
2^-24 of what is there, on the average half of it and of the end's value, are 128 * 2^-26 = 1.9e-6; they and the scores' errors do not agree.)  A bf16 result is off by half a step more, 2^-8 of each value."""
import numpy as np
import pytest
import torch

import kv8_oracle as O
from pkgload import load_pkg

pytestmark = pytest.mark.gpu
K = load_pkg("kv8")
DT = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
F32_TOL, BF16_STEP = 6e-6, 2.0 ** -8
LAYERS, LAYER = 3, 1


class Mirror:
    """A cache on the GPU, and what it should hold: every slot's rows, as they were written last."""

    def __init__(self, slots, longest, kv_heads, block, dim, vdim, fmt, seed=0, spare=3):
        self.fmt, self.B, self.H, self.dim, self.vdim = fmt, block, kv_heads, dim, vdim
        self.per = -(-longest // block)
        rng = np.random.default_rng(seed)
        self.rng, blocks = rng, slots * self.per + spare
        self.cache = K.Kv8Cache.empty(blocks=blocks, layers=LAYERS, kv_heads=kv_heads, block_size=block, dim=dim, vdim=vdim, slots=slots, table_stride=self.per, dtype=DT[fmt])
        self.table = rng.permutation(blocks)[:slots * self.per].reshape(slots, self.per).astype(np.int32)
        self.cache.table.copy_(torch.from_numpy(self.table))
        for t in (self.cache.k_pool, self.cache.v_pool):        # what a kernel must not touch keeps its bytes
            t.view(torch.int8).fill_(55)
        for t in (self.cache.k_scale, self.cache.v_scale, self.cache.k_open, self.cache.v_open):
            t.fill_(7.25)
        self.rows = [{"k": np.zeros((0, kv_heads, dim), np.float32), "v": np.zeros((0, kv_heads, vdim), np.float32)} for _ in range(slots)]
        self.touched = {}                                       # (slot, block) -> rows that were there when it was written last

    def write(self, portions, k, v, call=None):
        r = K.Rows.of(portions)
        (call or self.cache.write)(r, k, v, layer=LAYER)
        at = 0
        for slot, p, n in portions:
            for side, t in (("k", k), ("v", v)):
                new = t[at:at + n].float().cpu().numpy().reshape(n, self.H, -1)
                if p >= 0:
                    self.rows[slot][side] = np.concatenate([self.rows[slot][side][:p], new])
            at += n
            if p >= 0:
                for b in range(p // self.B, (p + n - 1) // self.B + 1):
                    self.touched[(slot, b)] = min(self.B, p + n - b * self.B)

    def expect(self, side, slot, b, count):
        """numbers [head, position, channel] and scales [head] of a block with `count` rows"""
        x = np.zeros((self.B, self.H, self.rows[slot][side].shape[2]), np.float32)
        x[:count] = self.rows[slot][side][b * self.B:b * self.B + count]
        got = [O.quantise(x[:, h], self.fmt) for h in range(self.H)]
        return np.stack([g[0] for g in got]), np.array([g[1] for g in got], np.float32)

    def check(self):
        c = self.cache
        for side, pool, scale, kept in (("k", c.k_pool, c.k_scale, c.k_open), ("v", c.v_pool, c.v_scale, c.v_open)):
            codes, scale, kept = pool.view(torch.int8).cpu().numpy(), scale.cpu().numpy(), kept.cpu().numpy()
            seen = np.zeros(codes.shape[:2], bool)
            for (slot, b), count in self.touched.items():
                want, s = self.expect(side, slot, b, count)
                at = self.table[slot, b]
                seen[at, LAYER] = True
                assert np.array_equal(scale[at, LAYER], s), (side, slot, b)
                assert np.array_equal(O.numbers(codes[at, LAYER], self.fmt), want), (side, slot, b)
                n = len(self.rows[slot][side])
                if b == n // self.B and n % self.B:
                    rows = self.rows[slot][side][b * self.B:n].transpose(1, 0, 2)
                    assert np.array_equal(kept[slot, LAYER][:, :n % self.B], rows, equal_nan=True)
            assert (codes[~seen] == 55).all() and (scale[~seen] == 7.25).all()
            assert (np.delete(kept, LAYER, 1) == 7.25).all()

    def random(self, n, width, dtype, pitch=0, lead=0):
        """[n, H * width] of values over a few powers of two, as columns of a wider array"""
        x = torch.from_numpy(self.rng.standard_normal((n, self.H * width + pitch)).astype(np.float32) * np.exp2(self.rng.integers(-6, 3, (n, 1))).astype(np.float32))
        return x.to(dtype).cuda()[:, lead:lead + self.H * width]

    def put(self, portions, dtype=torch.float32, **kw):
        n = sum(x[2] for x in portions)
        self.write(portions, self.random(n, self.dim, dtype, **kw), self.random(n, self.vdim, dtype, **kw))

    def values(self, side, slot, n, dtype=np.float64):
        """Cached rows 0 .. n - 1 as the pool holds them, [n, H, width]"""
        pool, scale = (self.cache.k_pool, self.cache.k_scale) if side == "k" else (self.cache.v_pool, self.cache.v_scale)
        pool, scale = pool.view(torch.int8).cpu().numpy(), scale.cpu().numpy()
        t = np.arange(n)
        ids = self.table[slot, t // self.B]
        return O.numbers(pool[ids, LAYER, :, t % self.B], self.fmt) * scale[ids, LAYER].astype(np.float64)[..., None]


STEPS = [[(0, 0, 37), (1, 0, 1), (2, -1, 1)], [(1, 1, 50), (0, 37, 1)], [(0, 38, 170), (2, 0, 16), (1, 51, 13)], [(2, 16, 1), (0, 208, 1), (1, 64, 64)],
         [(0, 209, 1), (1, 128, 1), (2, 17, 130)], [(0, 209, 3), (2, 144, 5)]]


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("block,kv_heads,dim,vdim", [(16, 2, 64, 64), (32, 3, 128, 128), (64, 1, 16, 80), (128, 2, 128, 112), (16, 5, 96, 32)])
@pytest.mark.parametrize("dtype,pitch,lead", [(torch.float32, 0, 0), (torch.float32, 9, 3), (torch.bfloat16, 8, 4), (torch.bfloat16, 0, 0), (torch.bfloat16, 5, 1)])
def test_rows_enter_block_by_block(fmt, block, kv_heads, dim, vdim, dtype, pitch, lead):
    """Portions that begin and end anywhere, beside single rows, an idle sequence and the last rows written anew: codes, scales, kept rows to the bit, nothing else touched."""
    m = Mirror(3, 256, kv_heads, block, dim, vdim, fmt)
    for step in STEPS:
        m.put(step, dtype, pitch=pitch, lead=lead)
        m.check()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_portions_do_not_show(fmt):
    """A context that enters at once and one that enters row by row have the same codes and scales."""
    n, B = 83, 32
    a, b = Mirror(1, 128, 2, B, 64, 64, fmt), Mirror(1, 128, 2, B, 64, 64, fmt)
    k, v = a.random(n, 64, torch.float32), a.random(n, 64, torch.float32)
    a.write([(0, 0, n)], k, v)
    for i in range(n):
        b.write([(0, i, 1)], k[i:i + 1], v[i:i + 1])
    for x, y in ((a.cache.k_pool, b.cache.k_pool), (a.cache.v_pool, b.cache.v_pool), (a.cache.k_scale, b.cache.k_scale), (a.cache.v_scale, b.cache.v_scale)):
        assert bool((x.view(torch.int8) == y.view(torch.int8)).all())


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_values_at_borders_and_ends(fmt):
    """Quotients on and beside every border between two codes, under scales that make them inexact; zeros; the smallest numbers; infinities and NaN."""
    m = Mirror(1, 2048, 1, 32, 128, 128, fmt)
    lv = O.levels(fmt)
    edge = np.concatenate([(lv[1:] + lv[:-1]) / 2, lv])
    rows = []
    for top in (1.0, 3.0, 0.1, 1e-30, 7e20, O.MOST[fmt], 2.0 ** -120):
        s = np.float32(np.float64(np.float32(top)) / O.MOST[fmt])
        x = (edge * np.float64(s)).astype(np.float32)
        x = np.concatenate([x, np.nextafter(x, np.float32(np.inf)), np.nextafter(x, np.float32(0)), -x])
        x = x[np.abs(x) <= np.float32(top)]
        x = np.resize(np.concatenate([[np.float32(top)], x]), (32, 128))
        rows.append(x)
    tiny = np.float32(1e-45)
    rows.append(np.resize(np.array([0, tiny, -tiny, 5 * tiny, 2.0 ** -126, 2.0 ** -130], np.float32), (32, 128)))
    rows.append(np.zeros((32, 128), np.float32))
    rows.append(np.resize(np.array([np.inf, -np.inf, np.nan, 1.5, -0.25, 0, 3.0], np.float32), (32, 128)))
    rows.append(np.resize(np.array([np.inf, -np.inf, np.nan, 0], np.float32), (32, 128)))
    rows.append(np.resize(np.array([3.4e38, -3.4e38, 1e38, 1.0, np.inf], np.float32), (32, 128)))
    x = torch.from_numpy(np.concatenate(rows)).cuda()
    m.write([(0, 0, len(x))], x, x.flip(1).contiguous())
    m.check()
    k, v = m.cache.read(K.Rows.of([(0, 0, len(x))]), layer=LAYER)
    assert bool(torch.isfinite(k).all()) and bool(torch.isfinite(v).all())


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("block,kv_heads,dim,vdim", [(16, 2, 64, 64), (128, 3, 128, 48), (32, 1, 16, 112)])
@pytest.mark.parametrize("dtype,pitch,lead", [(torch.float32, 0, 0), (torch.bfloat16, 0, 0), (torch.float32, 7, 2), (torch.bfloat16, 16, 8), (torch.bfloat16, 3, 1)])
def test_rows_come_back(fmt, block, kv_heads, dim, vdim, dtype, pitch, lead):
    m = Mirror(3, 256, kv_heads, block, dim, vdim, fmt)
    m.put([(0, 0, 200), (1, 0, 77), (2, 0, 1)])
    parts = [(1, 13, 60), (2, -1, 1), (0, 150, 50), (1, 0, 1), (2, 0, 1)]
    n = sum(x[2] for x in parts)
    outs = [torch.full((n, kv_heads * w + pitch), 9.0, device="cuda", dtype=dtype) for w in (dim, vdim)]
    views = [o[:, lead:lead + kv_heads * w] for o, w in zip(outs, (dim, vdim))]
    m.cache.read(K.Rows.of(parts), layer=LAYER, k_out=views[0], v_out=views[1])
    for side, out, view, w in (("k", outs[0], views[0], dim), ("v", outs[1], views[1], vdim)):
        want = np.concatenate([m.values(side, s, p + c)[p:] if p >= 0 else np.zeros((c, kv_heads, w)) for s, p, c in parts]).reshape(n, -1)
        want = torch.from_numpy(want).float().to(dtype).cuda()         # float64 holds the product; two roundings to bf16 as in the kernel
        assert bool((view == want).all())
        rest = torch.ones(out.shape[1], dtype=torch.bool)
        rest[lead:lead + kv_heads * w] = False
        assert bool((out[:, rest.cuda()] == 9.0).all())


def test_blocks_that_do_not_exist():
    """Ids beside the pool: not written, zeros when read, keys that are not seen; a row that sees no key gets zeros."""
    m = Mirror(2, 128, 2, 16, 64, 64, "int8")
    m.put([(0, 0, 100), (1, 0, 40)])
    before = [t.clone() for t in (m.cache.k_pool, m.cache.v_pool, m.cache.k_scale, m.cache.v_scale)]
    bad = m.cache.table.clone()
    bad[0, 2], bad[0, 4], bad[1, :] = -1, m.cache.k_pool.shape[0], 1 << 30
    m.cache.table.copy_(bad)
    n = 100
    k, v = m.cache.read(K.Rows.of([(0, 0, n)]), layer=LAYER)
    absent = np.isin(np.arange(n) // 16, (2, 4))
    q = torch.randn(3, 4 * 64, device="cuda")
    for r, lo in ((K.Rows.of([(0, 97, 3)]), 97), (K.Rows.of([(0, 99, 1), (1, 39, 1), (1, -1, 1)]), 99)):
        out = m.cache.attend(K.Attention(4, 2, 64, scale=0.125), r, q, layer=LAYER)
        rows = 3 if lo == 97 else 1
        want = O.attend({"scale": 0.125}, q[:rows].double().cpu().numpy().reshape(rows, 4, 64), m.values("k", 0, n), m.values("v", 0, n), lo, absent)
        assert rel(out[:rows], want.reshape(rows, -1)) < F32_TOL
        assert lo == 97 or bool((out[1:] == 0).all())
    for side, got in (("k", k), ("v", v)):
        want = np.where(absent[:, None, None], 0, m.values(side, 0, n)).reshape(n, -1)
        assert np.array_equal(got.cpu().numpy(), want.astype(np.float32))
    m.cache.write(K.Rows.of([(0, 32, 8), (1, 0, 20)]), torch.ones(28, 128, device="cuda"), torch.ones(28, 128, device="cuda"), layer=LAYER)
    torch.cuda.synchronize()
    for t, b in zip((m.cache.k_pool, m.cache.v_pool, m.cache.k_scale, m.cache.v_scale), before):
        assert bool((t == b).all())


def rel(got, want):
    w = torch.from_numpy(np.ascontiguousarray(want)).cuda()
    return float((got.double() - w).norm() / w.norm())


def attend(m, a, parts, dtype, q_seed=5, scale_q=1.0, gate=None):
    """(result, float64) of the rows of `parts` over m's cache; a: what O.attend takes, with heads."""
    heads, g = a["heads"], torch.Generator(device="cuda").manual_seed(q_seed)
    n = sum(x[2] for x in parts)
    q = torch.randn(n, heads * m.dim, device="cuda", generator=g) * scale_q
    dev = lambda x: None if x is None else torch.from_numpy(np.ascontiguousarray(x, np.float32)).cuda()  # noqa: E731
    at = K.Attention(heads, m.H, m.dim, m.vdim, scale=a["scale"], chunk=a.get("chunk", 0), window=a.get("window", 0), keep_first=a.get("keep_first", 0), sink=dev(a.get("sink")),
                     head_scale=dev(a.get("head_scale")), softcap=a.get("softcap", 0.0), rel=dev(a.get("rel")), head_gate=gate is not None, gate_column=3)
    proj = None
    if gate is not None:
        proj = torch.zeros(n, heads + 5, device="cuda")
        proj[:, 3:3 + heads] = torch.from_numpy(gate).cuda()
    out = m.cache.attend(at, K.Rows.of(parts), q, layer=LAYER, dtype=dtype, proj=proj)
    want, row = [], 0
    qn = q.double().cpu().numpy().reshape(n, heads, m.dim)
    for slot, p, c in parts:
        b = dict(a)
        if gate is not None:
            b["gate"] = gate[row:row + c].astype(np.float64)
        want.append(O.attend(b, qn[row:row + c], m.values("k", slot, p + c), m.values("v", slot, p + c), p) if p >= 0 else np.zeros((c, heads, m.vdim)))
        row += c
    return out, np.concatenate(want).reshape(n, -1)


def close(out, want, f32_tol=F32_TOL):
    assert bool(torch.isfinite(out).all())
    assert rel(out, want) < (f32_tol if out.dtype == torch.float32 else f32_tol + BF16_STEP)


SINGLES = [(2, 40, 1), (1, -1, 1), (0, 700, 1), (3, 255, 1), (4, 0, 1), (1, 256, 1), (2, 1100, 1)]
PORTIONS = [(2, 0, 40), (0, 690, 11), (3, 250, 6), (4, 0, 1), (1, 100, 157)]


def filled(block, kv_heads, dim, vdim, fmt, lengths=(701, 257, 1101, 256, 1)):
    m = Mirror(len(lengths), max(lengths), kv_heads, block, dim, vdim, fmt)
    n = sum(lengths)
    # keys and values of order one
    k, v = (torch.from_numpy(m.rng.standard_normal((n, kv_heads * w)).astype(np.float32)).cuda() for w in (dim, vdim))
    m.write([(i, 0, c) for i, c in enumerate(lengths)], k, v)
    return m


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("block,heads,kv_heads,dim,vdim", [(16, 4, 4, 64, 64), (32, 8, 2, 128, 128), (64, 8, 1, 128, 64), (128, 20, 2, 96, 112), (16, 3, 3, 16, 128), (16, 16, 1, 80, 16)])
@pytest.mark.parametrize("parts", [SINGLES, PORTIONS], ids=["singles", "portions"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attention(fmt, block, heads, kv_heads, dim, vdim, parts, dtype):
    m = filled(block, kv_heads, dim, vdim, fmt)
    out, want = attend(m, dict(heads=heads, scale=dim ** -0.5), parts, dtype)
    close(out, want)
    for i in [i for i, x in enumerate(parts) if x[1] < 0]:
        at = sum(x[2] for x in parts[:i])
        assert bool((out[at] == 0).all())


MASKS = [dict(window=1), dict(window=33, keep_first=4), dict(window=300, keep_first=70), dict(window=100000, keep_first=3), dict(chunk=64), dict(chunk=50), dict(chunk=1),
         dict(sink=True), dict(sink=True, window=5), dict(softcap=3.0), dict(softcap=20.0, window=100, keep_first=33), dict(rel=1), dict(rel=40, sink=True),
         dict(rel=2000, softcap=9.0), dict(head_scale=True), dict(gate=True, sink=True), dict(head_scale=True, gate=True, chunk=200)]


@pytest.mark.parametrize("mask", MASKS, ids=lambda m: "-".join(f"{k}{'' if v is True else v}" for k, v in m.items()))
@pytest.mark.parametrize("fmt,heads,kv_heads,dim,vdim,block", [("int8", 6, 2, 128, 128, 16), ("e4m3", 5, 1, 64, 48, 64)])
@pytest.mark.parametrize("parts", [SINGLES, PORTIONS], ids=["singles", "portions"])
def test_masks_and_options(mask, fmt, heads, kv_heads, dim, vdim, block, parts):
    """tanh multiplies a score's error by at most 1; a distance bias is added in fp32."""
    m = filled(block, kv_heads, dim, vdim, fmt)
    rng = np.random.default_rng(3)
    a = dict(mask, heads=heads, scale=dim ** -0.5)
    if a.get("sink"):
        a["sink"] = rng.standard_normal(heads).astype(np.float32)
    if a.get("head_scale"):
        a["head_scale"] = rng.uniform(-1.5, 1.5, heads).astype(np.float32)
    if a.get("rel"):
        a["rel"] = rng.standard_normal((heads, a["rel"])).astype(np.float32)
    gate = rng.standard_normal((sum(x[2] for x in parts), heads)).astype(np.float32) if a.pop("gate", None) else None
    out, want = attend(m, a, parts, torch.float32, gate=gate)
    close(out, want)


@pytest.mark.parametrize("mask", MASKS, ids=lambda m: "-".join(f"{k}{'' if v is True else v}" for k, v in m.items()))
@pytest.mark.parametrize("fmt,heads,kv_heads,dim,vdim,block,dtype", [("int8", 12, 4, 128, 128, 16, torch.float32), ("e4m3", 20, 4, 64, 48, 64, torch.float32),
                                                                     ("e4m3", 16, 4, 112, 128, 32, torch.bfloat16)])
def test_masks_and_options_of_prompts(mask, fmt, heads, kv_heads, dim, vdim, block, dtype):
    parts = [(0, 300, 700), (1, 0, 40)]
    m = filled(block, kv_heads, dim, vdim, fmt, (1000, 40))
    rng = np.random.default_rng(3)
    a = dict(mask, heads=heads, scale=dim ** -0.5)
    if a.get("sink"):
        a["sink"] = rng.standard_normal(heads).astype(np.float32)
    if a.get("head_scale"):
        a["head_scale"] = rng.uniform(-1.5, 1.5, heads).astype(np.float32)
    if a.get("rel"):
        a["rel"] = rng.standard_normal((heads, a["rel"])).astype(np.float32)
    gate = rng.standard_normal((740, heads)).astype(np.float32) if a.pop("gate", None) else None
    assert takes_tiles(a, m, parts, dtype) or a.get("window", 10000) < 100 or a.get("chunk", 10000) < 100    # few keys: no tiles pay
    out, want = attend(m, a, parts, dtype, gate=gate)
    close(out, want)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("parts", [[(0, 1299, 1)], [(0, 700, 600)]], ids=["single", "portion"])
def test_blocks_of_very_different_scales(fmt, parts):
    """Values of blocks 2^20 apart: what is small beside the largest block's is off by less than 2^-28 of a weight times the largest scale's values."""
    m = Mirror(1, 1300, 2, 16, 64, 64, fmt)
    k, v = (torch.from_numpy(m.rng.standard_normal((1300, 128)).astype(np.float32)).cuda() for _ in range(2))
    up = torch.exp2(torch.from_numpy(m.rng.integers(-20, 1, 82).repeat(16)[:1300].astype(np.float32))).cuda()
    m.write([(0, 0, 1300)], k * 0.3, v * up[:, None])
    assert takes_tiles(dict(heads=32, scale=0.125), m, parts, torch.float32) == (parts[0][2] > 1)
    out, want = attend(m, dict(heads=32, scale=0.125), parts, torch.float32)
    close(out, want)
    # ... and alone under a window that hides the others
    m.write([(0, 0, 1300)], k * 0.3, v * 2.0 ** -100)
    out, want = attend(m, dict(heads=32, scale=0.125, window=140), parts, torch.float32)
    close(out, want)


@pytest.mark.parametrize("parts", [[(0, 299, 1)], [(0, 200, 100)], [(0, 0, 1600)]], ids=["single", "portion", "prompt"])
def test_keys_of_zeros_and_scores_far_apart(parts):
    """A cache of zeros gives zeros; scores hundreds apart leave one key."""
    n = parts[0][1] + parts[0][2]
    m = Mirror(1, n, 1, 16, 64, 64, "int8")
    z = torch.zeros(n, 64, device="cuda")
    m.write([(0, 0, n)], z, z)
    a = dict(heads=8, scale=0.125)
    assert takes_tiles(a, m, parts, torch.float32) == (n == 1600)
    out, want = attend(m, a, parts, torch.float32)
    assert bool((out == 0).all())
    k, v = (torch.from_numpy(m.rng.standard_normal((n, 64)).astype(np.float32)).cuda() for _ in range(2))
    m.write([(0, 0, n)], k, v)
    out, want = attend(m, a, parts, torch.float32, scale_q=200.0)
    # scores of order 200 * 8 / 8: errors 200 times those of the head comment
    close(out, want, 200 * F32_TOL)


def test_a_query_that_is_not_a_number():
    m = filled(16, 1, 64, 64, "int8", (300,))
    q = torch.randn(2, 64, device="cuda")
    q[1, 5] = float("nan")
    for parts in ([(0, 298, 2)], [(0, 299, 1), (0, 299, 1)]):
        out = m.cache.attend(K.Attention(1, 1, 64, scale=0.125), K.Rows.of(parts), q, layer=LAYER)
        assert bool(torch.isfinite(out[0]).all()) and bool(torch.isnan(out[1]).all())


def test_a_query_of_a_portion_that_is_not_a_number():
    m = filled(32, 4, 128, 128, "int8", (900,))
    q = torch.randn(500, 16 * 128, device="cuda")
    q[123, 130] = float("nan")
    q[7, 400] = float("inf")
    for dtype in (torch.float32, torch.bfloat16):
        assert takes_tiles(dict(heads=16, scale=0.1), m, [(0, 400, 500)], dtype)
        out = m.cache.attend(K.Attention(16, 4, 128, scale=0.1), K.Rows.of([(0, 400, 500)]), q, layer=LAYER, dtype=dtype).view(500, 16, 128)
        bad = torch.zeros(500, 16, dtype=torch.bool, device="cuda")
        bad[123, 1] = bad[7, 3] = True
        assert bool((~torch.isfinite(out)).all(-1)[bad].all()) and bool(torch.isfinite(out)[~bad].all())


def takes_tiles(a, m, parts, dtype):
    """Whether the step's portions go to the tensor-core form of prompts: it stages the visible keys and values in fp16, which is most of the scratch that it asks for."""
    lib, r = K.lib(), K.Rows.of(parts)
    at = K.Attention(a["heads"], m.H, m.dim, m.vdim, scale=a["scale"], chunk=a.get("chunk", 0), window=a.get("window", 0), keep_first=a.get("keep_first", 0))
    floats = lib.c.tha_hyb_kv8_attn_scratch(K.DTYPES[dtype], at.ref, r.ref, m.cache.ref)
    keys = min(max(p + n for _, p, n in parts), a.get("window") or 1 << 30, a.get("chunk") or 1 << 30)
    return floats >= keys * m.H * (128 if max(m.dim, m.vdim) > 64 else 64)


LONG = [("int8", 16, 16, 4, 128, 128, [(0, 1500, 300)], {}), ("e4m3", 64, 16, 4, 128, 128, [(0, 3000, 250)], dict(window=1000, keep_first=40)),
        ("int8", 16, 8, 8, 64, 64, [(0, 100, 450), (1, 0, 520), (2, 2000, 400)], {}), ("int8", 32, 20, 4, 96, 80, [(0, 900, 460), (1, 17, 3), (2, 3, 1), (3, 40, 90)], dict(sink=True)),
        ("e4m3", 128, 32, 2, 128, 64, [(0, 2500, 177), (1, 30, 60)], dict(chunk=700)), ("int8", 16, 12, 4, 16, 128, [(0, 0, 900)], dict(softcap=5.0)),
        ("e4m3", 16, 12, 4, 112, 48, [(0, 1000, 500)], dict(rel=300)), ("int8", 16, 4, 4, 128, 128, [(i, 7 * i, 230 + i % 3) for i in range(40)], {}),
        ("e4m3", 32, 128, 1, 64, 16, [(0, 2000, 300)], {}), ("int8", 64, 5, 5, 48, 64, [(0, 0, 1300), (1, -1, 1)], dict(window=300))]


@pytest.mark.parametrize("case", LONG, ids=lambda c: f"{c[0]}-{c[1]}-{c[2]}-{c[3]}-{c[4]}-{c[5]}-{len(c[6])}")
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lead", [0, 1])
def test_prompt_portions(case, dtype, lead):
    """Portions for the tensor-core form, behind contexts that are cut and beside short ones; with lead 1 the result is on no 16-byte boundary."""
    fmt, block, heads, kv_heads, dim, vdim, parts, mask = case
    m = filled(block, kv_heads, dim, vdim, fmt, [max(1, p + n) for _, p, n in parts])
    rng = np.random.default_rng(3)
    a = dict(mask, heads=heads, scale=dim ** -0.5)
    if a.get("sink"):
        a["sink"] = rng.standard_normal(heads).astype(np.float32)
    if a.get("rel"):
        a["rel"] = rng.standard_normal((heads, a["rel"])).astype(np.float32)
    assert takes_tiles(a, m, parts, dtype)
    out, want = attend(m, a, parts, dtype)
    close(out, want)
    if lead:
        room = torch.full((out.numel() + 1,), 9.0, device="cuda", dtype=dtype)
        dev = lambda x: None if x is None else torch.from_numpy(x).cuda()  # noqa: E731
        at = K.Attention(heads, kv_heads, dim, vdim, scale=a["scale"], chunk=a.get("chunk", 0), window=a.get("window", 0), keep_first=a.get("keep_first", 0),
                         sink=dev(a.get("sink")), softcap=a.get("softcap", 0.0), rel=dev(a.get("rel")))
        q = torch.randn(out.shape[0], heads * dim, device="cuda", generator=torch.Generator(device="cuda").manual_seed(5))
        m.cache.attend(at, K.Rows.of(parts), q, layer=LAYER, out=room[1:].view(out.shape))
        close(room[1:].view(out.shape), want)
        assert float(room[0]) == 9.0


@pytest.mark.parametrize("rows", [30, 600])
def test_blocks_that_do_not_exist_under_a_portion(rows):
    m = filled(16, 4, 128, 128, "int8", (900,))
    bad = m.cache.table.clone()
    for b in (0, 9, 30, 50):
        bad[0, b] = -7 if b & 1 else m.cache.k_pool.shape[0]
    m.cache.table.copy_(bad)
    q, p0 = torch.randn(rows, 16 * 128, device="cuda"), 900 - rows
    assert takes_tiles(dict(heads=16, scale=0.1), m, [(0, p0, rows)], torch.float32) == (rows == 600)
    out = m.cache.attend(K.Attention(16, 4, 128, scale=0.1), K.Rows.of([(0, p0, rows)]), q, layer=LAYER)
    absent = np.isin(np.arange(900) // 16, (0, 9, 30, 50))
    want = O.attend(dict(scale=0.1), q.double().cpu().numpy().reshape(rows, 16, 128), m.values("k", 0, 900), m.values("v", 0, 900), p0, absent)
    assert rel(out, want.reshape(rows, -1)) < F32_TOL


@pytest.mark.parametrize("share", [0.0, 0.01, 0.5, 0.95, 0.99, 1.0, 1.5])
@pytest.mark.parametrize("parts", [[(0, 3700, 300)], [(0, 3700, 300), (1, 20, 90), (1, 30, 1), (0, 1000, 270)]], ids=["one", "four"])
def test_parts_of_a_portions_context_meet(share, parts):
    """With less room than the call would like, and nothing behind the room."""
    m = filled(16, 1, 128, 128, "int8", (4000, 111))
    heads, n = 8, sum(x[2] for x in parts)
    assert takes_tiles(dict(heads=heads, scale=128 ** -0.5), m, parts, torch.float32)
    out, want = attend(m, dict(heads=heads, scale=128 ** -0.5), parts, torch.float32)
    close(out, want)
    r, at, lib = K.Rows.of(parts), K.Attention(heads, 1, 128, scale=128 ** -0.5), K.lib()
    at.c.cache_layer = LAYER
    q = torch.randn(n, heads * 128, device="cuda", generator=torch.Generator(device="cuda").manual_seed(5))
    floats = int(share * lib.c.tha_hyb_kv8_attn_scratch(1, at.ref, r.ref, m.cache.ref))
    room = torch.full((floats + 512,), 3.25, device="cuda")
    got = torch.full_like(out, float("nan"))
    lib.check(lib.c.tha_hyb_kv8_attn(torch.cuda.current_stream().cuda_stream, 1, at.ref, r.ref, m.cache.ref, q.data_ptr(), got.data_ptr(), room.data_ptr() if floats else None,
                                     floats, None, 0))
    torch.cuda.synchronize()
    assert bool((room[floats:] == 3.25).all())
    close(got, want)


@pytest.mark.parametrize("scratch", [0, 1, 2, 7, 63, 1000])
def test_parts_of_a_context_meet(scratch):
    """With any room for partial results, and nothing behind the room."""
    m = filled(16, 2, 128, 128, "int8", (2100, 40))
    parts, heads = [(0, 2099, 1), (1, 39, 1), (1, -1, 1)], 4
    out, want = attend(m, dict(heads=heads, scale=128 ** -0.5), parts, torch.float32)
    close(out, want)
    r, at = K.Rows.of(parts), K.Attention(heads, 2, 128, scale=128 ** -0.5)
    at.c.cache_layer = LAYER
    q = torch.randn(3, heads * 128, device="cuda", generator=torch.Generator(device="cuda").manual_seed(5))
    floats = scratch * 3 * heads * 130
    room = torch.full((floats + 512,), 3.25, device="cuda")
    got = torch.full_like(out, float("nan"))
    lib = K.lib()
    lib.check(lib.c.tha_hyb_kv8_attn(torch.cuda.current_stream().cuda_stream, 1, at.ref, r.ref, m.cache.ref, q.data_ptr(), got.data_ptr(), room.data_ptr() if floats else None,
                                     floats, None, 0))
    torch.cuda.synchronize()
    assert bool((room[floats:] == 3.25).all())
    close(got, want)


def test_a_very_long_context():
    """Offsets of a pool beyond 2^31 bytes, and a table of more blocks than a block of threads holds at once."""
    n, D = 70000, 128
    assert n > 2 * 8192
    big = K.Kv8Cache.empty(blocks=180000, layers=LAYERS, kv_heads=2, block_size=16, dim=D, slots=1, table_stride=-(-n // 16))   # 2.2e9 bytes a pool
    ids = torch.arange(179999, 179999 - big.table.shape[1], -1, dtype=torch.int32)
    big.table[0] = ids.cuda()
    k, v = (torch.randn(n, 2 * D, device="cuda") for _ in range(2))
    big.write(K.Rows.of([(0, 0, n)]), k, v, layer=LAYER)
    kb, vb = big.read(K.Rows.of([(0, 0, n)]), layer=LAYER)
    step = torch.maximum(k.abs().max(), v.abs().max()) / 127
    assert float((kb - k).abs().max()) <= 0.5001 * float(step) and float((vb - v).abs().max()) <= 0.5001 * float(step)
    q = torch.randn(1, 2 * D, device="cuda")
    at = K.Attention(2, 2, D, scale=D ** -0.5)
    out = big.attend(at, K.Rows.of([(0, n - 1, 1)]), q, layer=LAYER)
    s = torch.einsum("hd,thd->ht", q.double().view(2, D), kb.double().view(n, 2, D)) * D ** -0.5
    want = torch.einsum("ht,the->he", torch.softmax(s, -1), vb.double().view(n, 2, D)).reshape(1, -1)
    assert rel(out, want.cpu().numpy()) < F32_TOL
    # without room for parts: one block of threads and all keys
    at.c.cache_layer = LAYER
    lib, r = K.lib(), K.Rows.of([(0, n - 1, 1)])
    out.fill_(float("nan"))
    lib.check(lib.c.tha_hyb_kv8_attn(torch.cuda.current_stream().cuda_stream, 1, at.ref, r.ref, big.ref, q.data_ptr(), out.data_ptr(), None, 0, None, 0))
    assert rel(out, want.cpu().numpy()) < F32_TOL
    # a portion, with tiles and parts, and without
    q = torch.randn(130, 2 * D, device="cuda")
    r = K.Rows.of([(0, n - 130, 130)])
    assert lib.c.tha_hyb_kv8_attn_scratch(1, at.ref, r.ref, big.ref) > n * 2 * 128
    hidden = torch.arange(n, device="cuda")[None] > torch.arange(n - 130, n, device="cuda")[:, None]
    s = torch.einsum("rhd,thd->hrt", q.double().view(130, 2, D), kb.double().view(n, 2, D)) * D ** -0.5
    want = torch.einsum("hrt,the->rhe", torch.softmax(s.masked_fill(hidden, float("-inf")), -1), vb.double().view(n, 2, D)).reshape(130, -1).cpu().numpy()
    out = big.attend(at, r, q, layer=LAYER)
    assert rel(out, want) < F32_TOL
    out.fill_(float("nan"))
    lib.check(lib.c.tha_hyb_kv8_attn(torch.cuda.current_stream().cuda_stream, 1, at.ref, r.ref, big.ref, q.data_ptr(), out.data_ptr(), None, 0, None, 0))
    assert rel(out, want) < F32_TOL


def test_other_streams_and_graphs():
    """A step (write, attend, read) on a stream of its own, captured and replayed with new rows, equals the eager one; two graphs share nothing but the cache."""
    m = filled(16, 2, 64, 64, "e4m3", (600, 300))
    at = K.Attention(8, 2, 64, scale=0.125)
    rows = K.Rows.of([(0, 601, 1), (1, 301, 1)])
    k, v, q = (torch.randn(2, w, device="cuda") for w in (128, 128, 512))

    def step():
        m.cache.write(rows, k, v, layer=LAYER)
        return m.cache.attend(at, rows, q, layer=LAYER), m.cache.read(rows, layer=LAYER)

    m.cache.write(K.Rows.of([(0, 600, 1), (1, 300, 1)]), k, v, layer=LAYER)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = step()
        graphs.append((g, got))
    for seed in (1, 2, 3):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        for t in (k, v, q):
            t.copy_(torch.randn(t.shape, device="cuda", generator=gen))
        want = step()
        torch.cuda.synchronize()
        for g, got in graphs:
            for x in (got[0], *got[1]):
                x.fill_(float("nan"))
            g.replay()
            torch.cuda.synchronize()
            assert bool((got[0] == want[0]).all()) and all(bool((a == b).all()) for a, b in zip(got[1], want[1]))


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("parts", [[(0, 110, 1), (1, 120, 1)], [(1, 100, 21), (0, 111, 1)], [(0, 96, 16), (1, 96, 25)]], ids=["single", "mixed", "portions"])
def test_full_blocks_of_two_slots(fmt, parts):
    """Two slots share a prefix of full blocks: each writes behind it, the prefix keeps its bytes, and both attend over it."""
    m = Mirror(2, 160, 2, 16, 64, 64, fmt)
    m.put([(0, 0, 96)])
    m.table[1, :6] = m.table[0, :6]
    m.cache.table.copy_(torch.from_numpy(m.table))
    ids = torch.from_numpy(m.table[0, :6].astype(np.int64)).cuda()
    before = [t.view(torch.int8)[ids].clone() for t in (m.cache.k_pool, m.cache.v_pool)] + [t[ids].clone() for t in (m.cache.k_scale, m.cache.v_scale)]
    for slot in (0, 1):
        m.rows[slot] = {side: m.rows[0][side][:96] for side in "kv"}
    m.put([(0, 96, 16), (1, 96, 25)])
    m.check()
    for was, t in zip(before, (m.cache.k_pool.view(torch.int8), m.cache.v_pool.view(torch.int8), m.cache.k_scale, m.cache.v_scale)):
        assert torch.equal(was, t[ids])
    for dtype in (torch.float32, torch.bfloat16):
        out, want = attend(m, dict(heads=8, scale=0.125), parts, dtype)
        close(out, want)


def test_a_step_of_idle_slots():
    m = filled(16, 2, 64, 64, "int8", (30, 30))
    before = m.cache.k_pool.clone()
    r = K.Rows.of([(1, -1, 1), (0, -1, 1)])
    m.cache.write(r, torch.ones(2, 128, device="cuda"), torch.ones(2, 128, device="cuda"), layer=LAYER)
    k, v = m.cache.read(r, layer=LAYER)
    out = m.cache.attend(K.Attention(4, 2, 64, scale=0.125, sink=torch.zeros(4, device="cuda")), r, torch.randn(2, 256, device="cuda"), layer=LAYER)
    assert bool((m.cache.k_pool == before).all()) and bool((k == 0).all()) and bool((v == 0).all()) and bool((out == 0).all())


def test_calls_side_by_side():
    """Attention of two steps on two streams at once over one cache."""
    m = filled(16, 2, 128, 128, "int8", (3000, 2900))
    at = [K.Attention(4, 2, 128, scale=0.1), K.Attention(8, 2, 128, scale=0.1)]
    rows = [K.Rows.of([(0, 2999, 1)]), K.Rows.of([(1, 2890, 10)])]
    q = [torch.randn(1, 512, device="cuda"), torch.randn(10, 1024, device="cuda")]
    want = [m.cache.attend(at[i], rows[i], q[i], layer=LAYER) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append((i, m.cache.attend(at[i], rows[i], q[i], layer=LAYER)))
    torch.cuda.synchronize()
    assert all(bool((o == want[i]).all()) for i, o in got)


def test_a_prompt_then_decoding():
    """The operators together, as a serving loop calls them: a prompt in portions beside another request's decoding; every result against the definition on the cache as it then was,
    and near the attention over the rows as they were."""
    H, D, heads = 2, 64, 6
    m = Mirror(2, 400, H, 16, D, D, "int8")
    rng = np.random.default_rng(0)
    at = [0, 0]
    for step, counts in enumerate([(120, 0), (64, 30), (1, 1), (1, 1), (0, 1), (77, 1), (1, 40), (1, 1)]):
        parts = [(s, at[s], c) for s, c in enumerate(counts) if c]
        n = sum(c for c in counts)
        k, v = (torch.from_numpy(rng.standard_normal((n, H * D)).astype(np.float32)).cuda() for _ in range(2))
        m.write(parts, k, v)
        at = [x + c for x, c in zip(at, counts)]
        out, want = attend(m, dict(heads=heads, scale=D ** -0.5), parts, torch.float32, q_seed=step)
        close(out, want)
        qn = torch.randn(n, heads * D, device="cuda", generator=torch.Generator(device="cuda").manual_seed(step)).double().cpu().numpy().reshape(n, heads, D)
        row, plain = 0, []
        for s, p, c in parts:
            plain.append(O.attend(dict(scale=D ** -0.5), qn[row:row + c], *(m.rows[s][x][:p + c].astype(np.float64) for x in ("k", "v")), p))
            row += c
        # a value of order one under a scale of about 3.5 / 127 is off by 1.4% of one, by half of that on the average of a step: uniform, 0.8% rms; scores by as much times |q| / 8
        assert rel(out, np.concatenate(plain).reshape(n, -1)) < 0.05
    m.check()
