"""Attention over the cache in 8 bits, every (row, head, channel) by itself against float64: rows that see little stand beside rows that see much, and a norm over all of them shows the
first alone.

The bound of a result o_c = sum_j p_j v_jc: an error of eps in every score or weight moves it by eps * (sum_j p_j |v_jc| + |o_c|).
eps, fp32 results: a score sums products of absolute sum T (its largest over the visible keys), q off by 2^-22, and dim / 16 sums of two operands cut off at 2^-23 of what is there; the score beside
its maximum, X in units of ln 2 and 16 more, is rounded twice; tanh is off by 2^-22 of the cap; a weight by 3 * 2^-22; 128 sums in a row, each cut off at 2^-23.
One fp16 an operand (bf16 results of long portions): 2^-11 of the products and of the weight more.
On top, 2^-29 of the row's largest weight times the largest VISIBLE scale for every visible key (the header's statement, a scale's largest number being 128 or more of its steps), doubled
for what the weights' sum takes of it; and the last rounding, 2^-24 or 2^-8 of the result."""
import numpy as np
import pytest
import torch

import kv8_oracle as O
import test_gpu_kv8 as T

pytestmark = pytest.mark.gpu
K, LAYER = T.K, T.LAYER


def expected(a, q, keys, values, p0, eps_more=0.0):
    """(results, bounds) [n, heads, vdim] of rows at p0 .. in float64."""
    n, heads, dim = q.shape
    group = heads // keys.shape[1]
    t, p = np.arange(keys.shape[0])[None], np.arange(p0, p0 + n)[:, None]
    vis = O.sees(a, t, p)
    out, far = np.zeros((n, heads, values.shape[2])), np.zeros((n, heads, values.shape[2]))
    for h in range(heads):
        k, v = keys[:, h // group], values[:, h // group]
        f = a["scale"] * (a["head_scale"][h] if a.get("head_scale") is not None else 1.0)
        s = q[:, h] @ k.T * f
        top = np.where(vis, np.abs(q[:, h]) @ np.abs(k).T * abs(f), 0).max(1)
        cap = a.get("softcap") or 0.0
        if cap:
            s = cap * np.tanh(s / cap)
        if a.get("rel") is not None:
            s = s + a["rel"][h].astype(np.float64)[np.clip(p - t, 0, a["rel"].shape[1] - 1)]
        s = np.where(vis, s, -np.inf)
        sink = float(a["sink"][h]) if a.get("sink") is not None else -np.inf
        m = np.maximum(s.max(1), sink)
        w = np.exp(s - np.where(np.isfinite(m), m, 0.0)[:, None])
        total = w.sum(1) + (np.exp(sink - m) if np.isfinite(sink) else 0.0)
        w = w / np.where(total > 0, total, 1)[:, None]
        o, size = w @ v, w @ np.abs(v)
        x = np.where(vis & np.isfinite(s), np.abs(s), 0).max(1) if a.get("rel") is None else np.full(n, 64.0)
        eps = top * (2.0 ** -22 + dim / 16 * 2.0 ** -22 + eps_more) + (1.45 * x + 16) * 2.0 ** -23 + cap * 2.0 ** -22 + 3 * 2.0 ** -22 + 128 * 2.0 ** -23 + eps_more
        largest = np.where(vis, np.abs(v).max(1)[None], 0).max(1) * w.max(1) * vis.sum(1)
        out[:, h] = o
        far[:, h] = eps[:, None] * (size + np.abs(o)) + (2.0 ** -28 * largest)[:, None]
    return out, far


def check(m, a, parts, dtype, seed=5, tiles=None, most=0, fp32_scores=False):
    """The rows of `parts` over m's cache: no number further off than its bound."""
    heads = a["heads"]
    assert tiles is None or T.takes_tiles(a, m, parts, dtype) == tiles
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = sum(x[2] for x in parts)
    q = torch.randn(n, heads * m.dim, device="cuda", generator=g)
    dev = lambda x: None if x is None else torch.from_numpy(np.ascontiguousarray(x, np.float32)).cuda()  # noqa: E731
    at = K.Attention(heads, m.H, m.dim, m.vdim, scale=a["scale"], chunk=a.get("chunk", 0), window=a.get("window", 0), keep_first=a.get("keep_first", 0), sink=dev(a.get("sink")),
                     head_scale=dev(a.get("head_scale")), softcap=a.get("softcap", 0.0), rel=dev(a.get("rel")), **({"fp32_scores": True} if fp32_scores else {}))
    rows = K.Rows.of(parts)
    rows.c.max_pos = max(rows.c.max_pos, most)                   # a step may be described by more than it has
    got = m.cache.attend(at, rows, q, layer=LAYER, dtype=dtype).double().cpu().numpy().reshape(n, heads, m.vdim)
    qn, row, worst = q.double().cpu().numpy().reshape(n, heads, m.dim), 0, 0.0
    for slot, p, c in parts:
        if p >= 0:
            want, far = expected(a, qn[row:row + c], m.values("k", slot, p + c), m.values("v", slot, p + c), p, 2.0 ** -11 if dtype == torch.bfloat16 and not fp32_scores else 0.0)
            far = far + np.abs(want) * (2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24) + 1e-44
            worst = max(worst, float((np.abs(got[row:row + c] - want) / far).max()))
        else:
            assert not got[row:row + c].any()
        row += c
    assert worst < 1.0
    return got


@pytest.mark.parametrize("case", T.LONG, ids=lambda c: f"{c[0]}-{c[1]}-{c[2]}-{c[3]}-{c[4]}-{c[5]}-{len(c[6])}")
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prompts(case, dtype):
    fmt, block, heads, kv_heads, dim, vdim, parts, mask = case
    m = T.filled(block, kv_heads, dim, vdim, fmt, [max(1, p + n) for _, p, n in parts])
    rng, a = np.random.default_rng(3), dict(mask, heads=heads, scale=dim ** -0.5)
    if a.get("sink"):
        a["sink"] = rng.standard_normal(heads).astype(np.float32)
    if a.get("rel"):
        a["rel"] = rng.standard_normal((heads, a["rel"])).astype(np.float32)
    check(m, a, parts, dtype, tiles=True)


@pytest.mark.parametrize("most", [0, 2111, 15999])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("parts", [[(0, 1400, 700)] + [(i, 19, 1) for i in range(1, 41)],
                                   [(i, 3, 1) for i in range(1, 20)] + [(0, 1200, 512), (41, 0, 30), (42, 50, 150), (43, 5, 8), (44, -1, 1), (45, 0, 260)] + [(i, 19, 1) for i in range(20, 41)]],
                         ids=["one prompt", "several portions"])
def test_prompts_beside_many_decoded_rows(parts, dtype, most):
    """... in a step whose contexts may be far longer than room for all of them would allow: the longest portions take tiles, the others the other form, and every row is right."""
    m = T.Mirror(1, 16, 32, 16, 128, 128, "int8", spare=400)
    m.table, at = np.full((46, 1000), -1, np.int32), 0
    for s, p, n in parts:
        if p >= 0:
            blocks = -(-(p + n) // 16)
            m.table[s, :blocks] = np.arange(at, at + blocks)[::-1]
            at += blocks
    c = m.cache
    m.cache = K.Kv8Cache(c.k_pool, c.v_pool, c.k_scale, c.v_scale, *(torch.zeros(46, T.LAYERS, 32, 16, 128, device="cuda") for _ in range(2)), torch.from_numpy(m.table).cuda())
    m.rows = [{x: np.zeros((0, 32, 128), np.float32) for x in "kv"} for _ in range(46)]
    parts_in = [(s, 0, p + n) for s, p, n in parts if p >= 0]
    n = sum(x[2] for x in parts_in)
    k, v = (torch.from_numpy(m.rng.standard_normal((n, 32 * 128)).astype(np.float32)).cuda() for _ in range(2))
    m.write(parts_in, k, v)
    check(m, dict(heads=32, scale=128 ** -0.5), parts, dtype, tiles=True, most=most)


@pytest.mark.parametrize("block,heads,kv_heads,dim,vdim,fmt", [(16, 4, 4, 64, 64, "int8"), (32, 8, 2, 128, 128, "e4m3"), (128, 20, 2, 96, 112, "int8")])
@pytest.mark.parametrize("parts", [T.SINGLES, T.PORTIONS], ids=["singles", "portions"])
@pytest.mark.parametrize("mask", [dict(), dict(window=33, keep_first=4), dict(chunk=50), dict(softcap=3.0)], ids=str)
def test_few_rows(block, heads, kv_heads, dim, vdim, fmt, parts, mask):
    m = T.filled(block, kv_heads, dim, vdim, fmt)
    check(m, dict(mask, heads=heads, scale=dim ** -0.5), parts, torch.float32)


def uneven(n, heads, dim, vdim, block, fmt, up, which):
    """A context whose value blocks `which(block number)` are 2^up larger than the others."""
    m = T.Mirror(1, n, heads, block, dim, vdim, fmt)
    k = torch.from_numpy(m.rng.standard_normal((n, heads * dim)).astype(np.float32)).cuda()
    v = m.rng.standard_normal((n, heads * vdim)).astype(np.float32)
    v *= np.where(which(np.arange(n) // block), np.float32(2.0 ** up), np.float32(1))[:, None]
    m.write([(0, 0, n)], k, torch.from_numpy(v).cuda())
    return m


HIDING = [(dict(), lambda b: b % 8 == 3), (dict(window=40), lambda b: b % 8 == 3), (dict(window=70, keep_first=5), lambda b: b % 16 == 5), (dict(chunk=48), lambda b: b % 3 == 2),
          (dict(chunk=64, window=30, keep_first=200), lambda b: b % 4 == 1), (dict(softcap=5.0, window=33), lambda b: b % 8 == 1)]


@pytest.mark.parametrize("mask,which", HIDING, ids=lambda x: str(x) if isinstance(x, dict) else "")
@pytest.mark.parametrize("up", [13, 26, 60])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,kv_heads,dim,fmt", [(32, 8, 128, "int8"), (64, 16, 64, "e4m3")])
def test_scales_of_keys_that_a_row_of_a_prompt_does_not_see(mask, which, up, dtype, heads, kv_heads, dim, fmt):
    """Blocks of values far larger than the others, ahead of a row's window or chunk or behind the row itself, while rows of the same tile see them: they cost the row no bit."""
    m = uneven(640, kv_heads, dim, dim, 16, fmt, up, which)
    check(m, dict(mask, heads=heads, scale=dim ** -0.5), [(0, 0, 640)], dtype, tiles=None if "window" in mask or "chunk" in mask else True)


@pytest.mark.parametrize("mask,which", HIDING, ids=lambda x: str(x) if isinstance(x, dict) else "")
@pytest.mark.parametrize("up", [13, 40, 70])
@pytest.mark.parametrize("parts", [[(0, p, 1) for p in (47, 80, 100, 127, 200, 255)], [(0, 30, 9), (0, 60, 40), (0, 120, 1)]], ids=["singles", "portions"])
@pytest.mark.parametrize("heads,kv_heads,dim,fmt", [(4, 2, 128, "e4m3"), (3, 3, 64, "int8")])
def test_scales_of_keys_that_one_of_few_rows_does_not_see(mask, which, up, parts, heads, kv_heads, dim, fmt):
    m = uneven(256, kv_heads, dim, dim, 16, fmt, up, which)
    check(m, dict(mask, heads=heads, scale=dim ** -0.5), parts, torch.float32)


@pytest.mark.parametrize("parts", [[(0, 599, 1)], [(0, 599, 1)] * 48, [(0, 560, 40)], [(0, 0, 600)]], ids=["single", "singles", "portion", "prompt"])
@pytest.mark.parametrize("up", [-112, -124, 100, 124])
def test_values_at_the_ends_of_fp32(parts, up):
    """Values of 2^-124 under the smallest scales keep their bits, and means of values of 2^126 are finite."""
    m = T.Mirror(1, 600, 4, 16, 128, 128, "int8")
    k, v = (torch.from_numpy(m.rng.standard_normal((600, 512)).astype(np.float32)).cuda() for _ in range(2))
    m.write([(0, 0, 600)], k, (1 + v.abs().clamp(max=4)) * 2.0 ** up)
    check(m, dict(heads=16, scale=128 ** -0.5), parts, torch.float32)


@pytest.mark.parametrize("up", [-124, 124])
def test_parts_of_a_prompts_context_at_the_ends_of_fp32(up):
    m = T.Mirror(1, 4000, 1, 16, 128, 128, "int8")
    k, v = (torch.from_numpy(m.rng.standard_normal((4000, 128)).astype(np.float32)).cuda() for _ in range(2))
    m.write([(0, 0, 4000)], k, (1 + v.abs().clamp(max=4)) * 2.0 ** up)
    check(m, dict(heads=8, scale=128 ** -0.5), [(0, 3700, 300)], torch.float32, tiles=True)


LOW = float(np.finfo(np.float32).min)


@pytest.mark.parametrize("parts", [[(0, 599, 1), (1, 3, 1)], [(0, 590, 10), (1, 0, 4)], [(0, 0, 600), (1, 0, 4)]], ids=["singles", "portions", "prompt"])
@pytest.mark.parametrize("softcap", [0.0, 30.0])
@pytest.mark.parametrize("sink", [False, True])
def test_biases_of_the_lowest_number(parts, softcap, sink):
    """A bias of the type's lowest number hides a key as long as another is seen; a row that has no other is a mean of what it sees, because the biases leave nothing of the scores.
    -inf hides a key for good."""
    m = T.filled(16, 4, 128, 128, "int8", (600, 4))
    rel = np.zeros((16, 600), np.float32)
    rel[0] = LOW
    rel[1, 3:] = LOW
    rel[2, :3] = LOW
    rel[3] = -np.inf
    rel[4, 1:] = -np.inf
    rel[5, :] = -np.inf
    rel[5, 7] = LOW
    rel[6, :] = LOW
    rel[6, 5] = 0.97 * LOW                                       # finite, below what log2(e) times it could be
    a = dict(heads=16, scale=128 ** -0.5, rel=rel, softcap=softcap)
    if sink:
        a["sink"] = np.random.default_rng(1).standard_normal(16).astype(np.float32)
    got = check(m, a, parts, torch.float32)
    assert not got[:, 3].any()
    if not sink:
        assert np.abs(got[:, 0]).max(1).min() > 0


def test_a_head_scale_that_is_not_a_number():
    """... shows in the results of its head, in every form."""
    m = T.filled(16, 4, 128, 128, "int8", (900,))
    hs = torch.ones(16, device="cuda")
    hs[5] = float("nan")
    for dtype in (torch.float32, torch.bfloat16):
        for parts, tiles in (([(0, 899, 1)], False), ([(0, 300, 600)], True)):
            assert T.takes_tiles(dict(heads=16, scale=0.1), m, parts, dtype) == tiles
            n = sum(p[2] for p in parts)
            out = m.cache.attend(K.Attention(16, 4, 128, scale=0.1, head_scale=hs), K.Rows.of(parts), torch.randn(n, 2048, device="cuda"), layer=LAYER, dtype=dtype).view(n, 16, 128)
            bad = torch.isnan(out)
            assert bool(bad[:, 5].all()) and not bool(bad[:, torch.arange(16) != 5].any())


def test_no_kernel_gave_up():
    """After a prompt: the question that a host asks behind its stream."""
    m = T.filled(16, 4, 128, 128, "int8", (900,))
    check(m, dict(heads=16, scale=0.1), [(0, 300, 600)], torch.float32, tiles=True)
    m.cache.check_error()


@pytest.mark.parametrize("heads,kv_heads,dim,vdim,fmt,mask", [(16, 4, 128, 128, "int8", dict()), (20, 4, 64, 48, "e4m3", dict(window=400, keep_first=4)), (12, 4, 112, 128, "e4m3", dict(softcap=5.0)),
                                                              (8, 8, 64, 64, "int8", dict())])
@pytest.mark.parametrize("parts", [[(0, 0, 700), (1, 0, 40), (2, 100, 1)], [(0, 2500, 200)]], ids=["prompt", "behind"])
def test_fp32_scores_with_bf16_results(heads, kv_heads, dim, vdim, fmt, mask, parts):
    """A caller that asks for fp32 scores gets the bounds of fp32 results and the last rounding, however long a portion is."""
    m = T.filled(16, kv_heads, dim, vdim, fmt, [p + n for _, p, n in parts])
    check(m, dict(mask, heads=heads, scale=dim ** -0.5), parts, torch.bfloat16, tiles=None if mask else True, fp32_scores=True)


@pytest.mark.parametrize("heads,kv_heads,dim,fmt,parts", [(16, 4, 128, "int8", [(0, 0, 1000)]), (16, 4, 128, "e4m3", [(0, 1500, 500)]), (32, 8, 64, "int8", [(0, 800, 700)])])
def test_bf16_results_of_prompts_are_little_more_than_their_rounding_off(heads, kv_heads, dim, fmt, parts):
    """For every row over its heads, and for every head over its rows.  A number rounded to fp16 is off by 2^-11 / 3^1/2 of it or, its place in the binade taken in, 2.0e-4 (rms).  A score is
    sum q k / dim^1/2 with q, k of order one: errors of q make 2.0e-4 of it; a weight's are as large, and results, sums of values that do not agree, are off by 2^1/2 times that of themselves,
    2.8e-4; 4.5e-4 is allowed beside the rounding itself, which is what it is for the exact result.  A row's 1024 values or more have an rms within 15 %, a head's within 5 %.  (Weights of
    three bits fewer: 1.6e-3 beside 1.65e-3.)"""
    m = T.filled(16, kv_heads, dim, dim, fmt, [p + n for _, p, n in parts])
    a, (slot, p, n) = dict(heads=heads, scale=dim ** -0.5), parts[0]
    got = check(m, a, parts, torch.bfloat16, tiles=True)
    q = torch.randn(n, heads * dim, device="cuda", generator=torch.Generator(device="cuda").manual_seed(5)).double().cpu().numpy().reshape(n, heads, dim)
    want, _ = expected(a, q, m.values("k", slot, p + n), m.values("v", slot, p + n), p)
    rounded = torch.from_numpy(want).to(torch.bfloat16).double().numpy()
    for axes, slack in (((1, 2), 1.15), ((0, 2), 1.05)):
        size = np.sqrt((want ** 2).mean(axes))
        off, least = np.sqrt(((got - want) ** 2).mean(axes)) / size, np.sqrt(((rounded - want) ** 2).mean(axes)) / size
        assert (off < slack * np.sqrt(least ** 2 + 4.5e-4 ** 2)).all()


def prompt_of(m, heads, parts, dtype, seed):
    """(call, result of an eager call) of a step over m's cache"""
    n = sum(x[2] for x in parts)
    at, rows = K.Attention(heads, m.H, m.dim, m.vdim, scale=m.dim ** -0.5), K.Rows.of(parts)
    q = torch.randn(n, heads * m.dim, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))
    return lambda: m.cache.attend(at, rows, q, layer=LAYER, dtype=dtype)


PROMPTS = [(16, [(0, 0, 700), (1, 290, 10), (2, 900, 1)], torch.bfloat16), (16, [(0, 300, 600), (2, 0, 900)], torch.float32), (32, [(1, 299, 1), (0, 899, 1)], torch.float32),
           (32, [(1, 0, 300)], torch.bfloat16)]


def test_prompts_captured_and_replayed():
    """Four steps, prompts, portions and single rows, each in a graph of its own: replayed in any order, with other calls between them, they give the eager calls' bits."""
    m = T.filled(16, 4, 128, 128, "int8", (900, 300, 901))
    calls = [prompt_of(m, h, parts, dt, i) for i, (h, parts, dt) in enumerate(PROMPTS)]
    want = [c().clone() for c in calls]
    torch.cuda.synchronize()
    graphs = []
    for c in calls:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = c()
        graphs.append((g, out))
    for order in ((0, 1, 2, 3), (3, 1, 1, 0), (2, 0, 3, 1)):
        for _, out in graphs:
            out.fill_(float("nan"))
        for i in order:
            graphs[i][0].replay()
            calls[3 - i]()
        torch.cuda.synchronize()
        for i in set(order):
            assert torch.equal(graphs[i][1], want[i]), i
    m.cache.check_error()


def test_prompts_side_by_side():
    """The same steps on four streams at once, again and again."""
    m = T.filled(16, 4, 128, 128, "int8", (900, 300, 901))
    calls = [prompt_of(m, h, parts, dt, i) for i, (h, parts, dt) in enumerate(PROMPTS)]
    want = [c().clone() for c in calls]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in calls], []
    for _ in range(15):
        for i, (s, c) in enumerate(zip(streams, calls)):
            with torch.cuda.stream(s):
                got.append((i, c()))
    torch.cuda.synchronize()
    assert all(torch.equal(out, want[i]) for i, out in got)
    m.cache.check_error()


def test_threads_with_layers_of_their_own():
    """Two threads, one attention, two layers: each gets its layer's rows."""
    import threading
    c = K.Kv8Cache.empty(blocks=40, layers=3, kv_heads=2, block_size=16, dim=64, slots=1, table_stride=40)
    c.table.copy_(torch.arange(40, dtype=torch.int32)[None])
    rows, at, q = K.Rows.of([(0, 0, 300)]), K.Attention(8, 2, 64, scale=0.125), torch.randn(1, 512, device="cuda")
    for layer in range(3):
        c.write(rows, *(torch.randn(300, 128, device="cuda") for _ in "kv"), layer=layer)
    one = K.Rows.of([(0, 299, 1)])
    want = [c.attend(at, one, q, layer=layer) for layer in range(3)]
    torch.cuda.synchronize()
    bad = []

    def work(layer):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(200):
                if not torch.equal(c.attend(at, one, q, layer=layer), want[layer]):
                    bad.append(layer)

    threads = [threading.Thread(target=work, args=(layer,)) for layer in (0, 1, 2, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(120)
    assert not bad


@pytest.mark.parametrize("heads,kv_heads", [(130, 1), (384, 2), (1, 1), (7, 7)])
@pytest.mark.parametrize("parts", [[(0, 199, 1), (1, 0, 1)], [(0, 50, 90), (1, 0, 1)]], ids=["singles", "portion"])
def test_unusual_numbers_of_heads(heads, kv_heads, parts):
    m = T.filled(16, kv_heads, 64, 128, "int8", (200, 1))
    for dtype in (torch.float32, torch.bfloat16):
        check(m, dict(heads=heads, scale=0.125), parts, dtype)


@pytest.mark.parametrize("parts", [[(i, 40 * i + 7, 1) for i in range(6)], [(0, 3, 30), (1, 0, 5), (2, 100, 1)], [(0, 0, 400), (1, 0, 400), (2, 390, 7)]], ids=["singles", "portions", "prompts"])
@pytest.mark.parametrize("fmt,dtype", [("int8", torch.float32), ("e4m3", torch.bfloat16)])
def test_steps_described_by_more_than_they_have(parts, fmt, dtype):
    """A longest portion and a largest position beyond the step's own, as a captured step whose rows change has them: written, read and attended to alike."""
    n, got = sum(x[2] for x in parts), []
    g = torch.Generator(device="cuda").manual_seed(0)
    k, v, q = (torch.randn(n, w, device="cuda", generator=g) for w in (128, 256, 512))
    for more in (False, True):
        big = K.Kv8Cache.empty(blocks=200, layers=T.LAYERS, kv_heads=2, block_size=32, dim=64, vdim=128, slots=len(parts), table_stride=30, dtype=T.DT[fmt])
        big.table.copy_(torch.arange(30 * len(parts), dtype=torch.int32).view(len(parts), 30))
        first = [(s, 0, p) for s, p, _ in parts if p]
        if first:
            gen = torch.Generator(device="cuda").manual_seed(1)
            total = sum(x[2] for x in first)
            big.write(K.Rows.of(first), *(torch.randn(total, w, device="cuda", generator=gen) for w in (128, 256)), layer=LAYER)
        rows = K.Rows.of(parts)
        if more:
            rows.c.max_seq_rows, rows.c.max_pos = n, 900
        big.write(rows, k, v, layer=LAYER)
        back = big.read(rows, layer=LAYER, dtype=dtype)
        got.append((*back, big.k_scale, big.v_scale, big.k_open, big.attend(K.Attention(8, 2, 64, 128, scale=0.125), rows, q, layer=LAYER, dtype=dtype)))
    for x, y in list(zip(*got))[:5]:
        assert torch.equal(x, y)
    a, b = got[0][5].double(), got[1][5].double()              # the form may differ
    assert float((a - b).norm() / a.norm()) < (2e-5 if dtype == torch.float32 else 2.0 ** -7)
