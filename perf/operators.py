"""The key/value cache in 8 bits: what writes it, what reads it back and the attention over it, on calls that a serving loop makes.

Every value x of a block of tokens and a key/value head is kept as one byte, round(x / s), under one scale s = max|x| / M of the whole
block and head (M: the format's largest number, 127 or 448).  Rows of a slot's last block, while it is not full, are kept in fp32 beside it, so that a block's
codes are always one rounding of its rows.

  write   rows of several sequences enter the cache and are read back as the values they stand for
  read    rows of cached contexts as plain rows
  attend  softmax attention of rows over the cache: single tokens behind their contexts, or portions of prompts

With `own` the calls go to the framework (hip_llama.cpp_b200/kv8.py); without it they are plain torch.
"""
import importlib
import importlib.util
import math
import os
import sys

import numpy as np
import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LAYERS, LAYER = 2, 1                                     # the pools hold two cache layers, the calls are for the second
MOST = {"int8": 127.0, "e4m3": 448.0}
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
TINY = 2.0 ** -126


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
SMALL = dict(heads=12, kv_heads=12, dim=64, vdim=64)     # stories110M
WIDE = dict(heads=32, kv_heads=32, dim=128, vdim=128)    # Llama-2-7B
GROUPED = dict(heads=32, kv_heads=8, dim=128, vdim=128)  # the same with grouped queries
SERVED = dict(heads=16, kv_heads=4, dim=128, vdim=128)   # the layer-program designs at width 2048
MASKS = dict(window=0, keep=0, chunk=0, sink=False, cap=0.0, rel=0)


def _case(name, kind, shape, **more):
    """p0 .. p1: positions of the sequences' first rows, n0 .. n1: their rows, from the first sequence to the last (in a shuffled order)."""
    return dict(shape, name=name, kind=kind, **dict(MASKS, **more))


def listed():
    return [
        # one user's chat loop on the small model: one token enters the cache
        _case("write 1 token small", "write", SMALL, format="int8", dtype="f32", block=16, seqs=1, p0=211, p1=211, n0=1, n1=1),
        # a batch of decoded tokens at positions of their own
        _case("write 64 tokens e4m3", "write", GROUPED, format="e4m3", dtype="bf16", block=32, seqs=64, p0=3, p1=2030, n0=1, n1=1),
        # prompts of the large model enter, two of them behind an earlier portion
        _case("write 3 prompts", "write", WIDE, format="int8", dtype="f32", block=16, seqs=3, p0=0, p1=530, n0=37, n1=2048),
        # the first rows of one context are handed to an operator that takes plain rows
        _case("read 700 rows", "read", SERVED, format="int8", dtype="f32", block=64, seqs=1, p0=0, p1=0, n0=700, n1=700),
        # a batch of contexts is handed over
        _case("read 8 contexts e4m3", "read", WIDE, format="e4m3", dtype="bf16", block=16, seqs=8, p0=0, p1=77, n0=301, n1=2048),
        # one user's chat loop on the small model: one token behind a short context
        _case("attend 1 token small", "attend", SMALL, format="int8", dtype="f32", block=16, seqs=1, p0=211, p1=211, n0=1, n1=1),
        # a full batch of the large model, contexts of all lengths
        _case("attend 64 tokens 7B", "attend", WIDE, format="int8", dtype="f32", block=16, seqs=64, p0=3, p1=2047, n0=1, n1=1),
        # long contexts with grouped queries
        _case("attend 16 tokens grouped e4m3", "attend", GROUPED, format="e4m3", dtype="bf16", block=32, seqs=16, p0=501, p1=8190, n0=1, n1=1),
        # one user behind a very long document
        _case("attend 1 token at 131071", "attend", GROUPED, format="int8", dtype="bf16", block=64, seqs=1, p0=131070, p1=131070, n0=1, n1=1),
        # a prompt in full precision
        _case("attend prompt 7B f32", "attend", WIDE, format="int8", dtype="f32", block=16, seqs=1, p0=0, p1=0, n0=1024, n1=1024),
        # two prompts in bf16: what decides the time to the first token
        _case("attend 2 prompts 7B bf16", "attend", WIDE, format="int8", dtype="bf16", block=16, seqs=2, p0=0, p1=0, n0=777, n1=2048),
        # a portion of a long prompt under a window with kept first tokens and a sink
        _case("attend portion behind 16384", "attend", SERVED, format="e4m3", dtype="bf16", block=64, seqs=1, p0=16384, p1=16384, n0=509, n1=509,
              window=8192, keep=64, sink=True),
    ]


def _log_between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["write", "read", "attend", "attend", "attend", "attend"])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 12, 32])
    group = rng.choice([1, 1, 2, 4, 5, 8, 16]) if kv_heads <= 4 else rng.choice([1, 2, 4]) if kv_heads <= 12 else 1
    dim = rng.choice([64, 128, 128, 16 * rng.randint(2, 8)])
    vdim = dim if rng.random() < 0.75 else 16 * rng.randint(2, 8)
    c = dict(kind=kind, heads=kv_heads * group, kv_heads=kv_heads, dim=dim, vdim=vdim, format=rng.choice(["int8", "int8", "e4m3"]), dtype=rng.choice(["f32", "bf16"]),
             block=rng.choice([16, 16, 32, 64, 128]), **MASKS)
    if kind != "attend":
        n = 1 if kind == "write" and rng.random() < 0.4 else _log_between(rng, 2, 2048)
        seqs = min(_log_between(rng, 1, 96), max(1, 3100 // n))
        p0 = rng.choice([0, rng.randint(0, 700)])
        return dict(c, seqs=seqs, p0=p0, p1=p0 + rng.randint(0, 300), n0=max(1, int(n * rng.uniform(0.1, 1.0))), n1=n)
    if rng.random() < 0.55:                              # single tokens: bytes of the caches decide
        last = _log_between(rng, 1, 60000)
        most = int(5.0e8 / (kv_heads * (dim + vdim) * (last + 1)))
        seqs = max(1, min(_log_between(rng, 1, 128), most))
        if most < 1:
            last = int(5.0e8 / (kv_heads * (dim + vdim)))
        c.update(seqs=seqs, p0=int(last * rng.uniform(0.0, 1.0)), p1=last, n0=1, n1=1)
    else:                                                # portions: products decide
        n = _log_between(rng, 2, 2048)
        seqs = rng.choice([1, 1, 2, 3, 5])
        p = rng.choice([0, 0, _log_between(rng, 1, 8000)])
        while seqs * n * (n + 2 * p) * c["heads"] * max(128, dim + vdim) > 3.5e10:
            n, p, seqs = max(2, n * 3 // 4), p * 3 // 4, max(1, seqs - 1)
        c.update(seqs=seqs, p0=int(p * rng.uniform(0.0, 1.0)), p1=p, n0=max(1, int(n * rng.uniform(0.1, 1.0))), n1=n)
    if rng.random() < 0.3:
        c.update(window=_log_between(rng, 1, 4000), keep=rng.choice([0, 4, 70]))
    elif rng.random() < 0.1:
        c["chunk"] = _log_between(rng, 16, 4096)
    c["sink"] = rng.random() < 0.25
    if rng.random() < 0.12:
        c["cap"] = rng.choice([20.0, 50.0])
    elif rng.random() < 0.08 and c["seqs"] * c["n1"] * (c["p1"] + c["n1"]) * c["heads"] < 2e8:
        c["rel"] = rng.randint(1, 200)
    return c


def _portions(case):
    """[(slot, first position, rows)]"""
    s = case["seqs"]
    at = np.random.default_rng(s).permutation(s)
    spread = lambda lo, hi: [lo + (hi - lo) * i // max(1, s - 1) for i in range(s)]  # noqa: E731
    p, n = spread(case["p0"], case["p1"]), spread(case["n0"], case["n1"])
    if s == 1:
        p, n = [case["p1"]], [case["n1"]]
    return [(s - 1 - i, p[at[i]], n[at[-1 - i]]) for i in range(s)]


def _first_seen(case, p):
    """Keys 0 .. p that a query at p does not see are those from `keep` (or the chunk's start) to below this one."""
    lo = p // case["chunk"] * case["chunk"] if case["chunk"] else 0
    return max(lo, p - case["window"] + 1) if case["window"] else lo


def work(case):
    H, D, E = case["kv_heads"], case["dim"], case["vdim"]
    size = 4 if case["dtype"] == "f32" else 2
    parts = _portions(case)
    rows = sum(n for _, _, n in parts)
    blocks = sum((p + n - 1) // case["block"] - p // case["block"] + 1 for _, p, n in parts)
    if case["kind"] != "attend":
        read_back = 4 if case["kind"] == "write" else size
        taken = rows * H * (D + E) * size if case["kind"] == "write" else 0
        return {"bytes": taken + rows * H * (D + E) * (1 + read_back) + 8 * blocks * H, "flops": 2 * rows * H * (D + E)}
    keys = pairs = 0
    for _, p, n in parts:
        seen = np.arange(p, p + n)
        lo = np.array([_first_seen(case, t) for t in (p, p + n - 1)])
        every = np.array([_first_seen(case, int(t)) for t in seen])
        kept = np.minimum(every, case["keep"]) if case["window"] else 0 * every
        kept = np.where(case["chunk"] > 0, 0, kept) if case["chunk"] else kept
        pairs += int((seen - every + 1 + kept).sum())
        keys += p + n - int(lo[0]) + (min(int(lo[0]), case["keep"]) if case["window"] else 0)
    heads = case["heads"]
    return {"bytes": keys * H * (D + E) + 8 * H * -(-keys // case["block"]) + rows * heads * (4 * D + size * E), "flops": 2 * pairs * heads * (D + E)}


# ---- inputs ---------------------------------------------------------------------------------------------------------------
def _round_e4m3(y):
    """Nearest multiple of the step of |y|'s binade (ties to even), y in fp64 and inside the format's range."""
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
    return (torch.round(y / step) * step).clamp(-448, 448)


def _quantise(x, fmt):
    """x [.., head, position, channel] -> (codes as bytes, scales [.., head]); the quotients in fp64, where none falls on the wrong side of a border."""
    top = x.float().abs().amax((-1, -2))
    scale = torch.where(top > 0, (top.double() / MOST[fmt]).float().clamp_min(TINY), torch.zeros_like(top))
    y = x.double() / torch.where(scale > 0, scale, torch.ones_like(scale)).double()[..., None, None]
    if fmt == "int8":
        return torch.round(y).clamp(-127, 127).to(torch.int8), scale
    return _round_e4m3(y).float().to(torch.float8_e4m3fn).view(torch.int8), scale


def _numbers(codes, fmt):
    return codes.float() if fmt == "int8" else codes.view(torch.float8_e4m3fn).float()


def _channels(g, heads, width, device):
    """What distinguishes channels of real keys: a few are several times larger than the others."""
    return torch.exp(0.6 * torch.randn(heads, 1, width, device=device, generator=g))


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    H, B, fmt = case["kv_heads"], case["block"], case["format"]
    parts = _portions(case)
    S, R = len(parts), sum(n for _, _, n in parts)
    per = max(-(-(p + n) // B) for _, p, n in parts) + 1
    used = [-(-(p + n) // B) for _, p, n in parts]
    total = sum(used) + 1                                # block 0 is nobody's
    ids = np.random.default_rng(int(seed)).permutation(np.arange(1, total))
    table = np.zeros((S, per), np.int32)
    at = 0
    for (slot, _, _), u in zip(parts, used):
        table[slot, :u] = ids[at:at + u]
        at += u
    s = {"case": case, "parts": parts}
    put = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(dev)  # noqa: E731
    first = np.cumsum([0] + [n for _, _, n in parts])
    pos = np.concatenate([np.arange(p, p + n) for _, p, n in parts])
    s["pos"], s["row_seq"], s["seq_first"], s["seq_slot"] = put(pos), put(np.repeat(np.arange(S), np.diff(first))), put(first), put([x[0] for x in parts])
    s["max_seq_rows"], s["max_pos"], s["table"] = int(max(n for _, _, n in parts)), int(pos.max()), put(table)

    # the cache: quantised contexts, and the fp32 rows of the slots' last blocks (behind the context that a write finds)
    behind = {slot: p if case["kind"] == "write" else p + n for slot, p, n in parts}
    for side, width in (("k", case["dim"]), ("v", case["vdim"])):
        chan = _channels(g, H, width, dev)
        codes = torch.zeros(total, LAYERS, H, B, width, dtype=torch.int8, device=dev)
        scales = torch.zeros(total, LAYERS, H, device=dev)
        open_ = torch.zeros(S, LAYERS, H, B, width, device=dev)
        step = max(1, (1 << 25) // (H * B * width))
        for b in range(0, total, step):
            m = min(step, total - b)
            x = torch.randn(m, H, B, width, device=dev, generator=g) * chan * torch.exp(0.3 * torch.randn(m, H, 1, 1, device=dev, generator=g))
            codes[b:b + m, LAYER], scales[b:b + m, LAYER] = _quantise(x, fmt)
        slots = torch.tensor(sorted(behind), device=dev)
        filled = torch.tensor([behind[t] % B for t in sorted(behind)], device=dev)
        blocks = torch.tensor([int(table[t, behind[t] // B]) if behind[t] % B else 0 for t in sorted(behind)], device=dev)
        x = torch.randn(S, H, B, width, device=dev, generator=g) * chan
        x = x * (torch.arange(B, device=dev)[None, :] < filled[:, None])[:, None, :, None]
        open_[slots, LAYER] = x
        c, f = _quantise(x, fmt)
        some = blocks > 0
        codes[blocks[some], LAYER], scales[blocks[some], LAYER] = c[some], f[some]
        s[side + "_codes"], s[side + "_scale"], s[side + "_open"] = codes, scales, open_
        if case["kind"] == "write":
            wide = torch.randn(R, H * width + 16, device=dev, generator=g) * torch.nn.functional.pad(chan.reshape(-1), (0, 16), value=1.0)
            s[side] = wide.to(TYPES[case["dtype"]])[:, :H * width]     # columns of a wider product
    if case["kind"] == "attend":
        s["q"] = torch.randn(R, case["heads"] * case["dim"], device=dev, generator=g)
        s["scale"] = case["dim"] ** -0.5
        s["sink"] = torch.randn(case["heads"], device=dev, generator=g) if case["sink"] else None
        s["rel"] = torch.randn(case["heads"], case["rel"], device=dev, generator=g) if case["rel"] else None
    if case["kind"] == "write":
        # where every row of every touched block comes from: a row of the call, a row of the slot's last block, or nothing
        src, blk, slot_of, keeps = [], [], [], []
        none = R + S * B
        for i, (slot, p, n) in enumerate(parts):
            for b in range(p // B, (p + n - 1) // B + 1):
                t = b * B + np.arange(B)
                src.append(np.where(t < p, R + slot * B + np.arange(B), np.where(t < p + n, first[i] + t - p, none)))
                blk.append(table[slot, b])
                slot_of.append(slot)
                keeps.append(b == (p + n) // B)
        put64 = lambda a: torch.from_numpy(np.asarray(a, np.int64)).to(dev)  # noqa: E731
        keeps = np.flatnonzero(keeps)
        s["src"], s["blk"], s["kept"], s["kept_slot"] = put64(np.stack(src)), put64(blk), put64(keeps), put64(np.asarray(slot_of)[keeps])
    else:
        # padded portions: row of (sequence, i), and where each row is
        most = s["max_seq_rows"]
        pad = first[:-1, None] + np.arange(most)[None]
        there = np.arange(most)[None] < np.diff(first)[:, None]
        s["pad"] = torch.from_numpy(np.where(there, pad, 0)).to(dev)
        s["p"] = torch.from_numpy(np.array([p for _, p, _ in parts])[:, None] + np.where(there, np.arange(most)[None], 0)).to(dev)
        s["flat"] = torch.from_numpy(np.flatnonzero(there)).to(dev)
        s["pages"] = torch.from_numpy(np.stack([table[slot] for slot, _, _ in parts]).astype(np.int64)).to(dev)
    return s


# ---- plain forms ----------------------------------------------------------------------------------------------------------
def _rows_of(s, side, dtype):
    """The call's rows as the values they stand for, [rows, heads * width]."""
    case, pos, slot = s["case"], s["pos"].long(), s["seq_slot"].long()[s["row_seq"].long()]
    blk = s["table"][slot, pos // case["block"]].long()
    x = _numbers(s[side + "_codes"][blk, LAYER, :, pos % case["block"]], case["format"]) * s[side + "_scale"][blk, LAYER][..., None]
    return x.to(dtype).flatten(1)


def _plain_write(s):
    case = s["case"]
    for side in ("k", "v"):
        H, open_ = case["kv_heads"], s[side + "_open"]
        rows = s[side].float().unflatten(1, (H, -1))
        every = torch.cat([rows, open_[:, LAYER].transpose(1, 2).flatten(0, 1), torch.zeros_like(rows[:1])])
        x = every[s["src"]].transpose(1, 2)              # [block, head, position, channel]
        codes, scale = _quantise(x, case["format"])
        s[side + "_codes"][s["blk"], LAYER] = codes
        s[side + "_scale"][s["blk"], LAYER] = scale
        new = (s["src"][s["kept"]] < rows.shape[0])[:, None, :, None]
        open_[s["kept_slot"], LAYER] = torch.where(new, x[s["kept"]], open_[s["kept_slot"], LAYER])


def _visible(case, p, t):
    see = t <= p
    if case["chunk"]:
        see = see & (t >= p // case["chunk"] * case["chunk"])
    if case["window"]:
        see = see & ((p - t < case["window"]) | (t < case["keep"]))
    return see


def _plain_attend(s):
    case = s["case"]
    H, D, E, fmt = case["kv_heads"], case["dim"], case["vdim"], case["format"]
    G = case["heads"] // H
    K, V = ((_numbers(s[x + "_codes"][s["pages"], LAYER], fmt) * s[x + "_scale"][s["pages"], LAYER][..., None, None]).transpose(1, 2).flatten(2, 3) for x in ("k", "v"))
    q = s["q"][s["pad"]].unflatten(-1, (H, G, D)).permute(0, 2, 3, 1, 4)                  # [sequence, kv head, group, row, channel]
    x = (q.flatten(2, 3) @ K.transpose(-1, -2)).unflatten(2, (G, -1)) * s["scale"]        # [.., group, row, key]
    if case["cap"]:
        x = case["cap"] * torch.tanh(x / case["cap"])
    t, p = torch.arange(K.shape[2], device=q.device), s["p"][:, None, None, :, None]
    if s["rel"] is not None:
        back = (p - t).clamp(0, case["rel"] - 1)
        x = x + s["rel"][:, back[:, 0, 0]].transpose(0, 1).unflatten(1, (H, G))
    x = x.masked_fill(~_visible(case, p, t), float("-inf"))
    top = x.amax(-1, keepdim=True)
    if s["sink"] is not None:
        top = torch.maximum(top, s["sink"].view(1, H, G, 1, 1))
    w = torch.exp(x - top)
    total = w.sum(-1, keepdim=True)
    if s["sink"] is not None:
        total = total + torch.exp(s["sink"].view(1, H, G, 1, 1) - top)
    o = ((w.flatten(2, 3) @ V).unflatten(2, (G, -1)) / total).permute(0, 3, 1, 2, 4).flatten(0, 1)[s["flat"]]
    return o.flatten(1).to(TYPES[case["dtype"]])


# ---- the framework's calls ------------------------------------------------------------------------------------------------
def _bind(s):
    """What a serving program keeps beside its cache: the handle of the pools, the description of the step's rows, the layer's attention."""
    kv8, case = _package("kv8"), s["case"]
    kind = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}[case["format"]]
    s["cache"] = kv8.Kv8Cache(s["k_codes"].view(kind), s["v_codes"].view(kind), s["k_scale"], s["v_scale"], s["k_open"], s["v_open"], s["table"])
    s["rows"] = kv8.Rows(s["pos"], s["row_seq"], s["seq_first"], s["seq_slot"], s["max_seq_rows"], s["max_pos"])
    if case["kind"] == "attend":
        s["attn"] = kv8.Attention(case["heads"], case["kv_heads"], case["dim"], case["vdim"], scale=s["scale"], chunk=case["chunk"], window=case["window"],
                                  keep_first=case["keep"], sink=s["sink"], softcap=case["cap"], rel=s["rel"])


def run(state):
    s, case = state, state["case"]
    if own:
        if "cache" not in s:
            _bind(s)
        if case["kind"] == "attend":
            return s["cache"].attend(s["attn"], s["rows"], s["q"], layer=LAYER, dtype=TYPES[case["dtype"]])
        if case["kind"] == "read":
            return s["cache"].read(s["rows"], layer=LAYER, dtype=TYPES[case["dtype"]])
        s["cache"].write(s["rows"], s["k"], s["v"], layer=LAYER)
        back = s["cache"].read(s["rows"], layer=LAYER, dtype=torch.float32)
    elif case["kind"] == "attend":
        return _plain_attend(s)
    elif case["kind"] == "read":
        return tuple(_rows_of(s, x, TYPES[case["dtype"]]) for x in ("k", "v"))
    else:
        _plain_write(s)
        back = tuple(_rows_of(s, x, torch.float32) for x in ("k", "v"))
    return {"k": back[0], "v": back[1], **{n: s[n] for n in ("k_scale", "v_scale", "k_open", "v_open")}}


# ---- from the definitions, in 64 bits -------------------------------------------------------------------------------------
def _levels(fmt):
    """The format's numbers from 0 up, and the borders between them."""
    if fmt == "int8":
        v = torch.arange(128, dtype=torch.float64)
    else:
        v = torch.tensor([(m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)) for e in range(16) for m in range(8)][:127], dtype=torch.float64)
    return v.cuda(), ((v[1:] + v[:-1]) / 2).cuda()


def _nearest(x, scale, fmt):
    """The format's number nearest to x / scale: a border belongs to the even one of its neighbours."""
    v, edge = _levels(fmt)
    y = torch.where(scale > 0, x / scale, 0.0)
    a = y.abs().clamp(max=float(v[-1]))
    i = torch.searchsorted(edge, a.contiguous())         # borders below a
    i = i + ((i < len(edge)) & (edge[i.clamp(max=len(edge) - 1)] == a) & (i % 2 == 1)).long()
    return torch.copysign(v[i], y)


def exact(case, seed):
    s = prepare(case, seed)
    H, B, fmt, G = case["kv_heads"], case["block"], case["format"], case["heads"] // case["kv_heads"]
    table = s["table"].cpu().numpy()

    def stored(side, slot, count):
        """Rows 0 .. count - 1 of a slot, [heads, count, width]"""
        ids = torch.from_numpy(table[slot, :-(-count // B)].astype(np.int64)).cuda()
        c = s[side + "_codes"][ids, LAYER]
        c = c.double() if fmt == "int8" else c.view(torch.float8_e4m3fn).double()
        return (c * s[side + "_scale"][ids, LAYER].double()[:, :, None, None]).permute(1, 0, 2, 3).flatten(1, 2)[:, :count]

    if case["kind"] == "read":
        return tuple(torch.cat([stored(x, slot, p + n)[:, p:].transpose(0, 1).flatten(1) for slot, p, n in s["parts"]]) for x in ("k", "v"))
    if case["kind"] == "write":
        out, at = {}, 0
        for side in ("k", "v"):
            scales, open_ = s[side + "_scale"].double(), s[side + "_open"].double()
            back, at = [], 0
            for slot, p, n in s["parts"]:
                new = s[side][at:at + n].double().unflatten(1, (H, -1)).transpose(0, 1)
                at += n
                lead = p % B
                x = torch.cat([open_[slot, LAYER, :, :lead], new], 1)
                x = torch.nn.functional.pad(x, (0, 0, 0, -x.shape[1] % B)).unflatten(1, (-1, B))       # [head, block, position, channel]
                top = x.abs().amax((-1, -2))
                f = torch.where(top > 0, (top / MOST[fmt]).float().clamp_min(TINY).double(), 0.0)
                back.append((_nearest(x, f[..., None, None], fmt) * f[..., None, None]).flatten(1, 2)[:, lead:lead + n].transpose(0, 1).flatten(1))
                ids = torch.from_numpy(table[slot, p // B:p // B + x.shape[1]].astype(np.int64)).cuda()
                scales[ids, LAYER] = f.T
                rest = (p + n) % B
                if rest:
                    fresh = min(rest, n)
                    open_[slot, LAYER, :, rest - fresh:rest] = new[:, n - fresh:]
            out[side], out[side + "_scale"], out[side + "_open"] = torch.cat(back), scales, open_
        return out
    out, at = [], 0
    for slot, p, n in s["parts"]:
        K, V = stored("k", slot, p + n), stored("v", slot, p + n)
        q = s["q"][at:at + n].double().unflatten(1, (H, G, -1)).permute(1, 2, 0, 3)
        at += n
        t, rows = torch.arange(p + n, device="cuda"), torch.arange(p, p + n, device="cuda")[:, None]
        hidden = t > rows
        if case["chunk"]:
            hidden = hidden | (t < rows - rows % case["chunk"])
        if case["window"]:
            hidden = hidden | ((rows - t >= case["window"]) & (t >= case["keep"]))
        got = []
        for h in range(H):
            x = torch.einsum("gnd,td->gnt", q[h], K[h]) * s["scale"]
            if case["cap"]:
                x = case["cap"] * torch.tanh(x / case["cap"])
            if s["rel"] is not None:
                x = x + s["rel"].double()[h * G:(h + 1) * G][:, (rows - t).clamp(0, case["rel"] - 1)]
            x = x.masked_fill(hidden, float("-inf"))
            if s["sink"] is not None:
                x = torch.cat([x, s["sink"].double()[h * G:(h + 1) * G, None, None].expand(-1, n, 1)], -1)
            w = torch.softmax(x, -1)[..., :p + n]
            got.append(torch.einsum("gnt,te->nge", w, V[h]))
        out.append(torch.stack(got, 1).flatten(1))
    return torch.cat(out)
