"""What the binding of the cache in 8 bits hands to the library, with a recorder in the library's place: no GPU."""
import os
import re
import threading
import types

import pytest
import torch

from pkgload import load_pkg

K = load_pkg("kv8")


def recorded(monkeypatch, **calls):
    """A cache on the CPU whose calls go to `calls`."""
    cache = K.Kv8Cache.empty(blocks=4, layers=3, kv_heads=2, block_size=16, dim=32, slots=2, table_stride=2, device="cpu")
    monkeypatch.setattr(cache, "_stream", lambda rows: 0)
    cache.calls = types.SimpleNamespace(**calls)
    return cache


@pytest.mark.parametrize("layers", [(0, 1), (2, 0), (1, 1)])
def test_threads_share_an_attention(monkeypatch, layers):
    """The library lets go of the interpreter in every call: both threads are in their first call before either makes its second."""
    both, seen = threading.Barrier(2, timeout=30), {}

    def scratch(kind, a, rows, kv):
        both.wait()
        seen.setdefault(threading.get_ident(), []).append(a._obj.cache_layer)
        return 0

    def attn(stream, kind, a, rows, kv, *rest):
        both.wait()
        seen[threading.get_ident()].append(a._obj.cache_layer)
        return 0

    cache = recorded(monkeypatch, tha_hyb_kv8_attn_scratch=scratch, tha_hyb_kv8_attn=attn)
    at, rows, q = K.Attention(4, 2, 32, scale=1.0), K.Rows.of([(0, 0, 1)], "cpu"), torch.zeros(1, 128)
    want = {}

    def work(layer):
        want[threading.get_ident()] = [layer] * 6
        for _ in range(3):
            cache.attend(at, rows, q, layer=layer)

    threads = [threading.Thread(target=work, args=(layer,)) for layer in layers]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert seen == want


def test_changes_of_an_attention_reach_the_next_call():
    at = K.Attention(4, 2, 32, scale=1.0)
    first = at.of(1)
    assert first is at.of(1) and first._obj.cache_layer == 1 and at.of(0)._obj.cache_layer == 0 and at.c.cache_layer == 0
    at.c.window = 7
    assert at.of(1)._obj.window == 7 and at.of(0)._obj.window == 7 and first._obj.window == 0


def test_a_kernel_that_gave_up_is_an_error(monkeypatch):
    answers = [0, 1, 0]
    cache = recorded(monkeypatch, tha_gemm_check_error=lambda: answers.pop(0))
    cache.check_error()
    with pytest.raises(K.cabi.ThaError):
        cache.check_error()
    cache.check_error()


def test_a_wait_that_gives_up_shows_in_its_rows():
    """No wait of the prompt kernel runs out in a sound pipeline, so this is read from its source: the outcome of a row's waits goes into its sum as NaN ahead of its two threads joining their
    sums, from which maximum, factor and partial results follow; and no store of a result is left out where a wait gave up."""
    src = os.path.join(os.path.dirname(K.__file__), "csrc", "kv8_attn_tc.cu")
    text = re.sub(r"//[^\n]*", "", open(src).read())
    kernel = text[text.index("kv8_attn_tc_kernel(tha_attn_t a"):]
    softmax = kernel[kernel.index("if (warp < KT_SOFTMAX) {"):kernel.index("else if (warp == KT_LOAD)")]
    waits = [m.start() for m in re.finditer(r"tc_mbar_wait", softmax)]
    gave_up, joined = softmax.index("if (!ok) l = NAN;"), softmax.index("l = both(l,")
    assert len(waits) >= 4 and max(waits) < gave_up < joined < softmax.index("if (l != l) m = l;") < softmax.index("k8_final(")
    assert all("ok" in softmax[softmax.rindex("\n", 0, w):softmax.index("\n", w)] for w in waits)
    assert not re.search(r"if \([^)]*\bok\b[^)]*\)", softmax[joined:])


def test_open_end_is_refused_where_it_does_not_fit():
    good = K.Kv8Cache.empty(blocks=4, layers=3, kv_heads=2, block_size=16, dim=32, slots=2, table_stride=2, device="cpu")
    assert bool((good.open_end == -1).all()) and good.c.open_end == good.open_end.data_ptr()
    parts = (good.k_pool, good.v_pool, good.k_scale, good.v_scale, good.k_open, good.v_open, good.table)
    assert K.Kv8Cache(*parts).c.open_end is None
    assert K.Kv8Cache(*parts, torch.zeros(2 * 3 * 2 * 2, dtype=torch.int32)).open_end is not None
    for bad in (torch.zeros(2, 3, 2, 2), torch.zeros(2, 3, 2, dtype=torch.int32), torch.zeros(2, 3, 2, 4, dtype=torch.int32)[..., ::2]):
        with pytest.raises(ValueError):
            K.Kv8Cache(*parts, bad)
