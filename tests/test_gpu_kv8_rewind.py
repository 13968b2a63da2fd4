"""Tokens dropped from the end of a slot of the cache in 8 bits, across borders of blocks too: what is written next, against the definition to the bit.  Rows of a block that the open rows
no longer hold are the values that their codes stand for, code * scale in fp32."""
import numpy as np
import pytest
import torch

import kv8_oracle as O
import test_gpu_kv8 as T

pytestmark = pytest.mark.gpu
K, LAYER = T.K, T.LAYER


class Rewound(T.Mirror):
    """A mirror whose portions may begin anywhere.  held[slot]: behind which position the slot's open rows end."""

    def __init__(self, *a, **kw):
        super().__init__(*a, **kw)
        self.held = [0] * len(self.rows)

    def write(self, portions, k, v, call=None):
        B = self.B
        for slot, p, n in portions:
            if p < 0:
                continue
            begin = p // B * B
            if p > begin and not begin < self.held[slot] <= begin + B or self.held[slot] < p:
                for side in "kv":
                    have = self.rows[slot][side]
                    if p > begin:
                        numbers, scale = self.now(side, slot, p // B)
                        have[begin:p] = (numbers.astype(np.float32) * scale[:, None, None]).transpose(1, 0, 2)[:p - begin]
            end = p + n
            self.held[slot] = end if end % B else p if p > begin else 0
            for b in [b for s, b in self.touched if s == slot and b > (end - 1) // B]:
                del self.touched[(slot, b)]                     # gone, though their bytes are there
        super().write(portions, k, v, call)

    def now(self, side, slot, b):
        """numbers [head, position, channel] and scales [head] of a block as the pool holds it"""
        pool, scale = (self.cache.k_pool, self.cache.k_scale) if side == "k" else (self.cache.v_pool, self.cache.v_scale)
        at = int(self.table[slot, b])
        return O.numbers(pool[at, LAYER].view(torch.int8).cpu().numpy(), self.fmt), scale[at, LAYER].cpu().numpy()

    def check(self):
        """Codes, scales and open rows of everything that the slots hold."""
        c = self.cache
        for side, pool, scale, kept in (("k", c.k_pool, c.k_scale, c.k_open), ("v", c.v_pool, c.v_scale, c.v_open)):
            codes, scale, kept = pool.view(torch.int8).cpu().numpy(), scale.cpu().numpy(), kept.cpu().numpy()
            for (slot, b), count in self.touched.items():
                want, s = self.expect(side, slot, b, count)
                at = self.table[slot, b]
                assert np.array_equal(scale[at, LAYER], s), (side, slot, b)
                assert np.array_equal(O.numbers(codes[at, LAYER], self.fmt), want), (side, slot, b)
            for slot, rows in enumerate(self.rows):
                n = len(rows[side])
                if n % self.B:
                    begin = n // self.B * self.B
                    assert np.array_equal(kept[slot, LAYER][:, :n - begin], rows[side][begin:].transpose(1, 0, 2)), (side, slot)
        assert bool((c.open_end[:, [x for x in range(T.LAYERS) if x != LAYER]] == -1).all())


# block 16: back by one across a border, into the middle of an earlier block by single rows and by portions, to a block's start, twice in a row, into a block that was filled at once
STEPS = [[(0, 0, 33), (1, 0, 16), (2, 0, 40)], [(0, 31, 1), (1, 15, 1), (2, 40, 24)], [(0, 32, 5), (1, 16, 3), (2, 63, 2)], [(0, 30, 4), (1, 7, 1), (2, -1, 1)], [(0, 16, 40), (1, 8, 40), (2, 50, 14)],
         [(0, 55, 1), (1, 47, 2), (2, 49, 1)], [(0, 3, 1), (1, 1, 120), (2, 5, 60)], [(0, 4, 12), (1, 120, 1), (2, 64, 1)], [(0, 15, 1), (1, 119, 9), (2, 63, 1)], [(0, 14, 2), (1, 127, 1), (2, 48, 16)],
         [(0, 16, 1), (1, 100, 20), (2, 60, 1)]]


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("block,kv_heads,dim,vdim", [(16, 2, 64, 64), (16, 5, 128, 128), (32, 3, 96, 32), (128, 1, 16, 128)])
def test_slots_that_are_written_again_from_earlier_positions(fmt, block, kv_heads, dim, vdim):
    m = Rewound(3, 256, kv_heads, block, dim, vdim, fmt)
    for step in STEPS:
        m.put(step)
        m.check()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("block,kv_heads,dim,vdim", [(16, 9, 32, 64), (32, 2, 128, 128), (64, 3, 48, 16), (128, 2, 128, 64)])
def test_positions_anywhere(fmt, block, kv_heads, dim, vdim):
    m, rng = Rewound(4, 6 * block, kv_heads, block, dim, vdim, fmt), np.random.default_rng(block)
    for _ in range(25):
        step = []
        for slot in rng.permutation(4)[:rng.integers(1, 5)]:
            have = len(m.rows[slot]["k"])
            p = int(rng.choice([have, max(0, have - 1), rng.integers(0, have + 1), have // block * block]))
            n = int(rng.choice([1, 1, rng.integers(1, block + 1), rng.integers(1, 3 * block)]))
            if p + n > 6 * block:
                p, n = 0, 1
            step.append((int(slot), p, n))
        m.put(step)
        m.check()


def test_drafted_tokens_that_are_dropped():
    """Decoding with drafts of four tokens, of which some stay: the attention of every step is that over the cache as it then is."""
    H, D, heads = 2, 64, 6
    m = Rewound(2, 200, H, 16, D, D, "int8")
    fill = lambda parts: m.write(parts, *(torch.from_numpy(m.rng.standard_normal((sum(x[2] for x in parts), H * D)).astype(np.float32)).cuda() for _ in "kv"))  # noqa: E731
    fill([(0, 0, 13), (1, 0, 30)])
    at, rng = [13, 30], np.random.default_rng(4)
    for step in range(30):
        parts = [(s, at[s], 4) for s in (0, 1)]
        fill(parts)
        out, want = T.attend(m, dict(heads=heads, scale=D ** -0.5), parts, torch.float32, q_seed=step)
        T.close(out, want)
        at = [a + int(rng.integers(1, 5)) for a in at]
    m.check()


def test_open_rows_that_a_host_fills():
    """With -1 the open rows are taken as they are; without open_end they are too."""
    for known in (True, False):
        m = T.Mirror(1, 64, 2, 16, 64, 64, "int8")
        m.put([(0, 0, 37)])
        c = m.cache
        rows = [t.clone() for t in (c.k_open, c.v_open)]
        m.put([(0, 37, 20)])                                    # the open rows are those of block 3 now
        c.k_open.copy_(rows[0])
        c.v_open.copy_(rows[1])
        if known:
            c.open_end.fill_(-1)
        else:
            m.cache = K.Kv8Cache(c.k_pool, c.v_pool, c.k_scale, c.v_scale, c.k_open, c.v_open, c.table)
        m.touched = {k: v for k, v in m.touched.items() if k[1] < 2}
        m.put([(0, 37, 1)])
        for side in "kv":
            numbers, scale = m.expect(side, 0, 2, 6)
            pool, s = (c.k_pool, c.k_scale) if side == "k" else (c.v_pool, c.v_scale)
            assert np.array_equal(O.numbers(pool[int(m.table[0, 2]), LAYER].view(torch.int8).cpu().numpy(), "int8"), numbers)
            assert np.array_equal(s[int(m.table[0, 2]), LAYER].cpu().numpy(), scale)
