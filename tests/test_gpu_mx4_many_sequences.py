"""Rows of many sequences written to the 4-bit cache and read back: the same as
on the host, whichever sequences a wave's units lie in."""
import numpy as np
import pytest

from doe_amd import DeviceBuffer, mx4, ops

pytestmark = pytest.mark.gpu

up = DeviceBuffer.from_array
i32 = lambda x: np.asarray(x, np.int32)  # noqa: E731


class Case:
    def __init__(self, seed, lens, counts, hkv, d, ps, starts=True):
        rng = np.random.default_rng(seed)
        self.lens, self.counts, self.hkv, self.d, self.ps = np.asarray(lens), np.asarray(counts), hkv, d, ps
        held = -(-self.lens // ps)
        self.pages, self.stride = int(held.sum()) + 1, max(1, int(held.max()))
        ids = list(rng.permutation(self.pages))
        self.table = np.full((len(lens), self.stride), -1, np.int32)
        for b, n in enumerate(held):
            for i in range(n):
                self.table[b, i] = ids.pop()
        self.rows = int(self.counts.sum())
        self.k, self.v = (rng.standard_normal((self.rows, hkv, d)).astype(np.float32) for _ in "kv")
        self.pool = rng.integers(0, 256, (self.pages, mx4.page_bytes(ps, hkv, d))).astype(np.uint8)
        self.dpool = up(self.pool)
        self.cache = ops.Mx4Cache(self.dpool, up(self.table), up(i32(lens)), num_pages=self.pages, page_size=ps, num_kv_heads=hkv,
                                  head_dim=d, batch=len(lens), table_stride=self.stride)
        self.starts = up(i32(np.cumsum([0, *self.counts]))) if starts else None

    def check(self):
        ops.mx4_kv_write(self.cache, up(self.k), up(self.v), self.rows, row_starts=self.starts)
        kr, vr = (up(np.full((self.rows, self.hkv, self.d), np.nan, np.float32)) for _ in "kv")
        ops.mx4_kv_read(self.cache, kr, vr, self.rows, row_starts=self.starts)
        parts = [p.copy() for p in mx4.unpack_pages(self.pool, self.ps, self.hkv, self.d)]
        coded = [mx4.quantise(x) for x in (self.k, self.v)]
        row = 0
        for b, n in enumerate(self.counts):
            for i in range(n):
                pos = self.lens[b] - n + i
                page, at = self.table[b, pos // self.ps], pos % self.ps
                for j, (codes, scales) in enumerate(coded):
                    parts[2 * j][page, :, at], parts[2 * j + 1][page, :, at] = codes[row], scales[row]
                row += 1
        assert np.array_equal(self.dpool.download(), mx4.pack_pages(*parts))
        for got, (codes, scales) in zip((kr, vr), coded):
            assert np.array_equal(got.download(), mx4.dequantise(codes, scales))


@pytest.mark.parametrize("counts", ["few", "mostly none", "one long"])
@pytest.mark.parametrize("batch", [64, 65, 129, 700, 4099])
@pytest.mark.parametrize("hkv,d", [(1, 64), (3, 64), (1, 128), (2, 256), (1, 512)])
def test_ragged(dev, hkv, d, batch, counts):
    rng = np.random.default_rng(batch + d)
    n = {"few": lambda: rng.integers(0, 5, batch), "mostly none": lambda: (rng.random(batch) < 0.02).astype(int),
         "one long": lambda: (rng.random(batch) < 0.1).astype(int)}[counts]()
    n[-1] = 2
    if counts == "one long":
        n[batch // 2] = 300
    Case(batch, n + rng.integers(0, 9, batch), n, hkv, d, 32).check()


@pytest.mark.parametrize("batch", [1, 4, 63, 257, 2049])
@pytest.mark.parametrize("hkv,d", [(3, 64), (2, 128), (2, 160), (1, 256), (1, 512)])
def test_one_row_a_sequence(dev, hkv, d, batch):
    """At every place of a unit of four positions, of a page's ends among them."""
    Case(d, 1 + np.arange(batch) % 67, [1] * batch, hkv, d, 32, starts=False).check()
