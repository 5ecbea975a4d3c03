"""Low-rank adapters of many requests against the same in 64 bits.

The bound, element by element: t = A x sums k products in f32, in any order and
grouping of at least sixteen runs of k / 16 (k / 16 + 24 steps of 2^-24 of
sum |a x|), x carried with 22 bits or more (2^-22); s B t sums rank products
(rank + 8 steps), t carried with 22 bits or more (2^-22); y is rounded twice.
Of an x far below its row's largest 2^-38 of that one may be lost."""
import numpy as np
import pytest

from doe_amd import DeviceBuffer, Graph, Stream, ops, synchronize

pytestmark = pytest.mark.gpu

up = DeviceBuffer.from_array
i32 = lambda x: np.asarray(x, np.int32)  # noqa: E731


def bf16_bits(x):
    b = np.asarray(x, np.float32).view(np.uint32)
    return ((b + 0x7fff + (b >> 16 & 1)) >> 16).astype(np.uint16)


def bf16_values(bits):
    return (bits.astype(np.uint32) << 16).view(np.float32)


class Case:
    def __init__(self, seed, rows, k, slice_n, rank, adapters=3, bf16=False, counts=None, x_pad=0, y_pad=0, scales=True, wide=1.0):
        rng = np.random.default_rng(seed)
        self.rows, self.k, self.slice_n, self.rank, self.adapters = rows, k, list(slice_n), rank, adapters
        self.n, s = sum(slice_n), len(slice_n)
        a = (rng.standard_normal((adapters, s * rank, k)) / np.sqrt(k)).astype(np.float32)
        b = (rng.standard_normal((adapters, self.n, rank)) / np.sqrt(rank)).astype(np.float32)
        if bf16:
            self.a_bits, self.b_bits = bf16_bits(a), bf16_bits(b)
            self.a, self.b = (bf16_values(v).astype(np.float64) for v in (self.a_bits, self.b_bits))
        else:
            self.a_bits, self.b_bits = a.astype(np.float16), b.astype(np.float16)
            self.a, self.b = self.a_bits.astype(np.float64), self.b_bits.astype(np.float64)
        self.scales = rng.uniform(0.2, 2, adapters).astype(np.float32) if scales else None
        self.counts = counts
        self.ids = i32(rng.integers(-1, adapters + 1, len(counts) if counts else rows))  # some name none
        if len(self.ids):
            self.ids[0] = adapters - 1
        self.x = (rng.standard_normal((rows, k + x_pad)) * np.exp(rng.uniform(0, np.log(wide) if wide > 1 else 0, (rows, k + x_pad)))).astype(np.float32)
        self.y = rng.standard_normal((rows, self.n + y_pad)).astype(np.float32)
        self.lora = ops.Lora(up(self.a_bits), up(self.b_bits), up(self.scales) if scales else None, num_adapters=adapters,
                             rank=rank, k=k, slice_n=slice_n, bf16=bf16)
        self.bufs = dict(adapters=up(self.ids), x=up(self.x), y=up(self.y))
        self.how = dict(x_row_stride=k + x_pad, y_row_stride=self.n + y_pad)
        if counts:
            self.starts = i32(np.cumsum([0] + list(counts)))
            self.how |= dict(row_starts=up(self.starts), segments=len(counts))
        self.ws = DeviceBuffer(ops.lora_workspace(self.lora, rows) + 64)
        self.ws.upload(np.full(self.ws.nbytes, 0xff, np.uint8))  # NaNs of other calls

    def row_ids(self):
        if self.counts is None:
            return self.ids
        ids = np.full(self.rows, -1)
        for s, a in enumerate(self.ids):
            ids[self.starts[s]:self.starts[s + 1]] = a
        return ids

    def run(self, stream=None):
        ws = self.ws.view(0, self.ws.nbytes - 64)
        ops.lora_add(self.lora, self.bufs["adapters"], self.bufs["x"], self.bufs["y"], self.rows, workspace=ws, stream=stream, **self.how)

    def want(self, y=None):
        out = (self.y if y is None else y).astype(np.float64)
        bound = np.zeros_like(out)
        ids, r, e = self.row_ids(), self.rank, 2.0 ** -24
        for a in range(self.adapters):
            at = np.flatnonzero(ids == a)
            x = self.x[at, :self.k].astype(np.float64)
            t, mass = x @ self.a[a].T, np.abs(x) @ np.abs(self.a[a]).T
            dt = ((self.k / 16 + 24) * e + 2.0 ** -22) * mass
            dt += 2.0 ** -38 * np.abs(x).max(1, initial=0)[:, None] * np.abs(self.a[a]).sum(1)
            s, col = float(self.scales[a]) if self.scales is not None else 1.0, 0
            for i, width in enumerate(self.slice_n):
                b, j = self.b[a, col:col + width].T, slice(i * r, (i + 1) * r)
                cols = slice(col, col + width)
                out[np.ix_(at, range(col, col + width))] += s * (t[:, j] @ b)
                m = np.abs(t[:, j]) @ np.abs(b)
                bound[at, cols] = s * (dt[:, j] @ np.abs(b) + ((r + 8) * e + 2.0 ** -22) * m + 2.0 ** -38 * np.abs(t[:, j]).max(1, initial=0)[:, None] * np.abs(b).sum(0)) + 2 * e * (np.abs(out[at, cols]) + s * m)
                col += width
        return out, bound

    def check(self, y=None):
        got = self.bufs["y"].download()
        want, bound = self.want(y)
        off = np.abs(got - want)
        print(f"  at most {np.max(off / np.maximum(bound, 1e-300), initial=0, where=bound > 0):.3f} of the bound", flush=True)
        assert np.all(off <= bound)  # (0 where nothing is added: those rows keep their bits)
        assert np.array_equal(self.ws.download()[-64:], np.full(64, 0xff, np.uint8))
        return got


SHAPES = [
    # rows, k, slices, rank
    (1, 64, [8], 8), (1, 2304, [4096], 16), (3, 8, [1], 8), (2, 200, [33, 7, 5, 100], 24), (17, 136, [50, 51], 16),
    (64, 2304, [256, 128, 128], 16), (33, 72, [515], 64), (5, 1032, [31, 1], 128), (40, 264, [129], 256), (130, 640, [2048, 640], 32),
]


@pytest.mark.parametrize("rows,k,slice_n,rank", SHAPES)
@pytest.mark.parametrize("bf16", [False, True], ids=["f16", "bf16"])
def test_rows_with_adapters_of_their_own(dev, rows, k, slice_n, rank, bf16):
    print(f"[lora] {rows} {k} {slice_n} {rank}", flush=True)
    c = Case(rows + k, rows, k, slice_n, rank, bf16=bf16)
    c.run()
    c.check()


RAGGED = [
    # counts, k, slices, rank
    ([5, 0, 1, 70, 31], 136, [50, 51], 16), ([200], 2304, [300], 16), ([1, 1, 1], 64, [64], 8), ([33, 95, 64, 1, 0, 0, 7], 328, [131, 5], 24),
    ([300, 41], 96, [1030], 64), ([129], 1032, [260, 60, 30], 128), ([65, 64], 520, [96], 256), ([600], 72, [40], 8),
]


@pytest.mark.parametrize("counts,k,slice_n,rank", RAGGED)
@pytest.mark.parametrize("bf16", [False, True], ids=["f16", "bf16"])
def test_ragged_segments(dev, counts, k, slice_n, rank, bf16):
    print(f"[lora] {counts} {k} {slice_n} {rank}", flush=True)
    c = Case(k, sum(counts) + 3, k, slice_n, rank, bf16=bf16, counts=counts)  # the last three rows of no segment
    c.run()
    c.check()


TILES = [
    # counts, k, slices, rank: enough bytes of weights for tiles of 32 rows
    ([300, 1, 0, 0, 31, 33, 64, 95], 2304, [1000, 501], 16), ([129, 200], 1032, [260, 3000, 30], 128), ([700], 5000, [2049], 8),
    ([65, 64, 0, 100], 520, [1096, 40], 256), ([40] * 70, 1000, [333], 24), ([500], 8, [4100, 70, 1, 33], 32), ([1500], 72, [9001], 64),
    (list(np.random.default_rng(0).integers(0, 6, 4300)), 512, [500], 8),
]
# ... or workgroups
TILES_OF_FEW_BYTES = [([500, 145], 64, [33], 8), ([60, 0, 91, 100], 136, [1, 1030, 7], 24), ([350], 72, [1025], 16)]


@pytest.mark.parametrize("counts,k,slice_n,rank", TILES)
@pytest.mark.parametrize("bf16", [False, True], ids=["f16", "bf16"])
def test_tiles(dev, counts, k, slice_n, rank, bf16):
    print(f"[lora] {counts[:8]} {k} {slice_n} {rank}", flush=True)
    assert 2 * sum(counts) * rank * (len(slice_n) * k + sum(slice_n)) > 48 << 20
    c = Case(k, sum(counts) + 3, k, slice_n, rank, bf16=bf16, counts=counts)
    c.run()
    c.check()


@pytest.mark.parametrize("counts,k,slice_n,rank", TILES_OF_FEW_BYTES)
@pytest.mark.parametrize("bf16", [False, True], ids=["f16", "bf16"])
def test_tiles_of_few_bytes(dev, counts, k, slice_n, rank, bf16):
    assert sum(counts) * sum(-(-n // 1024) for n in slice_n) > 640
    c = Case(k, sum(counts) + 3, k, slice_n, rank, bf16=bf16, counts=counts)
    c.run()
    c.check()


@pytest.mark.parametrize("rows,k,slice_n,rank", [(30, 2304, [9216, 300], 64), (3, 5376, [700], 256), (150, 264, [2000], 128), (200, 2304, [2000, 99], 16)])
@pytest.mark.parametrize("bf16", [False, True], ids=["f16", "bf16"])
def test_rows_in_two_launches(dev, rows, k, slice_n, rank, bf16):
    c = Case(rows, rows, k, slice_n, rank, bf16=bf16)
    c.run()
    c.check()


@pytest.mark.parametrize("counts", [None, [90, 6], [900, 300]])
def test_strides_and_no_scales(dev, counts):
    c = Case(7, sum(counts or [96]), 2064, [337, 164], 64, x_pad=12, y_pad=3, counts=counts, scales=False)
    c.run()
    got = c.check()
    assert np.array_equal(got[:, c.n:], c.y[:, c.n:])


@pytest.mark.parametrize("rows", [4, 200, 3000])
def test_rows_of_widely_different_values(dev, rows):
    """Dims from 1 to 2^20 side by side, and rows of zeros, keep their bits."""
    c = Case(3, rows, 520, [370], 16, counts=[rows], wide=2.0 ** 20)
    c.x[1] = 0
    c.x[2] *= np.float32(2.0 ** 90)
    c.x[3] *= np.float32(2.0 ** -90)
    c.bufs["x"] = up(c.x)
    c.run()
    c.check()


@pytest.mark.parametrize("rows,bf16", [(3, False), (3, True), (150, False), (150, True), (4000, False), (4000, True)])
def test_infinities_stay_in_their_rows(dev, rows, bf16):
    c = Case(5, rows, 136, [440], 16, counts=[rows], bf16=bf16)
    c.x[1, 7], c.x[2, 3] = np.inf, np.nan
    c.bufs["x"] = up(c.x)
    c.run()
    got = c.bufs["y"].download()
    c.x[1:3] = 0
    want, bound = c.want()
    keep = np.delete(np.arange(rows), [1, 2])
    assert np.all(np.abs(got - want)[keep] <= bound[keep])
    assert not np.isfinite(got[1]).any() and np.isnan(got[2]).all()


@pytest.mark.parametrize("counts", [None, [100, 30, 70], [1000, 5, 600]])
def test_captured_calls_replay(dev, counts):
    """Twice the same bits, captured or not, on a stream of its own and with other ids between replays."""
    s = Stream()
    c = Case(9, sum(counts or [200]), 520, [130, 170], 32, counts=counts)
    c.run(s)
    s.synchronize()
    first = c.check()
    g = Graph.capture(s, lambda: c.run(s))
    for turn in range(3):
        c.bufs["y"].upload(c.y)
        synchronize()
        g.launch(s)
        s.synchronize()
        assert np.array_equal(c.bufs["y"].download(), first)
    c.ids = i32(c.ids[::-1].copy())
    c.bufs["adapters"].upload(c.ids)
    c.bufs["y"].upload(c.y)
    synchronize()
    g.launch(s)
    s.synchronize()
    c.check()
    g.destroy()
    s.destroy()


def test_two_calls_at_once_with_workspaces_of_their_own(dev):
    s, t = Stream(), Stream()
    c, d = Case(1, 1300, 1032, [700], 16, counts=[1300]), Case(2, 64, 2304, [900], 16)
    synchronize()
    for _ in range(3):
        c.run(s)
        d.run(t)
    s.synchronize()
    t.synchronize()
    for case in (c, d):
        want, bound = case.want()
        once = want - case.y
        assert np.all(np.abs(case.bufs["y"].download() - (case.y + 3 * once)) <= 3 * bound + 2.0 ** -22 * (np.abs(case.y) + 3 * np.abs(once)))
    s.destroy()
    t.destroy()


def test_nothing_to_do(dev):
    c = Case(4, 0, 64, [8], 8)
    ops.lora_add(c.lora, c.bufs["adapters"], c.bufs["x"], c.bufs["y"], 0, workspace=c.ws)
    d = Case(4, 5, 64, [8], 8)
    d.bufs["adapters"] = up(i32([-1, 3, 99, -5, 1 << 30]))  # no adapter at all
    d.run()
    assert np.array_equal(d.bufs["y"].download(), d.y)


def test_beside_a_quantized_projection(dev):
    """A decode step's projection in Q4_K with a request's adapter: one row after the GEMV."""
    from doe_amd import q4k
    rng = np.random.default_rng(6)
    n, k = 512, 768
    w = q4k.random_q4k(rng, n, k)
    c = Case(8, 1, k, [n], 16)
    ops.matmul_q4k(up(w), c.bufs["x"], c.bufs["y"], n, k)
    base = c.bufs["y"].download()
    c.run()
    c.check(base)


@pytest.mark.parametrize("counts", [None, [30], [1100]])
def test_rows_of_y_past_four_gigabytes(dev, counts):
    """The same sums as beside each other, 5 MB and more from row to row."""
    rows = sum(counts or [30])
    c = Case(11, rows, 1024, [3000], 24, counts=counts)
    c.run()
    near = c.bufs["y"].download()
    stride = ((5 << 30) // 4 + (rows - 2)) // (rows - 1)
    far = DeviceBuffer(4 * ((rows - 1) * stride + c.n))
    assert far.nbytes > 5 << 30
    parts = [far.view(4 * r * stride, 4 * c.n, np.float32, (c.n,)) for r in range(rows)]
    for part, y in zip(parts, c.y):
        part.upload(y)
    c.bufs["y"], c.how["y_row_stride"] = far, stride
    c.run()
    assert all(np.array_equal(part.download(), row) for part, row in zip(parts, near))
    far.free()
