"""K / V rows into the 4-bit cache and back, against the host's quantisation:
every byte of the pages equal, and no other byte touched."""
import numpy as np
import pytest

from doe_amd import DeviceBuffer, Graph, Stream, mx4, ops, synchronize

pytestmark = pytest.mark.gpu

up = DeviceBuffer.from_array
SHAPES = [(64, 3, 32), (128, 2, 64), (160, 2, 32), (256, 4, 64), (512, 1, 256)]


class Pool:
    """A pool filled with 0xa5 and a table of scattered pages for `lens`."""

    def __init__(self, rng, lens, d, h, ps, stride=None):
        self.lens, self.d, self.h, self.ps = list(lens), d, h, ps
        held = [-(-max(n, 0) // ps) for n in lens]
        self.stride = stride or max(1, max(held))
        self.num_pages = sum(held) + 2
        ids = list(rng.permutation(self.num_pages))
        self.table = np.full((len(lens), self.stride), -1, np.int32)
        for b, n in enumerate(held):
            for i in range(min(n, self.stride)):
                self.table[b, i] = ids.pop()
        self.host = np.full((self.num_pages, mx4.page_bytes(ps, h, d)), 0xa5, np.uint8)
        self.dev = up(self.host)
        self.table_dev, self.lens_dev = up(self.table), up(np.array(lens, np.int32))
        self.cache = ops.Mx4Cache(self.dev, self.table_dev, self.lens_dev, num_pages=self.num_pages, page_size=ps,
                                  num_kv_heads=h, head_dim=d, batch=len(lens), table_stride=self.stride)

    def place(self, b, pos):
        if pos < 0:
            return None
        page = self.table[b, pos // self.ps]
        return (page, pos % self.ps) if 0 <= page < self.num_pages else None

    def expect(self, k, v, rows, skip=0):
        """The pages after the rows (sequence by sequence, from row `skip` on)."""
        kc, ks, vc, vs = (x.copy() for x in mx4.unpack_pages(self.host, self.ps, self.h, self.d))
        (qk, sk), (qv, sv) = mx4.quantise(k.astype(np.float32)), mx4.quantise(v.astype(np.float32))
        at, back = skip, {}
        for b, n in enumerate(rows):
            for i in range(n):
                where = self.place(b, min(self.lens[b], self.stride * self.ps) - n + i)
                if where:
                    page, x = where
                    kc[page, :, x], ks[page, :, x], vc[page, :, x], vs[page, :, x] = qk[at], sk[at], qv[at], sv[at]
                    back[at] = mx4.dequantise(qk[at], sk[at]), mx4.dequantise(qv[at], sv[at])
                else:
                    back[at] = 0.0, 0.0
                at += 1
        return mx4.pack_pages(kc, ks, vc, vs), back


def special(rng, shape):
    """Normal rows with wide channels, and blocks at every border of the format."""
    x = rng.standard_normal(shape).astype(np.float32) * (1 + 9 * (rng.random(shape[-1]) < 0.1)).astype(np.float32)
    flat = x.reshape(-1, 32)
    for i, v in enumerate([0.0, -0.0, np.nan, np.inf, -np.inf, 3e38, -1e-30, 1e-9, 65504.0, 7.0, 6.99, 2.0 ** -21]):
        if i < len(flat):
            flat[i, i % 32] = v
            if i in (0, 1, 6, 7, 11):
                flat[i] = v
    return x


@pytest.mark.parametrize("d,h,ps", SHAPES)
@pytest.mark.parametrize("f16", [False, True])
def test_write_tokens(dev, d, h, ps, f16):
    """One row a sequence, at positions around the borders of pages and blocks."""
    rng = np.random.default_rng(d + f16)
    lens = [1, 2, 31, 32, 33, ps, ps + 1, 2 * ps, 0, 3 * ps - 1, 17]
    p = Pool(rng, lens, d, h, ps)
    k, v = special(rng, (len(lens), h, d)), special(rng, (len(lens), h, d))
    if f16:
        with np.errstate(over="ignore"):
            k, v = k.astype(np.float16), v.astype(np.float16)
    print(f"[write] d={d} h={h} ps={ps} f16={f16}", flush=True)
    ops.mx4_kv_write(p.cache, up(k), up(v), len(lens), in_f16=f16)
    want, back = p.expect(k, v, [1] * len(lens))
    assert np.array_equal(p.dev.download(), want)
    ko, vo = DeviceBuffer.empty(k.shape, np.float32), DeviceBuffer.empty(k.shape, np.float32)
    ops.mx4_kv_read(p.cache, ko, vo, len(lens))
    ko, vo = ko.download(), vo.download()
    for i, (bk, bv) in back.items():
        assert np.array_equal(ko[i], np.broadcast_to(bk, ko[i].shape), equal_nan=True)
        assert np.array_equal(vo[i], np.broadcast_to(bv, vo[i].shape), equal_nan=True)


@pytest.mark.parametrize("d,h,ps", SHAPES)
@pytest.mark.parametrize("pad", [0, 32])
def test_write_prompts(dev, d, h, ps, pad):
    """Ragged prompts: sequences without rows, rows before the first and behind
    the last, prompts longer than their length, lengths beyond the table row
    (they count as what it holds), pages outside the pool, rows of a wider
    matrix."""
    rng = np.random.default_rng(7 * d + pad)
    rows = [5, 0, 70, 1, 33, 100, 64, 9]
    lens = [5, 40, 75, 90, 20, 130, 64 + ps, 2 * ps]
    p = Pool(rng, lens, d, h, ps, stride=-(-140 // ps))
    p.table[5, 0], p.table[7, 0] = p.num_pages, -7
    p.table_dev.upload(p.table)
    skip, behind = 3, 4
    total = skip + sum(rows) + behind
    starts = up(np.cumsum([skip] + rows).astype(np.int32))
    k, v = special(rng, (total, h, d)), special(rng, (total, h, d))
    width = h * d + pad
    wide = [np.full((total, width), np.nan, np.float32) for _ in "kv"]
    for w, x in zip(wide, (k, v)):
        w[:, :h * d] = x.reshape(total, -1)
    print(f"[write prompts] d={d} h={h} ps={ps} pad={pad}", flush=True)
    ops.mx4_kv_write(p.cache, up(wide[0]), up(wide[1]), total, row_starts=starts, row_stride=width)
    want, back = p.expect(k, v, rows, skip)
    assert np.array_equal(p.dev.download(), want)
    out = [up(np.full((total, width), -5, np.float32)) for _ in "kv"]
    ops.mx4_kv_read(p.cache, *out, total, row_starts=starts, row_stride=width)
    out = [o.download() for o in out]
    expect = [np.full((total, width), -5, np.float32) for _ in "kv"]
    for i, b in back.items():
        for e, x in zip(expect, b):
            e[i, :h * d] = np.asarray(x).reshape(-1) if np.ndim(x) else x
    for o, e in zip(out, expect):
        assert np.array_equal(o, e, equal_nan=True)


@pytest.mark.parametrize("d,h,ps", [(64, 1, 32), (128, 3, 64), (160, 1, 32), (512, 2, 128)])
def test_write_many_short_prompts(dev, d, h, ps):
    """More sequences than a wave has lanes, of no rows to a few, at any place in a four."""
    rng = np.random.default_rng(d)
    rows = rng.integers(0, 10, 150).tolist()
    lens = [int(n + rng.integers(-2, 40)) if n else 7 for n in rows]
    p = Pool(rng, lens, d, h, ps)
    total = sum(rows)
    starts = up(np.cumsum([0] + rows).astype(np.int32))
    k, v = special(rng, (total, h, d)), special(rng, (total, h, d))
    ops.mx4_kv_write(p.cache, up(k), up(v), total, row_starts=starts)
    want, back = p.expect(k, v, rows)
    assert np.array_equal(p.dev.download(), want)
    out = [up(np.full(k.shape, -5, np.float32)) for _ in "kv"]
    ops.mx4_kv_read(p.cache, *out, total, row_starts=starts)
    out = [o.download() for o in out]
    assert sorted(back) == list(range(total))
    for i, b in back.items():
        for o, x in zip(out, b):
            assert np.array_equal(o[i], np.broadcast_to(x, o[i].shape), equal_nan=True)


def test_every_border_and_scale(dev):
    """Values next to every rounding border, under every scale."""
    near = []
    for t in (0.25, 0.5, 0.75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6):
        t = np.float32(t)
        near += [t, np.nextafter(t, np.float32(9)), np.nextafter(t, np.float32(0))]
    near = np.array(near + [-x for x in near], np.float32)
    blocks = []
    for e in range(-26, 16):
        for i in range(0, len(near), 31):
            block = np.zeros(32, np.float32)
            block[:len(near[i:i + 31])] = near[i:i + 31]
            block[31] = 6.5  # the scale's exponent is e wherever it may be
            blocks.append(np.ldexp(block, e))
    rows = -(-len(blocks) // 2)
    x = np.zeros((rows, 1, 64), np.float32)
    x.reshape(-1, 32)[:len(blocks)] = blocks
    p = Pool(np.random.default_rng(0), [rows], 64, 1, 32)
    ops.mx4_kv_write(p.cache, up(x), up(-x), rows, row_starts=up(np.array([0, rows], np.int32)))
    assert np.array_equal(p.dev.download(), p.expect(x, -x, [rows])[0])


def test_write_captured_and_replayed_with_a_growing_length(dev):
    rng = np.random.default_rng(3)
    p = Pool(rng, [70, 130], 128, 2, 64)
    k, v = up(np.zeros((2, 2, 128), np.float32)), up(np.zeros((2, 2, 128), np.float32))
    st = Stream()
    graph = Graph.capture(st, lambda: ops.mx4_kv_write(p.cache, k, v, 2, stream=st))
    for lens in ([1, 1], [2, 64], [64, 65], [70, 130]):
        kv = [special(rng, (2, 2, 128)) for _ in "kv"]
        synchronize()
        k.upload(kv[0])
        v.upload(kv[1])
        p.lens_dev.upload(np.array(lens, np.int32))
        graph.launch(st)
        st.synchronize()
        p.lens = lens
        p.host = p.expect(*kv, [1, 1])[0]
        assert np.array_equal(p.dev.download(), p.host)
    graph.destroy()
    st.destroy()


def test_rows_of_no_batch_and_no_rows(dev):
    p = Pool(np.random.default_rng(0), [5], 64, 1, 32)
    k = up(np.ones((1, 64), np.float32))
    ops.mx4_kv_write(p.cache, k, k, 0, row_starts=up(np.zeros(2, np.int32)))
    empty = ops.Mx4Cache(p.dev, p.table_dev, p.lens_dev, num_pages=p.num_pages, page_size=32, num_kv_heads=1, head_dim=64,
                         batch=0, table_stride=1)
    ops.mx4_kv_write(empty, k, k, 0)
    ops.mx4_kv_read(empty, k, k, 0)
    assert np.array_equal(p.dev.download(), p.host)
