"""Rows rotated and appended to paged caches: bit for bit the same as on the
host (f32 products and sums each rounded, then f16 or the 4-bit cache's codes),
and as the calls for one sequence's contiguous cache."""
import numpy as np
import pytest

from doe_amd import DeviceBuffer, Graph, Stream, mx4, ops, synchronize

pytestmark = pytest.mark.gpu

up = DeviceBuffer.from_array
i32 = lambda x: np.asarray(x, np.int32)  # noqa: E731


def rotate(x, cs, interleaved):
    """[rows][heads][rot] by [rows][rot / 2][2]."""
    half = x.shape[-1] // 2
    c, s = cs[:, None, :, 0], cs[:, None, :, 1]
    x0, x1 = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :half], x[..., half:])
    a, b = x0 * c - x1 * s, x0 * s + x1 * c
    return np.stack([a, b], -1).reshape(x.shape) if interleaved else np.concatenate([a, b], -1)


class Case:
    def __init__(self, seed, lens, counts, *, hq, hkv, d, ps, rot=None, interleaved=False, q_f16=False, mx4_cache=False,
                 pad=0, q_pad=0, positions=None, spare=2, starts=True, in_place=False, lead=0):
        rng = np.random.default_rng(seed)
        self.rng = rng
        self.lens, self.counts, self.hq, self.hkv, self.d, self.ps = list(lens), list(counts), hq, hkv, d, ps
        self.rot = d if rot is None else rot
        self.interleaved, self.q_f16, self.mx4 = interleaved, q_f16, mx4_cache
        self.batch, self.stride = len(lens), max(1, max(-(-n // ps) for n in lens)) + 1
        self.num_pages = sum(-(-max(0, n) // ps) for n in lens) + spare
        ids = list(rng.permutation(self.num_pages))
        self.table = np.full((self.batch, self.stride), -1, np.int32)
        for b, n in enumerate(lens):
            for i in range(-(-n // ps)):
                self.table[b, i] = ids.pop()
        self.lead = lead  # rows before the first sequence's
        self.rows = lead + sum(counts) + (2 if starts else 0)  # and two behind the last one's
        self.width = (hq + 2 * hkv) * d
        self.qkv = rng.standard_normal((self.rows, self.width + pad)).astype(np.float32)
        self.positions = max(max(lens), 1) if positions is None else positions
        angle = rng.uniform(-np.pi, np.pi, (self.positions, self.rot // 2)).astype(np.float32)
        self.freq = np.stack([np.cos(angle), np.sin(angle)], -1).astype(np.float32)
        self.starts = i32(lead + np.cumsum([0] + self.counts))
        self.row_starts = up(self.starts) if starts else None
        self.in_place = in_place
        self.q = rng.standard_normal((self.rows, hq * d + q_pad)).astype(np.float16 if q_f16 else np.float32)
        self.dq, self.dqkv = up(self.q), up(self.qkv)
        self.dtable, self.dlens = up(self.table), up(i32(lens))
        how = dict(num_pages=self.num_pages, page_size=ps, num_kv_heads=hkv, head_dim=d, batch=self.batch, table_stride=self.stride)
        if mx4_cache:
            self.pool = rng.integers(0, 256, (self.num_pages, mx4.page_bytes(ps, hkv, d))).astype(np.uint8)
            self.dpools = [up(self.pool)]
            self.cache = ops.Mx4Cache(self.dpools[0], self.dtable, self.dlens, **how)
        else:
            self.pools = [rng.standard_normal((self.num_pages, ps, hkv, d)).astype(np.float16) for _ in "kv"]
            self.dpools = [up(p) for p in self.pools]
            self.cache = ops.F16Cache(*self.dpools, self.dtable, self.dlens, **how)
        self.how = how

    def run(self, stream=None):
        kw = dict(row_stride=self.qkv.shape[1], q_row_stride=self.q.shape[1])
        q = self.dq
        if self.in_place:
            q, kw["q_row_stride"] = self.dqkv, self.qkv.shape[1]
        ops.qkv_rope_append(self.cache, self.dqkv, q if self.hq else None, self.rows, num_heads=self.hq, freq_cis=up(self.freq) if self.freq.size else None,
                            max_positions=self.positions, rotary_dim=self.rot, interleaved=self.interleaved, q_f16=self.q_f16,
                            row_starts=self.row_starts, stream=stream, **kw)

    def places(self):
        """(row, position, page or -1) of the rows that have a sequence."""
        for b, n in enumerate(self.counts):
            length = min(max(self.lens[b], 0), self.stride * self.ps)
            for i in range(n):
                pos = length - n + i
                page = self.table[b, pos // self.ps] if pos >= 0 else -1
                yield self.starts[b] + i, pos, page if 0 <= page < self.num_pages and pos < self.positions else -1

    def check(self):
        x = self.qkv[:, :self.width].reshape(self.rows, -1, self.d)
        turned, want_q = x.copy(), self.q.copy()
        d, kv = self.d, self.hq
        places = list(self.places())
        for row, pos, _ in places:
            if 0 <= pos < self.positions:
                turned[row, :kv + self.hkv, :self.rot] = rotate(x[row:row + 1, :kv + self.hkv, :self.rot], self.freq[pos:pos + 1], self.interleaved)[0]
            want_q[row, :kv * d] = turned[row, :kv].reshape(-1).astype(want_q.dtype)
        if self.in_place:
            want = self.qkv.copy()
            for row, _, _ in places:
                want[row, :kv * d] = turned[row, :kv].reshape(-1)
            assert np.array_equal(self.dqkv.download(), want)
        else:
            assert np.array_equal(self.dqkv.download(), self.qkv)
            if kv:
                assert np.array_equal(self.dq.download(), want_q)
        if self.mx4:
            # the same rows, rotated before, by the call that takes them so
            kr, vr = turned[:, kv:kv + self.hkv].reshape(self.rows, -1), x[:, kv + self.hkv:].reshape(self.rows, -1)
            pool = up(self.pool)
            table = self.table.copy()
            for b in range(self.batch):  # (positions beyond the angles are not appended)
                table[b, -(-self.positions // self.ps):] = -1
            c = ops.Mx4Cache(pool, up(table), self.dlens, **self.how)
            ops.mx4_kv_write(c, up(kr), up(vr), self.rows, row_starts=self.row_starts)
            assert np.array_equal(self.dpools[0].download(), pool.download())
            return
        for pool, dpool, rows in zip(self.pools, self.dpools, (turned[:, kv:kv + self.hkv], x[:, kv + self.hkv:])):
            want = pool.copy()
            for row, pos, page in places:
                if page >= 0:
                    want[page, pos % self.ps] = rows[row].astype(np.float16)
            assert np.array_equal(dpool.download(), want)


SHAPES = [
    # lens, counts, heads, KV heads, head_dim, page size
    ([701], [1], 8, 4, 256, 64), ([1], [1], 1, 1, 64, 32), ([5, 90, 33], [5, 70, 1], 4, 2, 64, 32), ([200, 3, 0, 64], [130, 3, 0, 64], 6, 3, 128, 64),
    ([40, 41], [7, 9], 8, 1, 512, 32), ([300], [299], 4, 4, 160, 128), ([100, 7], [50, 7], 3, 1, 256, 256),
]


@pytest.mark.parametrize("mx4_cache", [False, True], ids=["f16", "mx4"])
@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "pairs"])
@pytest.mark.parametrize("lens,counts,hq,hkv,d,ps", SHAPES)
def test_rows(dev, lens, counts, hq, hkv, d, ps, interleaved, mx4_cache):
    print(f"[append] {lens} {counts} {hq} {hkv} {d} {ps}", flush=True)
    c = Case(d + len(lens), lens, counts, hq=hq, hkv=hkv, d=d, ps=ps, interleaved=interleaved, mx4_cache=mx4_cache)
    c.run()
    c.check()


@pytest.mark.parametrize("lens,counts,hq,hkv,d,ps", [([20, 9], [11, 9], 5, 5, 48, 7), ([130], [130], 2, 1, 8, 1), ([50, 0, 3], [4, 0, 1], 9, 3, 80, 48),
                                                     ([3000], [2900], 4, 1, 24, 100), ([33], [33], 1, 1, 1024, 16)])
@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "pairs"])
def test_f16_pages_of_any_size(dev, lens, counts, hq, hkv, d, ps, interleaved):
    c = Case(d, lens, counts, hq=hq, hkv=hkv, d=d, ps=ps, interleaved=interleaved)
    c.run()
    c.check()


@pytest.mark.parametrize("mx4_cache", [False, True], ids=["f16", "mx4"])
@pytest.mark.parametrize("rot", [0, 8, 64, 120, 128])
@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "pairs"])
def test_part_of_a_head(dev, rot, interleaved, mx4_cache):
    c = Case(rot, [70, 33], [70, 2], hq=4, hkv=2, d=128, ps=32, rot=rot, interleaved=interleaved, mx4_cache=mx4_cache, q_f16=True, pad=12, q_pad=8)
    c.run()
    c.check()


@pytest.mark.parametrize("mx4_cache", [False, True], ids=["f16", "mx4"])
@pytest.mark.parametrize("q_f16,in_place,pad", [(True, False, 4), (False, False, 0), (False, True, 8)])
@pytest.mark.parametrize("d", [64, 160])
def test_one_row_a_sequence(dev, q_f16, in_place, pad, d, mx4_cache):
    """Without row_starts; queries in f16, f32 and in place."""
    lens = [1, 700, 33, 64, 65]
    c = Case(d, lens, [1] * 5, hq=8, hkv=2, d=d, ps=64, q_f16=q_f16, in_place=in_place, pad=pad, starts=False, mx4_cache=mx4_cache)
    c.run()
    c.check()


@pytest.mark.parametrize("mx4_cache", [False, True], ids=["f16", "mx4"])
@pytest.mark.parametrize("d", [64, 160])
def test_rows_without_a_place(dev, d, mx4_cache):
    """Rows before the first sequence's, more rows than positions, pages outside
    the pool, positions beyond the angles and lengths beyond the table."""
    c = Case(3, [20, 90, 5, 100], [20, 60, 9, 3], hq=2, hkv=1, d=d, ps=32, positions=64, lead=3, mx4_cache=mx4_cache)
    c.table[0, 0], c.table[1, 1] = c.num_pages, -7
    c.dtable.upload(c.table)
    c.lens = [20, 90, 5, 100 + (1 << 20)]
    c.dlens.upload(i32(c.lens))
    c.run()
    c.check()
    c.lens = [-5, 90, 5, 100]
    c.dlens.upload(i32(c.lens))
    for pool, dev_pool in zip([c.pool] if mx4_cache else c.pools, c.dpools):
        dev_pool.upload(pool)
    c.dq.upload(c.q)
    c.run()
    c.check()


def test_no_queries_and_nothing(dev):
    c = Case(1, [40], [8], hq=0, hkv=2, d=64, ps=16)
    c.run()
    c.check()
    ops.qkv_rope_append(c.cache, c.dqkv, c.dq, 0, num_heads=0, freq_cis=None, max_positions=0, row_starts=c.row_starts)
    c.check()


@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "pairs"])
def test_same_as_the_call_for_one_sequence(dev, interleaved):
    c = Case(4, [90], [50], hq=4, hkv=2, d=128, ps=32, interleaved=interleaved)
    c.run()
    keep = c.qkv[:50].copy()
    dqkv, kc, vc = up(keep), DeviceBuffer.empty((2, 90, 128), np.float16), DeviceBuffer.empty((2, 90, 128), np.float16)
    fn = ops.qkv_rope_kv_rows if interleaved else ops.qkv_rope_half_kv_rows
    fn(dqkv, 50, c.width, 4, 2, 128, up(c.freq), 40, kc, vc, 90)
    assert np.array_equal(dqkv.download()[:, :512], c.dq.download()[:50])
    for pool, flat in zip(c.dpools, (kc, vc)):
        pages = pool.download()
        for pos in range(40, 90):
            assert np.array_equal(pages[c.table[0, pos // 32], pos % 32], flat.download()[:, pos])


def test_pages_are_read_by_the_attention_dispatch(dev, ora):
    """A prompt appended to f16 pages and attended through its page table."""
    c = Case(5, [70], [70], hq=4, hkv=2, d=64, ps=16)
    c.run()
    out = DeviceBuffer.empty((70, 4, 64), np.float32)
    ops.attention_dispatch(c.dq, *c.dpools, out, num_heads=4, num_kv_heads=2, head_dim=64, seq_len=70, query_len=70, scale=0.125,
                           is_causal=True, kv_layout=2, page_size=16, page_table=up(c.table[0, :5].astype(np.uint32)),
                           kv_capacity=c.num_pages * 16)
    q = c.dq.download()[:70].reshape(70, 4, 64).astype(np.float64)
    k, v = (np.concatenate([p.download()[page] for page in c.table[0, :5]])[:70].astype(np.float64) for p in c.dpools)
    for h in range(4):
        s = q[:, h] @ k[:, h // 2].T * 0.125
        s[np.triu_indices(70, 1)] = -np.inf
        p = np.exp(s - s.max(1, keepdims=True))
        want = p / p.sum(1, keepdims=True) @ v[:, h // 2]
        got = out.download()[:, h]
        assert np.linalg.norm(got - want) <= 1e-5 * np.linalg.norm(want)


@pytest.mark.parametrize("mx4_cache", [False, True], ids=["f16", "mx4"])
def test_captured_with_growing_sequences(dev, mx4_cache):
    s = Stream()
    c = Case(6, [40, 33, 90], [1, 1, 1], hq=4, hkv=2, d=64, ps=32, starts=False, mx4_cache=mx4_cache)
    freq = up(c.freq)
    g = Graph.capture(s, lambda: ops.qkv_rope_append(c.cache, c.dqkv, c.dq, 3, num_heads=4, freq_cis=freq, max_positions=c.positions, stream=s))
    for turn in range(3):
        c.lens = [40 - turn, 33 - turn, 90 - turn]
        c.dlens.upload(i32(c.lens))
        for pool, dev_pool in zip([c.pool] if mx4_cache else c.pools, c.dpools):
            dev_pool.upload(pool)
        synchronize()
        g.launch(s)
        s.synchronize()
        c.check()
    g.destroy()
    s.destroy()


@pytest.mark.parametrize("batch,d", [(65, 64), (130, 256), (200, 512), (4200, 128)])
def test_more_sequences_than_lanes(dev, batch, d):
    """The same pages and rows as by calls of fifty sequences each."""
    rng = np.random.default_rng(batch)
    counts = rng.integers(0, 6, batch)
    counts[[0, 40, batch - 1]] = 0
    c = Case(batch, list(counts + rng.integers(0, 40, batch)), list(counts), hq=1, hkv=1, d=d, ps=32, mx4_cache=True, lead=3)
    c.run()
    got = c.dpools[0].download()
    assert not np.array_equal(got, c.pool)
    kr, vr = (up(np.zeros((c.rows, d), np.float32)) for _ in "kv")
    ops.mx4_kv_read(c.cache, kr, vr, c.rows, row_starts=c.row_starts)
    pool = up(c.pool)
    ks, vs = (up(np.zeros((c.rows, d), np.float32)) for _ in "kv")
    for b in range(0, batch, 50):
        n = min(50, batch - b)
        how = dict(c.how, batch=n)
        part = ops.Mx4Cache(pool, c.dtable.view(4 * b * c.stride, 4 * n * c.stride), c.dlens.view(4 * b, 4 * n), **how)
        starts = c.row_starts.view(4 * b, 4 * (n + 1))
        ops.qkv_rope_append(part, c.dqkv, None if not c.hq else c.dq, c.rows, num_heads=c.hq, freq_cis=up(c.freq),
                            max_positions=c.positions, row_starts=starts, row_stride=c.qkv.shape[1], q_row_stride=c.q.shape[1])
        ops.mx4_kv_read(part, ks, vs, c.rows, row_starts=starts)
    assert np.array_equal(got, pool.download())
    assert np.array_equal(kr.download(), ks.download()) and np.array_equal(vr.download(), vs.download())


def test_pages_past_four_gigabytes(dev):
    """The last pages of pools of 5 GiB each."""
    ps, hkv, d = 64, 4, 128
    page_bytes = 2 * ps * hkv * d
    pages = (5 << 30) // page_bytes
    pools = [DeviceBuffer(pages * page_bytes) for _ in "kv"]
    last = [p.view((pages - 3) * page_bytes, 3 * page_bytes, np.float16, (3, ps, hkv, d)) for p in pools]
    c = Case(6, [70, 20], [70, 2], hq=2, hkv=hkv, d=d, ps=ps, spare=0)
    assert c.num_pages == 3
    for small, far in zip(c.dpools, last):
        far.upload(small.download())
    c.run()
    c.check()
    how = dict(c.how, num_pages=pages)
    c.cache = ops.F16Cache(*pools, up(np.where(c.table < 0, -1, c.table + np.int32(pages - 3))), c.dlens, **how)
    c.run()
    for small, far in zip(c.dpools, last):
        assert np.array_equal(small.download(), far.download())
    for p in pools:
        p.free()


@pytest.mark.parametrize("counts", ["few", "mostly none"])
@pytest.mark.parametrize("batch", [65, 300, 4500])
def test_many_sequences_to_f16_pages(dev, batch, counts):
    rng = np.random.default_rng(batch)
    counts = rng.integers(0, 4, batch) if counts == "few" else (rng.random(batch) < 0.01).astype(int)
    counts[-1] = 2
    c = Case(batch, list(counts + rng.integers(0, 40, batch)), list(counts), hq=2, hkv=1, d=16, ps=16, lead=5)
    c.run()
    c.check()


@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "pairs"])
@pytest.mark.parametrize("rot", [168, 512])
def test_units_that_begin_before_and_end_behind_the_rows(dev, rot, interleaved):
    """Heads of 512 dims, whose pairs are read again: positions 4 n + 1 to 4 n + 3 first and 4 n
    to 4 n + 2 last, in rows that fill their buffer."""
    for past, counts in ((1, [244, 6, 1]), (3, [2, 7, 90]), (2, [1])):
        c = Case(past, [past + 4 * i + n for i, n in enumerate(counts)], counts, hq=8, hkv=1, d=512, ps=32, rot=rot, interleaved=interleaved,
                 q_f16=True, mx4_cache=True)
        c.rows = sum(counts)
        c.qkv, c.q = c.qkv[:c.rows].copy(), c.q[:c.rows].copy()
        c.dqkv, c.dq = up(c.qkv), up(c.q)
        c.run()
        c.check()
