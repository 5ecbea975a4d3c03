"""Beam search's selection against the same in 64 bits, and states in the order
of their parents.

Scores: a term of a row's sum carries the rounding of its exponent's argument
(below 64: 2^-19 of the term) and of up to 80 f32 additions, so the logarithm is
within 2^-18; the sum itself is formed in 64 bits and rounded once."""
import numpy as np
import pytest

from doe_amd import DeviceBuffer, Graph, Stream, ops, synchronize

pytestmark = pytest.mark.gpu

up = DeviceBuffer.from_array
i32 = lambda x: np.asarray(x, np.int32)  # noqa: E731
TOL = 2.0 ** -18


def oracle(logits, scores, finished, select, factor, end):
    """(parents, tokens, scores, ended) and the least gap around the choices that is no tie."""
    batch, beams, vocab = logits.shape
    out = (np.full((batch, select), -1, np.int32), np.full((batch, select), -1, np.int32), np.full((batch, select), -np.inf),
           np.zeros((batch, select), np.int32))
    gap = np.inf
    for r in range(batch):
        offers = []
        for b in range(beams):
            s, row = float(scores[r, b]), logits[r, b].astype(np.float64) * factor
            if not np.isfinite(s):
                continue
            if finished is not None and finished[r, b]:
                offers.append((s, b, end))
                continue
            if np.isnan(row).any() or (row == np.inf).any() or not np.isfinite(row).any():
                continue
            top = row.max()
            lse = top + np.log(np.exp(row - top).sum())
            order = np.lexsort((np.arange(vocab), -row))[:select + 1]
            offers += [(s + row[t] - lse, b, int(t)) for t in order if row[t] > -np.inf]
        offers.sort(key=lambda o: (-o[0], o[1]))  # (of a beam in the order of the logits, then tokens)
        for i, (s, b, t) in enumerate(offers[:select]):
            out[0][r, i], out[1][r, i], out[2][r, i] = r * beams + b, t, s
            out[3][r, i] = int((finished is not None and finished[r, b] != 0) or t == end)
        v = np.array([o[0] for o in offers[:select + 1]])
        d = -np.diff(v)
        gap = min(gap, d[d > 0].min(initial=np.inf))
    return out, gap


class Case:
    def __init__(self, logits, scores, *, select, finished=None, factor=1.0, end=-1, pad=0, offset=0):
        self.logits, self.scores, self.finished = logits, np.asarray(scores, np.float32), finished
        self.select, self.factor, self.end = select, factor, end
        batch, beams, vocab = logits.shape
        self.shape = dict(batch=batch, beams=beams, vocab=vocab, select=select)
        flat = np.full(batch * beams * (vocab + pad) + offset, np.nan, np.float32)
        flat[offset:].reshape(batch * beams, vocab + pad)[:, :vocab] = logits.reshape(-1, vocab)
        base = up(flat)
        self.bufs = dict(logits=base.view(4 * offset, flat.nbytes - 4 * offset), scores=up(self.scores))
        self.out = [up(np.full((batch, select), 77, t)) for t in (np.int32, np.int32, np.float32, np.int32)]
        self.ws = DeviceBuffer(ops.beam_select_workspace(**self.shape) + 64)
        self.ws.upload(np.full(self.ws.nbytes, 0xff, np.uint8))
        self.kw = dict(row_stride=vocab + pad, inv_temperature=factor, end_token=end,
                       finished=None if finished is None else up(i32(finished)))

    def run(self, stream=None):
        p, t, s, f = self.out
        ops.beam_select(self.bufs["logits"], self.bufs["scores"], parents=p, tokens=t, out_scores=s, out_finished=f,
                        workspace=self.ws.view(0, self.ws.nbytes - 64), stream=stream, **self.shape, **self.kw)

    def check(self, clear=True):
        got = [o.download() for o in self.out]
        want, gap = oracle(self.logits, self.scores, self.finished, self.select, np.float64(np.float32(self.factor)), self.end)
        # (the inputs leave no doubt: candidates tie exactly or are further apart than scores can be off)
        assert not clear or gap > 2 * TOL, gap
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1]) and np.array_equal(got[3], want[3])
        full = want[0] >= 0
        assert np.all(got[2][~full] == -np.inf)
        off = np.abs(got[2].astype(np.float64) - want[2])[full]
        assert np.all(off <= TOL + 2.0 ** -24 * np.abs(want[2][full])), off.max(initial=0)
        assert np.array_equal(self.ws.download()[-64:], np.full(64, 0xff, np.uint8))
        return got


def rows_of(rng, batch, beams, vocab, spread=2.5):
    return (spread * rng.standard_normal((batch, beams, vocab))).astype(np.float32)


def clear_case(seed, batch, beams, vocab, select, **kw):
    """Inputs without near ties, by the oracle alone (the first seed from `seed` on)."""
    for s in range(seed, seed + 50):
        rng = np.random.default_rng(s)
        logits, scores = rows_of(rng, batch, beams, vocab), rng.uniform(-6, 0, (batch, beams)).astype(np.float32)
        if oracle(logits, scores, kw.get("finished"), select, np.float64(np.float32(kw.get("factor", 1.0))), kw.get("end", -1))[1] > 2 * TOL:
            return Case(logits, scores, select=select, **kw)
    raise AssertionError("no clear inputs")


SHAPES = [
    # batch, beams, vocab, select
    (1, 4, 256000, 4), (1, 1, 1, 1), (1, 1, 2, 3), (2, 3, 5, 8), (3, 2, 1023, 4), (1, 5, 1025, 64), (2, 4, 4097, 8), (2, 8, 50257, 16),
    (9, 8, 151937, 16), (1, 32, 300, 64), (1, 64, 700, 64), (1, 64, 20000, 64), (2, 40, 140000, 17), (1, 33, 40, 33), (5, 1, 16384, 2), (1, 2, 1000003, 5),
]


@pytest.mark.parametrize("batch,beams,vocab,select", SHAPES)
def test_select(dev, batch, beams, vocab, select):
    print(f"[beam] {batch} {beams} {vocab} {select}", flush=True)
    c = clear_case(vocab, batch, beams, vocab, select)
    c.run()
    c.check()


@pytest.mark.parametrize("pad,offset", [(0, 1), (3, 2), (1, 3), (5, 0)])
@pytest.mark.parametrize("vocab", [1000, 9001])
def test_rows_at_any_address(dev, vocab, pad, offset):
    c = clear_case(1, 2, 3, vocab, 6, pad=pad, offset=offset, factor=0.7)
    c.run()
    c.check()


@pytest.mark.parametrize("vocab", [77, 4000, 131072])
@pytest.mark.parametrize("factor", [0.25, 1.0, 3.0])
def test_finished_beams_and_the_end_token(dev, vocab, factor):
    fin = i32([[0, 1, 0, 0], [1, 1, 1, 1], [0, 0, 0, 0]])
    c = clear_case(5, 3, 4, vocab, 8, finished=fin, factor=factor, end=min(70, vocab - 1))
    c.logits[0, 0, c.end] = c.logits[2, 1, c.end] = 30.0  # the end is what these choose
    c = Case(c.logits, c.scores, select=8, finished=fin, factor=factor, end=c.end)
    c.run()
    got = c.check(clear=False)
    assert got[3].any() and (got[0][1] >= 0).sum() == 4


@pytest.mark.parametrize("vocab", [64, 5000, 262144])
def test_ties_go_to_the_lowest_beam_then_token(dev, vocab):
    """Rows of equal logits; the same row for every beam (at other alignments); -0 and 0."""
    logits = np.zeros((2, 3, vocab), np.float32)
    logits[0, :, ::2] = -0.0
    rng = np.random.default_rng(0)
    logits[1] = np.round(rng.standard_normal(vocab)).astype(np.float32)
    c = Case(logits, np.full((2, 3), -1.5), select=7, pad=1)
    c.run()
    got = c.check(clear=False)
    assert got[0][0].tolist() == [0] * 7 and got[1][0].tolist() == list(range(7))


@pytest.mark.parametrize("vocab", [3000, 20000, 300000])
@pytest.mark.parametrize("select", [1, 16, 64])
def test_large_logits_side_by_side(dev, vocab, select):
    """The largest in few lanes: in one lane's places, rising, falling, and all in one part."""
    rng = np.random.default_rng(2)
    logits = np.float32(1e-3) * rng.permutation(4 * vocab).reshape(1, 4, vocab).astype(np.float32) / vocab
    lane = (np.arange(vocab) // 4) % 64 == 5
    logits[0, 0, lane] += 3 + np.arange(lane.sum(), dtype=np.float32) / 8
    logits[0, 1] = np.arange(vocab, dtype=np.float32) / 1024
    logits[0, 2] = -np.arange(vocab, dtype=np.float32) / 1024
    logits[0, 3, 1000:1400] += 2 + np.arange(400, dtype=np.float32) / 16
    c = Case(logits, [[0, -0.37, -0.71, -1.13]], select=select)
    c.run()
    c.check(clear=False)


def test_more_lists_than_threads_and_pool(dev):
    """64 beams: lists whose places fall together hold low logits only; all logits equal;
    more than 8192 lists."""
    rng = np.random.default_rng(11)
    scores = -0.01 * np.arange(64, dtype=np.float32)[None]
    vocab = 20000
    logits = rows_of(rng, 1, 64, vocab)
    parts = -(-vocab // 1024)
    for b in range(64):
        for p in range(parts):
            if (b * parts + p) % 64 == 5:
                logits[0, b, 1024 * p:1024 * (p + 1)] -= 50
    for x in (logits, np.full((1, 64, vocab), 2.5, np.float32)):
        c = Case(x, scores, select=64)
        c.run()
        c.check(clear=False)
    c = clear_case(12, 1, 64, 300001, 20)
    c.run()
    c.check()


def test_rows_that_offer_nothing(dev):
    rng = np.random.default_rng(3)
    logits = rows_of(rng, 6, 4, 3000)
    scores = rng.uniform(-6, 0, (6, 4)).astype(np.float32)
    logits[0, 1] = -np.inf                     # all masked
    logits[0, 2, 5:] = -np.inf                 # five tokens left
    logits[1, 0, 17], logits[1, 1, 18], logits[1, 2, 2999] = np.nan, np.inf, -np.inf
    scores[2] = [-np.inf, np.nan, np.inf, -3]
    scores[3] = -np.inf                        # nothing at all
    logits[4] = -np.inf
    logits[5, :, 2:] = -np.inf                 # fewer offers than are asked for
    logits[5, 2] = np.nan
    c = Case(logits, scores, select=16)
    c.run()
    got = c.check()
    assert (got[0][3:5] == -1).all() and (got[0][5] >= 0).sum() == 6


@pytest.mark.parametrize("scale", [1e-30, 1e4, 1e30])
def test_logits_of_any_size(dev, scale):
    rng = np.random.default_rng(4)
    logits = (rng.standard_normal((2, 3, 4096)) * scale).astype(np.float32)
    c = Case(logits, [[0, -1, -2], [0, -1, -2]], select=4)
    c.run()
    got = [o.download() for o in c.out]
    want, _ = oracle(logits, c.scores, None, 4, 1.0, -1)
    if scale > 1:
        assert np.array_equal(got[1], want[1]) and np.array_equal(got[0], want[0])
        assert np.all(np.abs(got[2] - want[2]) <= 2.0 ** -20 * np.abs(want[2]) + TOL)
    else:  # one beam's tokens are ever so slightly apart
        assert np.array_equal(got[1], want[1]) and (got[0] == [[0], [3]]).all()


@pytest.mark.parametrize("batch,beams,vocab", [(1, 4, 50000), (12, 8, 131073)])
def test_captured_select_replays(dev, batch, beams, vocab):
    s = Stream()
    c = clear_case(3, batch, beams, vocab, beams, end=2)
    g = Graph.capture(s, lambda: c.run(s))
    for _ in range(3):
        synchronize()
        g.launch(s)
        s.synchronize()
        c.check()
    g.destroy()
    s.destroy()


@pytest.mark.parametrize("vocab", [900, 30000])
def test_masked_logits_at_the_least_inverse_temperature(dev, vocab):
    logits = rows_of(np.random.default_rng(10), 2, 3, vocab)
    logits[:, :, ::3] = -np.inf
    c = Case(logits, [[-3.0, -1.0, -2.0], [0.0, -4.0, -1.0]], select=5, factor=2.0 ** -64)
    c.run()
    c.check()


@pytest.mark.parametrize("batch,beams,vocab", [(3, 4, 5000), (20, 16, 9000)])
def test_scores_and_flags_in_place(dev, batch, beams, vocab):
    rng = np.random.default_rng(9)
    fin = i32(rng.random((batch, beams)) < 0.3)
    c = clear_case(9, batch, beams, vocab, beams, finished=fin, end=4)
    c.out[2], c.out[3] = c.bufs["scores"], c.kw["finished"]
    c.run()
    got = [o.download().reshape(batch, beams) for o in c.out]
    want, _ = oracle(c.logits, c.scores, fin, beams, 1.0, 4)
    assert all(np.array_equal(got[i], want[i]) for i in (0, 1, 3))
    assert np.all(np.abs(got[2] - want[2]) <= TOL + 2.0 ** -24 * np.abs(want[2]))


def test_rows_past_four_gigabytes(dev):
    c = clear_case(13, 2, 3, 20000, 8)
    stride = (1 << 28) + 1
    far = DeviceBuffer(4 * (5 * stride + 20000))
    for r in range(6):
        far.view(4 * r * stride, 80000, np.float32, (20000,)).upload(c.logits.reshape(6, -1)[r])
    c.bufs["logits"], c.kw["row_stride"] = far, stride
    c.run()
    c.check()
    far.free()


def test_no_requests_and_no_flags(dev):
    c = clear_case(6, 2, 3, 100, 3)
    p, t, s, _ = c.out
    ops.beam_select(c.bufs["logits"], c.bufs["scores"], parents=p, tokens=t, out_scores=s, workspace=c.ws, **{**c.shape, "batch": 0})
    assert (p.download() == 77).all()
    ops.beam_select(c.bufs["logits"], c.bufs["scores"], parents=p, tokens=t, out_scores=s, workspace=c.ws.view(0, c.ws.nbytes - 64), **c.shape)
    c.out[3].upload(np.zeros((2, 3), np.int32))
    c.check()


# ---- dense states ------------------------------------------------------------------

@pytest.mark.parametrize("rows,src_rows,row_bytes,layers,pad", [(1, 1, 4, 1, 0), (6, 6, 16, 3, 16), (5, 9, 20, 2, 8), (40, 7, 4100, 4, 0), (3, 3, 70000, 2, 32),
                                                                (2, 2, 65536, 1, 0), (700, 700, 12, 5, 4)])
def test_reorder_rows(dev, rows, src_rows, row_bytes, layers, pad):
    rng = np.random.default_rng(rows)
    src = rng.integers(0, 256, (layers, src_rows * row_bytes + pad)).astype(np.uint8)
    dst = rng.integers(0, 256, (layers, rows * row_bytes + 2 * pad)).astype(np.uint8)
    parents = i32(rng.integers(-1, src_rows + 1, rows))
    d = up(dst)
    ops.beam_reorder_rows(up(src), d, up(parents), rows, row_bytes=row_bytes, layers=layers, src_rows=src_rows,
                          src_layer_stride=src.shape[1], dst_layer_stride=dst.shape[1])
    for i, p in enumerate(parents):
        if 0 <= p < src_rows:
            dst[:, i * row_bytes:(i + 1) * row_bytes] = src[:, p * row_bytes:(p + 1) * row_bytes]
    assert np.array_equal(d.download(), dst)


def test_reorder_rows_of_unaligned_buffers_and_none(dev):
    src, dst = up(np.arange(200, dtype=np.int32)), up(np.zeros(200, np.int32))
    ops.beam_reorder_rows(src.view(4, 640), dst.view(12, 640), up(i32([2, 0])), 2, row_bytes=64, layers=5)
    want = np.zeros(200, np.int32)
    for layer in range(5):
        at = 3 + 32 * layer
        want[at:at + 16] = 0
        want[at + 16:at + 32] = np.arange(1 + 32 * layer, 17 + 32 * layer)
    assert np.array_equal(dst.download(), want)
    ops.beam_reorder_rows(src, dst, up(i32([0])), 0, row_bytes=64)
    ops.beam_reorder_rows(src, dst, up(i32([0])), 1, row_bytes=64, layers=0)
    assert np.array_equal(dst.download(), want)


def test_reordered_rows_past_four_gigabytes(dev):
    """Rows of 1 MiB - 4 in layers 2.5 GiB apart."""
    row, stride = (1 << 20) - 4, 5 << 29
    src, dst = DeviceBuffer(2 * stride + 3 * row), DeviceBuffer(2 * stride + 3 * row)
    rng = np.random.default_rng(1)
    rows = [rng.integers(0, 256, (3, row)).astype(np.uint8) for _ in range(3)]
    for i, r in enumerate(rows):
        src.view(i * stride, 3 * row, np.uint8, r.shape).upload(r)
    ops.beam_reorder_rows(src, dst, up(i32([2, 0, 2])), 3, row_bytes=row, layers=3, src_layer_stride=stride, dst_layer_stride=stride)
    for i, r in enumerate(rows):
        assert np.array_equal(dst.view(i * stride, 3 * row, np.uint8, r.shape).download(), r[[2, 0, 2]])
    src.free(), dst.free()


# ---- pages -------------------------------------------------------------------------

from test_gpu_kv_pages import Host as PagesHost  # noqa: E402


class Host(PagesHost):
    def reorder(self, parents, seqs=None):
        n = len(parents)
        seqs = list(range(n)) if seqs is None else list(seqs)
        table, lens = self.table.copy(), self.lens.copy()
        heirs = {p: [] for p in range(n)}
        for i, p in enumerate(parents):
            if p >= 0:
                heirs[p].append(i)
        keeps = {p: p if p in h else h[0] for p, h in heirs.items() if h}
        part = lambda p: bool(lens[seqs[p]] % self.ps)  # noqa: E731
        mine = [i for i in range(n) if parents[i] >= 0 and part(parents[i]) and keeps[parents[i]] != i]
        ids = self.take(len(mine))
        if ids is None:
            return len(mine) - int((self.refs == 0).sum())
        for p in range(n):
            s, full = seqs[p], int(lens[seqs[p]]) // self.ps
            for page in table[s, :full]:
                self.refs[page] += len(heirs[p]) - 1
            if part(p) and not heirs[p]:
                self.refs[table[s, full]] -= 1
        for i in range(n):
            p, s = parents[i], seqs[i]
            self.table[s] = -1
            self.lens[s] = 0
            if p < 0:
                continue
            held = self.held(lens[seqs[p]])
            self.table[s, :held] = table[seqs[p], :held]
            self.lens[s] = lens[seqs[p]]
            if i in mine:
                new = ids.pop(0)
                self.page(new)[:] = self.page(self.table[s, held - 1])
                self.table[s, held - 1], self.refs[new] = new, 1
        return 0

    def go(self, parents, seqs=None, n=None, stream=None):
        ws = DeviceBuffer(ops.beam_reorder_pages_workspace(len(self.refs), len(self.lens), len(parents)))
        ws.upload(np.full(ws.nbytes, 0x17, np.uint8))
        ops.beam_reorder_pages(self.pages, up(i32(parents)), len(parents), seqs=None if seqs is None else up(i32(seqs)),
                               status=self.status, workspace=ws, stream=stream)
        synchronize()


@pytest.mark.parametrize("seqs,stride,pages,ps,page_bytes", [(1, 2, 4, 16, 48), (4, 8, 60, 16, 48), (12, 40, 700, 32, 16400), (96, 31, 4000, 64, 64),
                                                             (1500, 6, 12000, 16, 16), (300, 300, 60000, 8, 16),
                                                             (8192, 3, 30000, 16, 16)])
def test_reorder_pages(dev, seqs, stride, pages, ps, page_bytes):
    rng = np.random.default_rng(seqs)
    print(f"[reorder] {seqs} {stride} {pages} {ps}", flush=True)
    lens = rng.integers(0, (stride - 1) * ps + 1, seqs) // (2 if seqs > 100 else 1)
    h = Host(rng, seqs, stride, pages, ps, lens, page_bytes=page_bytes)
    ws = DeviceBuffer(ops.kv_pages_workspace(pages, seqs, seqs))
    for turn in range(3):
        parents = rng.integers(-1 if turn else 0, seqs, seqs)
        if turn == 1:
            parents[::2] = np.arange(seqs)[::2]  # half of them stay
        h.go(parents)
        h.same(h.reorder(parents))
        # and on from there: sequences grow by a position each
        add = (h.lens < stride * ps).astype(np.int32)
        ops.kv_pages_extend(h.pages, up(i32(np.arange(seqs))), up(add), seqs, status=h.status, workspace=ws)
        h.same(h.extend(range(seqs), add))


def test_reorder_some_slots(dev):
    """Beams in slots of any order beside sequences that stay; rotation, swap, all from one."""
    for parents in ([1, 2, 3, 0], [1, 0, 3, 2], [2, 2, 2, 2], [-1, -1, 0, 0], [0, 1, 2, 3], [3, -1, -1, -1]):
        rng = np.random.default_rng(5)
        h = Host(rng, 9, 5, 50, 16, [16, 33, 0, 70, 5, 80, 31, 48, 1])
        seqs = [7, 1, 3, 8]
        h.go(parents, seqs)
        h.same(h.reorder(parents, seqs))


def test_reorder_that_is_refused_on_the_device(dev):
    for parents, seqs in (([0, 4, 0, 0], None), ([0, 0, 0, 0], [1, 2, 9, 0]), ([0, 0, 0, 0], [1, 2, 1, 0]), ([0, 0, 0, 0], [1, 2, -1, 0])):
        rng = np.random.default_rng(6)
        h = Host(rng, 9, 5, 50, 16, [16, 33, 0, 70, 5, 80, 31, 48, 1])
        h.go(parents, seqs)
        h.same(-1)
    # pages missing: three copies, one free page
    h = Host(np.random.default_rng(7), 4, 4, 6, 16, [20, 7, 30])
    h.go([0, 0, 0, 0])
    h.same(2)
    h.go([0, 0, 2, -1])
    h.same(h.reorder([0, 0, 2, -1]))
    # a length beyond the table's row
    h.lens[0] = 16 * 4 + 1
    h.dev[1].upload(h.lens)
    h.go([0, 0, 2, -1])
    h.same(-1)


def test_reorder_without_pools_and_captured(dev):
    rng = np.random.default_rng(8)
    h = Host(rng, 6, 8, 60, 16, [100, 3, 0, 17, 48, 50])
    h.pages = ops.KvPages(*h.dev[:3], max_seqs=6, table_stride=8, num_pages=60, page_size=16)
    keep = h.data.copy()
    h.go([0, 0, 1, 1, 5, 5])
    h.reorder([0, 0, 1, 1, 5, 5])
    h.data[:] = keep
    h.same()
    # captured, with other parents between replays
    h = Host(rng, 6, 8, 60, 16, [100, 3, 0, 17, 48, 50])
    s, parents = Stream(), up(i32([0] * 6))
    ws = DeviceBuffer(ops.beam_reorder_pages_workspace(60, 6, 6))
    g = Graph.capture(s, lambda: ops.beam_reorder_pages(h.pages, parents, 6, status=h.status, workspace=ws, stream=s))
    for turn in ([1, 0, 0, 3, 3, 5], [0, 1, 2, 3, 4, 5], [5, 5, 5, 0, -1, 2]):
        parents.upload(i32(turn))
        synchronize()
        g.launch(s)
        s.synchronize()
        h.same(h.reorder(turn))
    ops.beam_reorder_pages(h.pages, parents, 0, status=h.status, workspace=ws)
    h.same()
    g.destroy()
    s.destroy()
