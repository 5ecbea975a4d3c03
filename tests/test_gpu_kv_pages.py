"""The pages of a paged cache: every call against the same on the host, the
calls that are refused on the device, and a run of them with the 4-bit cache
as a serving program makes it."""
import numpy as np
import pytest

from doe_amd import DeviceBuffer, Graph, Stream, mx4, ops, synchronize
from mx4_cases import check

pytestmark = pytest.mark.gpu

up = DeviceBuffer.from_array
i32 = lambda x: np.asarray(x, np.int32)  # noqa: E731


class Host:
    """The pages on the host and on the device."""

    def __init__(self, rng, seqs, stride, pages, ps, lens=(), layers=2, page_bytes=48, extra=0):
        self.table = np.full((seqs, stride), -1, np.int32)
        self.lens, self.refs, self.ps = np.zeros(seqs, np.int32), np.zeros(pages, np.int32), ps
        ids = list(rng.permutation(pages))
        for s, n in enumerate(lens):
            self.lens[s] = n
            for i in range(-(-n // ps)):
                self.table[s, i] = ids.pop()
                self.refs[self.table[s, i]] = 1
        self.data = rng.integers(0, 256, (layers, pages * page_bytes + extra)).astype(np.uint8)
        self.layers, self.page_bytes, self.extra = layers, page_bytes, extra
        self.dev = [up(x) for x in (self.table, self.lens, self.refs, self.data)]
        self.status = up(i32([77]))
        self.ws = DeviceBuffer(ops.kv_pages_workspace(pages, seqs, 4096))
        self.ws.upload(rng.integers(0, 40, self.ws.nbytes // 4).astype(np.int32).view(np.uint8))  # leftovers of other calls
        self.pages = ops.KvPages(*self.dev[:3], max_seqs=seqs, table_stride=stride, num_pages=pages, page_size=ps,
                                 pools=self.dev[3], layers=layers, page_bytes=page_bytes,
                                 layer_stride=pages * page_bytes + extra)

    def page(self, p):
        return self.data[:, p * self.page_bytes:(p + 1) * self.page_bytes]

    def held(self, n):
        return -(-int(n) // self.ps)

    def take(self, n):
        free = np.flatnonzero(self.refs == 0)
        return list(free[:n]) if len(free) >= n else None

    def same(self, status=0):
        table, lens, refs, data = (d.download() for d in self.dev)
        assert self.status.download()[0] == status
        assert np.array_equal(lens, self.lens) and np.array_equal(refs, self.refs)
        assert np.array_equal(table, self.table)
        assert np.array_equal(data, self.data)

    # the operations on the host, entry by entry
    def extend(self, seqs, add):
        want = sum(self.held(self.lens[s] + a) - self.held(self.lens[s]) for s, a in zip(seqs, add))
        ids = self.take(want)
        if ids is None:
            return want - int((self.refs == 0).sum())
        for s, a in zip(seqs, add):
            for i in range(self.held(self.lens[s]), self.held(self.lens[s] + a)):
                self.table[s, i] = ids.pop(0)
                self.refs[self.table[s, i]] = 1
            self.lens[s] += a
        return 0

    def fork(self, parents, children):
        want = sum(bool(self.lens[p] % self.ps) for p in parents)
        ids = self.take(want)
        if ids is None:
            return want - int((self.refs == 0).sum())
        for p, c in zip(parents, children):
            n, full = int(self.lens[p]), int(self.lens[p]) // self.ps
            self.table[c] = -1
            self.table[c, :full] = self.table[p, :full]
            for page in self.table[p, :full]:
                self.refs[page] += 1
            if n % self.ps:
                new = ids.pop(0)
                self.table[c, full], self.refs[new] = new, 1
                self.page(new)[:] = self.page(self.table[p, full])
            self.lens[c] = n
        return 0

    def free(self, seqs):
        for s in seqs:
            for i in range(self.held(self.lens[s])):
                self.refs[self.table[s, i]] -= 1
            if self.lens[s]:
                self.table[s] = -1
            self.lens[s] = 0

    def compact(self):
        live = int((self.refs > 0).sum())
        high, low = [p for p in range(live, len(self.refs)) if self.refs[p]], [p for p in range(live) if not self.refs[p]]
        assert len(high) == len(low)
        to = dict(zip(high, low))
        for a, b in to.items():
            self.page(b)[:] = self.page(a)
            self.refs[b], self.refs[a] = self.refs[a], 0
        for s in range(len(self.lens)):
            for i in range(self.held(self.lens[s])):
                self.table[s, i] = to.get(self.table[s, i], self.table[s, i])


@pytest.mark.parametrize("seqs,pages,ps,n", [(6, 40, 16, 5), (1, 3, 32, 1), (300, 9000, 64, 300), (2500, 6000, 16, 2100)])
def test_extend(dev, seqs, pages, ps, n):
    rng = np.random.default_rng(seqs)
    lens = rng.integers(0, 2 * ps + 1, seqs) if seqs > 1 else [5]
    h = Host(rng, seqs, 8, pages, ps, lens)
    who = rng.permutation(seqs)[:n]
    add = rng.integers(0, 2 * ps, n)
    add[0] = 0 if n > 1 else 1
    print(f"[extend] {seqs} {pages} {ps} {n}", flush=True)
    ops.kv_pages_extend(h.pages, up(i32(who)), up(i32(add)), n, status=h.status, workspace=h.ws)
    h.same(h.extend(who, add))
    # once more, from there
    ops.kv_pages_extend(h.pages, up(i32(who)), up(i32(np.ones(n))), n, status=h.status, workspace=h.ws)
    h.same(h.extend(who, [1] * n))


def test_extend_that_does_not_fit_changes_nothing(dev):
    rng = np.random.default_rng(2)
    h = Host(rng, 4, 6, 10, 16, [16, 90, 0, 5])
    for who, add, status in (([0, 2], [33, 16], None), ([1], [7], -1), ([0, 0], [1, 1], -1), ([4], [1], -1), ([-1], [1], -1),
                             ([0], [-1], -1), ([3, 0, 2], [1, 2, 3], None), ([0], [2 ** 31 - 1], -1), ([], [], None)):
        print(f"[extend] {who} {add}", flush=True)
        ops.kv_pages_extend(h.pages, up(i32(who + [0])), up(i32(add + [0])), len(who), status=h.status, workspace=h.ws)
        h.same(h.extend(who, add) if status is None else status)
    assert h.extend([2], [60]) > 0


@pytest.mark.parametrize("seqs,forks,ps,page_bytes,extra", [(5, 3, 16, 48, 16), (1, 1, 32, 16, 0), (40, 20, 16, 4352, 0),
                                                            (3, 2, 16, 40016, 160)])
def test_fork(dev, seqs, forks, ps, page_bytes, extra):
    rng = np.random.default_rng(seqs)
    lens = list(rng.integers(0, 5 * ps, seqs))
    lens[0] = 3 * ps
    if seqs > 2:
        lens[1], lens[2] = 0, 3 * ps + 1
    slots = seqs * (1 + forks)
    h = Host(rng, slots, 6, seqs * (5 + forks) + 7, ps, lens, layers=3, page_bytes=page_bytes, extra=extra)
    children = seqs + rng.permutation(slots - seqs)
    parents = np.arange(len(children)) % seqs
    print(f"[fork] {seqs} x {forks}", flush=True)
    ops.kv_pages_fork(h.pages, up(i32(parents)), up(i32(children)), len(children), status=h.status, workspace=h.ws)
    h.same(h.fork(parents, children))


def test_fork_that_is_not_in_order_changes_nothing(dev):
    rng = np.random.default_rng(3)
    h = Host(rng, 8, 4, 9, 16, [20, 33, 0, 16, 0])
    for parents, children, status in (([0], [1], -1), ([0, 1], [5, 5], -1), ([0], [8], -1), ([8], [5], -1), ([-1], [5], -1),
                                      ([0], [-3], -1), ([0, 2], [2, 5], -1), ([2], [2], -1), ([0, 0, 0, 1], [4, 5, 6, 7], None),
                                      ([], [], None), ([2, 3], [5, 6], None), ([0, 6], [7, 4], None)):
        print(f"[fork] {parents} {children}", flush=True)
        ops.kv_pages_fork(h.pages, up(i32(parents + [0])), up(i32(children + [0])), len(parents), status=h.status,
                          workspace=h.ws)
        h.same(h.fork(parents, children) if status is None else status)


def test_free(dev):
    rng = np.random.default_rng(4)
    h = Host(rng, 50, 7, 300, 16, [0, 1, 16, 17, 100] + list(rng.integers(0, 112, 30)))
    ops.kv_pages_fork(h.pages, up(i32([4, 3])), up(i32([40, 41])), 2, status=h.status, workspace=h.ws)
    h.same(h.fork([4, 3], [40, 41]))
    for seqs, status in (([1], 0), ([4, 7, 7, 0, 7], 0), ([40, 50, 2, -1], -1), ([], 0), (list(range(50)), 0)):
        print(f"[free] {seqs}", flush=True)
        ops.kv_pages_free(h.pages, up(i32(seqs + [0])), len(seqs), status=h.status)
        h.free([s for s in seqs if 0 <= s < 50])
        h.same(status)
    assert not h.refs.any()


@pytest.mark.parametrize("seqs,pages,layers,page_bytes,extra", [(10, 100, 2, 48, 16), (1, 5, 1, 16, 0), (60, 7000, 1, 16, 0),
                                                                (30, 200, 5, 20000, 0)])
def test_compact(dev, seqs, pages, layers, page_bytes, extra):
    rng = np.random.default_rng(pages)
    h = Host(rng, seqs + 4, 9, pages, 16, list(rng.integers(0, 49, seqs)), layers=layers, page_bytes=page_bytes, extra=extra)
    if seqs > 1:  # shared pages move once, for all who hold them
        ops.kv_pages_fork(h.pages, up(i32([0, 1, 1])), up(i32(seqs + np.arange(3))), 3, status=h.status, workspace=h.ws)
        h.same(h.fork([0, 1, 1], seqs + np.arange(3)))
    for _ in range(2):
        print(f"[compact] {seqs} {pages}", flush=True)
        ops.kv_pages_compact(h.pages, status=h.status, workspace=h.ws)
        h.compact()
        h.same()
        gone = list(range(0, seqs, 2))
        ops.kv_pages_free(h.pages, up(i32(gone)), len(gone), status=h.status)
        h.free(gone)
    ops.kv_pages_free(h.pages, up(i32(np.arange(seqs + 4))), seqs + 4, status=h.status)
    h.free(range(seqs + 4))
    ops.kv_pages_compact(h.pages, status=h.status, workspace=h.ws)
    h.same()


def test_bookkeeping_without_pools(dev):
    rng = np.random.default_rng(5)
    h = Host(rng, 8, 6, 30, 16, [20, 33, 16, 5, 80])
    p = ops.KvPages(*h.dev[:3], max_seqs=8, table_stride=6, num_pages=30, page_size=16)
    before = h.data.copy()
    ops.kv_pages_fork(p, up(i32([0])), up(i32([6])), 1, status=h.status, workspace=h.ws)
    h.fork([0], [6])
    ops.kv_pages_free(p, up(i32([1])), 1, status=h.status)
    h.free([1])
    ops.kv_pages_compact(p, status=h.status, workspace=h.ws)
    h.compact()
    h.data = before
    h.same()


def test_extend_among_very_many_sequences(dev):
    """More sequences than are marked in LDS; more entries, and more pages, than are kept there."""
    rng = np.random.default_rng(70000)
    h = Host(rng, 70000, 2, 9000, 16, [16 * (i % 2) + i % 3 for i in range(4000)])
    for n in (1, 1500, 3000):
        seqs, add = rng.choice(70000, n, replace=False), rng.integers(0, 15, n)
        add = np.minimum(add, 32 - h.lens[seqs])
        print(f"[extend] 70000 sequences, {n} entries", flush=True)
        ops.kv_pages_extend(h.pages, up(i32(seqs)), up(i32(add)), n, status=h.status, workspace=h.ws)
        h.same(h.extend(seqs, add))
    for seqs in ([69999, 5, 69999], [70000], [-1]):
        ops.kv_pages_extend(h.pages, up(i32(seqs)), up(i32([1] * len(seqs))), len(seqs), status=h.status, workspace=h.ws)
        h.same(-1)


def test_fork_and_compact_of_many_pages(dev):
    """More copies than are kept in LDS."""
    rng = np.random.default_rng(2)
    h = Host(rng, 4000, 2, 9000, 16, [1 + i % 31 for i in range(1900)] + [0] * 2100)
    parents, children = rng.integers(0, 1900, 1800), 1900 + rng.permutation(2100)[:1800]
    ops.kv_pages_fork(h.pages, up(i32(parents)), up(i32(children)), 1800, status=h.status, workspace=h.ws)
    h.same(h.fork(parents, children))
    gone = rng.choice(3700, 1200, replace=False)
    ops.kv_pages_free(h.pages, up(i32(gone)), 1200, status=h.status)
    h.free(gone)
    h.same()
    ops.kv_pages_compact(h.pages, status=h.status, workspace=h.ws)
    h.compact()
    h.same()


def test_free_and_compact_of_a_damaged_state(dev):
    """A length beyond the table row counts as what the row holds; a page with a
    count below 0 is in use for all that moves."""
    rng = np.random.default_rng(8)
    h = Host(rng, 3, 4, 20, 16, [64, 30, 0])
    h.dev[1].upload(i32([2**31 - 1, 30, 0]).view(np.uint8))
    ops.kv_pages_free(h.pages, up(i32([0])), 1, status=h.status)
    h.free([0])
    h.same()
    h.refs[h.table[1, :2]] = -3
    h.dev[2].upload(h.refs.view(np.uint8))
    h.refs = np.abs(h.refs)
    ops.kv_pages_compact(h.pages, status=h.status, workspace=h.ws)
    h.compact()
    h.refs = -h.refs
    h.same()


def test_copy(dev):
    rng = np.random.default_rng(6)
    h = Host(rng, 1, 1, 50, 16, layers=3, page_bytes=16400, extra=48)
    ids = rng.permutation(50)
    how = dict(layers=3, num_pages=50, page_bytes=16400, layer_stride=50 * 16400 + 48, status=h.status, workspace=h.ws)
    for src, dst, status in ((ids[:20], ids[20:40], 0), ([3, 3, 3], [1, 0, 9], 0), ([1, 2], [5, 5], -1), ([1, 2], [2, 3], -1),
                             ([4], [4], -1), ([50], [1], -1), ([1], [-1], -1), ([], [], 0), ([7], [8], 0)):
        src, dst = list(src), list(dst)
        print(f"[copy] {len(src)} {status}", flush=True)
        ops.kv_pages_copy(h.dev[3], up(i32(src + [0])), up(i32(dst + [0])), len(src), **how)
        if status == 0:
            for a, b in zip(src, dst):
                h.page(b)[:] = h.page(a)
        h.same(status)


def test_captured_calls_follow_the_state(dev):
    """extend, fork, free and compact in one graph, replayed with other lists and
    eager calls between."""
    rng = np.random.default_rng(7)
    h = Host(rng, 12, 8, 70, 16, [20, 33, 16, 5, 80])
    grow, add, parent, child, end = (up(i32(x)) for x in ([0, 1], [1, 1], [0], [8], [8]))
    st = Stream()

    def body():
        ops.kv_pages_extend(h.pages, grow, add, 2, status=h.status, workspace=h.ws, stream=st)
        ops.kv_pages_fork(h.pages, parent, child, 1, status=h.status, workspace=h.ws, stream=st)
        ops.kv_pages_free(h.pages, end, 1, status=h.status, stream=st)
        ops.kv_pages_compact(h.pages, status=h.status, workspace=h.ws, stream=st)

    graph = Graph.capture(st, body)
    for g, a, p, c, e in (([0, 1], [1, 1], [0], [8], [3]), ([4, 2], [30, 16], [4], [9], [0]), ([1, 9], [14, 3], [2], [3], [4])):
        for buf, x in ((grow, g), (add, a), (parent, p), (child, c), (end, e)):
            buf.upload(i32(x))
        synchronize()
        graph.launch(st)
        st.synchronize()
        h.extend(g, a)
        h.fork(p, c)
        h.free(e)
        h.compact()
        h.same()
        ops.kv_pages_extend(h.pages, up(i32([11])), up(i32([1])), 1, status=h.status, workspace=h.ws)
        h.same(h.extend([11], [1]))
    graph.destroy()
    st.destroy()


def plain(k, v, q, scale):
    """(out, bound) of one query over values k, v [n][D] in 64 bits."""
    s = k @ q * scale
    p = np.exp(s - s.max())
    p /= p.sum()
    ds = np.max(np.abs(k) @ np.abs(q)) * scale * (2.0 ** -22 + (k.shape[1] / 16 + 9) * 2.0 ** -24)
    return p @ v, (2 * ds + 2.0 ** -16 + 2.0 ** -18) * (p @ np.abs(v))


@pytest.mark.parametrize("d,hq,hkv,ps", [(128, 4, 2, 32), (256, 4, 1, 64), (64, 3, 3, 32)])
def test_serving_run(dev, d, hq, hkv, ps):
    """Two layers, prompts, steps, two samples of one prompt, an end, compaction,
    more steps: after each, attention is what the held values give."""
    rng = np.random.default_rng(d)
    layers, slots, stride, pages, scale = 2, 6, 8, 40, d ** -0.5
    size = mx4.page_bytes(ps, hkv, d)
    pool = DeviceBuffer(layers * pages * size)
    table, lens, refs = up(np.full((slots, stride), -1, np.int32)), up(np.zeros(slots, np.int32)), up(np.zeros(pages, np.int32))
    status = up(i32([0]))
    ws = DeviceBuffer(ops.kv_pages_workspace(pages, slots, slots))
    kv = ops.KvPages(table, lens, refs, max_seqs=slots, table_stride=stride, num_pages=pages, page_size=ps, pools=pool,
                     layers=layers, page_bytes=size)
    cache = [ops.Mx4Cache(pool.view(i * pages * size, pages * size), table, lens, num_pages=pages, page_size=ps,
                          num_kv_heads=hkv, head_dim=d, batch=slots, table_stride=stride) for i in range(layers)]
    held = [[[np.zeros((0, hkv, d)) for _ in "kv"] for _ in range(slots)] for _ in range(layers)]

    def step(rows, prompt):
        """rows[s] new tokens for slot s: pages, K / V, attention."""
        who = [s for s in range(slots) if rows[s]]
        ops.kv_pages_extend(kv, up(i32(who)), up(i32([rows[s] for s in who])), len(who), status=status, workspace=ws)
        n = sum(rows) if prompt else slots
        starts = np.cumsum([0] + rows).astype(np.int32)
        for i in range(layers):
            k, v = (rng.standard_normal((n, hkv, d)).astype(np.float32) for _ in "kv")
            q = rng.standard_normal((n, hq, d)).astype(np.float32)
            out = up(np.zeros(q.shape, np.float32))
            how = dict(num_heads=hq, scale=scale)
            if prompt:
                ops.mx4_kv_write(cache[i], up(k), up(v), n, row_starts=up(starts))
                aw = DeviceBuffer(ops.attention_mx4_workspace(slots, hq, hkv, d, n))
                ops.attention_mx4_prompt(cache[i], up(q), out, n, row_starts=up(starts), workspace=aw, **how)
            else:  # every slot in use takes a token
                ops.mx4_kv_write(cache[i], up(k), up(v), n)
                aw = DeviceBuffer(ops.attention_mx4_workspace(slots, hq, hkv, d))
                ops.attention_mx4(cache[i], up(q), out, workspace=aw, **how)
            got = out.download()
            assert status.download()[0] == 0
            for s in range(slots):
                for j in range(rows[s]):
                    at = starts[s] + j if prompt else s
                    for x, new in zip(range(2), (k, v)):
                        value = mx4.dequantise(*mx4.quantise(new[at])).astype(np.float64)
                        held[i][s][x] = np.concatenate([held[i][s][x], value[None]])
                    for head in range(hq):
                        kk, vv = (held[i][s][x][:, head * hkv // hq] for x in range(2))
                        want, bound = plain(kk, vv, q[at, head].astype(np.float64), scale)
                        check(got[at, head], want, bound, np.float32)
                if not prompt and not rows[s]:
                    assert not got[s].any()

    step([ps + 5, 0, 40, 2 * ps, 0, 0], True)
    step([1, 0, 1, 1, 0, 0], False)
    ops.kv_pages_fork(kv, up(i32([0, 0, 3])), up(i32([1, 4, 5])), 3, status=status, workspace=ws)
    for layer in held:
        layer[1], layer[4], layer[5] = ([x.copy() for x in layer[s]] for s in (0, 0, 3))
    step([1] * 6, False)
    ops.kv_pages_free(kv, up(i32([0, 2])), 2, status=status)
    for layer in held:
        layer[0] = [np.zeros((0, hkv, d)) for _ in "kv"]
        layer[2] = [np.zeros((0, hkv, d)) for _ in "kv"]
    ops.kv_pages_compact(kv, status=status, workspace=ws)
    live = int((refs.download() > 0).sum())
    assert (refs.download()[:live] > 0).all()
    step([0, 1, 0, 1, 1, 1], False)
    step([33, 3, 0, 0, 10, 0], True)
    step([1, 1, 0, 1, 1, 1], False)
