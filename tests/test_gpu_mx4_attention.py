"""Attention over the 4-bit cache against the formula in 64 bits over the values
that the cache stands for (tests/mx4_cases.py derives the bounds)."""
import numpy as np
import pytest

from doe_amd import DeviceBuffer, Graph, Stream, mx4, ops, synchronize
from mx4_cases import Case, attention, check

pytestmark = pytest.mark.gpu

up = DeviceBuffer.from_array


def token(case, q, *, f16=False, scale=None, workspace=None, stream=None, **kw):
    hq = q.shape[1]
    t = np.float16 if f16 else np.float32
    out = up(np.full(q.shape, 7, t))
    ws = workspace or DeviceBuffer(ops.attention_mx4_workspace(case.batch, hq, case.h, case.d))
    ops.attention_mx4(case.cache, up(q.astype(t)), out, num_heads=hq, scale=scale or case.d ** -0.5, q_f16=f16, out_f16=f16,
                      workspace=ws, stream=stream, **kw)
    return out.download()


def prompt(case, q, rows, *, f16=False, scale=None, skip=0, behind=0, workspace=None, stride=None, **kw):
    """Rows of `q` between `skip` rows of nobody and `behind` ones, which stay as they are."""
    n, hq, d = q.shape
    t = np.float16 if f16 else np.float32
    width = stride or hq * d
    total = skip + n + behind
    wide = np.full((total, width), 3, t)
    wide[skip:skip + n, :hq * d] = q.reshape(n, -1).astype(t)
    out = up(np.full((total, width), 7, t))
    starts = up(np.cumsum([skip] + list(rows)).astype(np.int32))
    ws = workspace or DeviceBuffer(ops.attention_mx4_workspace(case.batch, hq, case.h, case.d, total))
    ops.attention_mx4_prompt(case.cache, up(wide), out, total, row_starts=starts, num_heads=hq,
                             scale=scale or case.d ** -0.5, q_f16=f16, out_f16=f16, q_row_stride=width,
                             out_row_stride=width, workspace=ws, **kw)
    got = out.download()
    assert (got[:skip] == 7).all() and (got[skip + n:] == 7).all() and (got[:, hq * d:] == 7).all()
    return got[skip:skip + n, :hq * d].reshape(q.shape)


HEADS = [(64, 8, 8), (64, 7, 1), (128, 16, 2), (128, 5, 5), (160, 8, 4), (160, 20, 2), (256, 8, 4), (256, 8, 1), (256, 24, 2),
         (512, 12, 1), (512, 2, 2)]


@pytest.mark.parametrize("d,hq,hkv", HEADS)
@pytest.mark.parametrize("f16", [False, True])
def test_tokens(dev, d, hq, hkv, f16):
    """Lengths of none and one, around blocks and pages, and long enough to be shared out."""
    rng = np.random.default_rng(d + hq)
    ps = 32 if d != 256 else 128
    case = Case(rng, [0, 1, 2, 31, 32, 33, 64, 65, 127, 300, 1025, 129], head_dim=d, num_kv_heads=hkv, page_size=ps)
    case.upload()
    q = rng.standard_normal((case.batch, hq, d)).astype(np.float16 if f16 else np.float32)
    print(f"[token] d={d} hq={hq} hkv={hkv} f16={f16}", flush=True)
    got = token(case, q, f16=f16)
    want, bound, _ = attention(case, q, [1] * case.batch, d ** -0.5)
    check(got, want, bound, got.dtype)
    assert not got[0].any()


@pytest.mark.parametrize("d,hq,hkv", [(64, 4, 2), (128, 12, 2), (160, 4, 2), (256, 4, 4), (512, 3, 1)])
@pytest.mark.parametrize("window,softcap", [(1, 0.0), (33, 0.0), (100, 20.0), (0, 5.0), (5000, 0.0)])
def test_tokens_window_and_softcap(dev, d, hq, hkv, window, softcap):
    rng = np.random.default_rng(d + window)
    case = Case(rng, [1, 33, 64, 250, 700, 0], head_dim=d, num_kv_heads=hkv, page_size=64)
    case.upload()
    q = rng.standard_normal((case.batch, hq, d)).astype(np.float32)
    print(f"[token] d={d} window={window} softcap={softcap}", flush=True)
    got = token(case, q, softcap=softcap, sliding_window=window)
    want, bound, _ = attention(case, q, [1] * case.batch, d ** -0.5, softcap, window)
    check(got, want, bound, got.dtype)


def test_tokens_long(dev):
    """One long sequence and a batch of very different lengths."""
    rng = np.random.default_rng(5)
    for lens, d, hq, hkv in (([20011], 64, 4, 1), ([9000, 1, 0, 17, 3001, 40, 900, 33], 128, 4, 2)):
        case = Case(rng, lens, head_dim=d, num_kv_heads=hkv, page_size=256)
        case.upload()
        q = rng.standard_normal((case.batch, hq, d)).astype(np.float32)
        print(f"[token] lens={lens}", flush=True)
        got = token(case, q)
        want, bound, _ = attention(case, q, [1] * case.batch, d ** -0.5)
        check(got, want, bound, got.dtype)


def test_tokens_many_sequences(dev):
    """More sequences than workgroups."""
    rng = np.random.default_rng(6)
    lens = [int(n) for n in rng.integers(0, 70, 700)]
    case = Case(rng, lens, head_dim=64, num_kv_heads=1, page_size=32)
    case.upload()
    q = rng.standard_normal((case.batch, 2, 64)).astype(np.float32)
    got = token(case, q)
    want, bound, _ = attention(case, q, [1] * case.batch, 64 ** -0.5)
    check(got, want, bound, got.dtype)


def test_tokens_sharp_and_extreme_scores(dev):
    """A softmax that falls on few positions, the largest held values, tiny
    ones, a negative scale, and scores of a wide range."""
    rng = np.random.default_rng(8)
    for scale, ks, vs in ((1.0, 1.0, 1.0), (-0.3, 1.0, 1.0), (1e-5, 9000.0, 9000.0), (3e4, 1e-5, 1e-6)):
        case = Case(rng, [500, 40], head_dim=128, num_kv_heads=2, page_size=32, k_scale=ks, v_scale=vs)
        case.upload()
        q = rng.standard_normal((2, 4, 128)).astype(np.float32)
        print(f"[token] scale={scale} k={ks} v={vs}", flush=True)
        got = token(case, q, scale=scale)
        want, bound, _ = attention(case, q, [1, 1], scale)
        check(got, want, bound, got.dtype)


@pytest.mark.parametrize("form", ["token", "prompt"])
def test_queries_of_every_size(dev, form):
    """Zero queries see the mean; queries far outside f16 keep their 22 bits."""
    rng = np.random.default_rng(9)
    case = Case(rng, [300, 77, 40], head_dim=64, num_kv_heads=1, page_size=32)
    case.upload()
    q = rng.standard_normal((3, 2, 64)).astype(np.float32)
    q[0] = 0
    q[1] *= 1e9
    q[2] *= 1e-9
    for scale in (0.1,):
        case_scale = np.array([scale, scale * 1e-9, scale * 1e9])
        for b in range(3):
            one = np.zeros_like(q)
            one[b] = q[b]
            got = token(case, one, scale=case_scale[b]) if form == "token" else prompt(case, one, [1, 1, 1], scale=case_scale[b])
            want, bound, _ = attention(case, one, [1, 1, 1], case_scale[b])
            check(got[b], want[b], bound[b], got.dtype)


def test_pages_outside_the_pool_are_not_attended(dev):
    rng = np.random.default_rng(10)
    case = Case(rng, [200, 90, 64], head_dim=128, num_kv_heads=2, page_size=32, stride=7)
    case.table[0, 2], case.table[0, 5], case.table[1, 0] = -1, case.num_pages, -2 ** 31
    case.table[2] = 2 ** 31 - 1
    case.upload()
    q = rng.standard_normal((3, 4, 128)).astype(np.float32)
    want, bound, _ = attention(case, q, [1] * 3, 0.1)
    got = token(case, q, scale=0.1)
    check(got, want, bound, got.dtype)
    assert not got[2].any()
    rows = [40, 90, 3]
    q = rng.standard_normal((sum(rows), 4, 128)).astype(np.float32)
    want, bound, _ = attention(case, q, rows, 0.1)
    got = prompt(case, q, rows, scale=0.1)
    check(got, want, bound, got.dtype)


@pytest.mark.parametrize("form", ["token", "prompt"])
def test_lengths_beyond_the_table(dev, form):
    """A length above what the table row can hold counts as that much, one below 0 as none."""
    rng = np.random.default_rng(11)
    case = Case(rng, [96, 64], head_dim=64, num_kv_heads=1, page_size=32, stride=3)
    case.lens = [150, 64]
    case.upload()
    rows = [1, 1] if form == "token" else [70, 5]
    q = rng.standard_normal((sum(rows), 2, 64)).astype(np.float32)
    want, bound, _ = attention(case, q, rows, 0.125)
    got = token(case, q, scale=0.125) if form == "token" else prompt(case, q, rows, scale=0.125)
    check(got, want, bound, got.dtype)
    case.lens_dev.upload(np.array([-5, 2 ** 31 - 1], np.int32))
    got = token(case, q[:2], scale=0.125) if form == "token" else prompt(case, q, rows, scale=0.125)
    assert np.isfinite(got).all() and not got[0].any()


def test_a_nan_block_reaches_its_own_sequence_and_head_only(dev, tile):
    rng = np.random.default_rng(12)
    case = Case(rng, [100, 100], head_dim=128, num_kv_heads=2, page_size=32)
    page = case.table[0, 1]
    case.vs[page, 1, 3, 2] = mx4.NAN_SCALE  # sequence 0, head 1, position 35, dims 64..95
    case.upload()
    q = rng.standard_normal((2, 4, 128)).astype(np.float32)
    got = token(case, q)
    assert np.isnan(got[0, 2:, 64:96]).all()
    got[0, 2:, 64:96] = 0
    assert np.isfinite(got).all()
    # behind the window it does not
    got = token(case, q, sliding_window=64)
    assert np.isfinite(got).all()
    rows = [50, 50]
    q = rng.standard_normal((100, 4, 128)).astype(np.float32)
    got = prompt(case, q, rows, sliding_window=10)
    assert np.isfinite(got[:, :2]).all() and np.isfinite(got[50:]).all()
    # of a prompt's rows it reaches those that see it, from its own position on
    case = Case(rng, [100], head_dim=128, num_kv_heads=2, page_size=32)
    case.vs[case.table[0, 1], 1, 3, 2] = mx4.NAN_SCALE
    case.ks[case.table[0, 2], 0, 6, 1] = mx4.NAN_SCALE  # position 70, head 0
    case.upload()
    q = rng.standard_normal((90, 4, 128)).astype(np.float32)
    got = prompt(case, q, [90])
    bad = np.zeros(got.shape, bool)
    bad[25:, 2:, 64:96] = True
    bad[60:, :2] = True
    assert np.array_equal(np.isnan(got), bad)
    got = prompt(case, q, [90], sliding_window=5)
    bad[30:] = False
    bad[60:65, :2] = True
    assert np.array_equal(np.isnan(got), bad)


@pytest.mark.parametrize("d,hq,hkv", [(64, 16, 2), (128, 8, 2), (160, 8, 4), (256, 8, 4), (512, 4, 2)])
@pytest.mark.parametrize("window", [0, 700])
@pytest.mark.parametrize("f16", [False, True])
def test_long_prompts(dev, tile, d, hq, hkv, window, f16):
    """Rows enough for several tiles and positions for several lists of pages;
    checked at some of the rows."""
    rng = np.random.default_rng(d + window)
    rows, lens = [300, 70], [300 + 4700, 70]
    case = Case(rng, lens, head_dim=d, num_kv_heads=hkv, page_size=32)
    case.upload()
    q = rng.standard_normal((sum(rows), hq, d)).astype(np.float16 if f16 else np.float32)
    got = prompt(case, q, rows, f16=f16, sliding_window=window)
    for at in (0, 31, 150, 299, 300, 340, 369):
        b, i = (0, at) if at < 300 else (1, at - 300)
        one = Case.__new__(Case)
        one.__dict__.update(case.__dict__, lens=[lens[b] - rows[b] + i + 1], table=case.table[b:b + 1], batch=1)
        want, bound, mass = attention(one, q[at:at + 1], [1], d ** -0.5, 0.0, window)
        check(got[at:at + 1], want, bound, got.dtype, mass if f16 else None)


@pytest.mark.parametrize("d", [64, 128, 160, 256])
def test_tokens_of_a_pool_beyond_the_last_level_cache(dev, d):
    """The form that reads past the caches gives the same bits."""
    rng = np.random.default_rng(d)
    case = Case(rng, [700, 31, 2000], head_dim=d, num_kv_heads=2, page_size=64)
    case.upload()
    q = rng.standard_normal((3, 8, d)).astype(np.float32)
    small = token(case, q)
    size = mx4.page_bytes(64, 2, d)
    case.num_pages = (300 << 20) // size
    pool = DeviceBuffer(case.num_pages * size)
    pool.view(0, case.pool.nbytes).upload(case.pages())
    case.cache = ops.Mx4Cache(pool, case.table_dev, case.lens_dev, num_pages=case.num_pages, page_size=64, num_kv_heads=2,
                              head_dim=d, batch=3, table_stride=case.stride)
    assert np.array_equal(token(case, q), small)
    pool.free()

PROMPTS = [
    # rows and lengths by sequence, head_dim, heads, page size
    ([100], [100], 128, 4, 2, 32),
    ([1, 0, 17, 64], [40, 12, 17, 200], 64, 8, 2, 64),
    ([33, 5, 0], [33, 5, 9], 160, 6, 2, 32),
    ([65, 129], [65, 400], 256, 8, 4, 128),
    ([20, 3], [50, 3], 512, 4, 1, 32),
    ([40, 300], [40, 333], 128, 5, 1, 256),
    ([5, 2, 7], [600, 1200, 7], 128, 12, 1, 64),
    ([30], [12], 64, 2, 1, 32),
    ([200, 77], [1000, 77], 64, 3, 3, 32),
]


@pytest.fixture(params=[32, 128])
def tile(request, dev):
    """Both tile sizes of the prompt's kernel (head_dim 512 has one)."""
    ops.tune("attn_mx4.tile", request.param)
    yield request.param
    ops.tune("attn_mx4.tile", 0)


@pytest.mark.parametrize("rows,lens,d,hq,hkv,ps", PROMPTS)
@pytest.mark.parametrize("f16", [False, True])
def test_prompts(dev, tile, rows, lens, d, hq, hkv, ps, f16):
    """Prompts from one row on, behind contexts of all lengths, more rows than
    positions among them; rows of nobody before and behind."""
    rng = np.random.default_rng(sum(rows) + d)
    case = Case(rng, lens, head_dim=d, num_kv_heads=hkv, page_size=ps)
    case.upload()
    q = rng.standard_normal((sum(rows), hq, d)).astype(np.float16 if f16 else np.float32)
    print(f"[prompt] rows={rows} lens={lens} d={d} hq={hq} hkv={hkv} f16={f16}", flush=True)
    got = prompt(case, q, rows, f16=f16, skip=2, behind=3, stride=hq * d + 64)
    want, bound, mass = attention(case, q, rows, d ** -0.5)
    check(got, want, bound, got.dtype, mass if f16 else None)


@pytest.mark.parametrize("d,hq,hkv", [(64, 4, 2), (128, 6, 2), (160, 4, 4), (256, 4, 2), (512, 2, 1)])
@pytest.mark.parametrize("window,softcap", [(1, 0.0), (40, 0.0), (64, 20.0), (0, 5.0), (5000, 0.0)])
def test_prompts_window_and_softcap(dev, tile, d, hq, hkv, window, softcap):
    rng = np.random.default_rng(d + window)
    rows, lens = [70, 1, 33], [150, 90, 33]
    case = Case(rng, lens, head_dim=d, num_kv_heads=hkv, page_size=64)
    case.upload()
    q = rng.standard_normal((sum(rows), hq, d)).astype(np.float32)
    print(f"[prompt] d={d} window={window} softcap={softcap}", flush=True)
    got = prompt(case, q, rows, softcap=softcap, sliding_window=window)
    want, bound, _ = attention(case, q, rows, d ** -0.5, softcap, window)
    check(got, want, bound, got.dtype)


@pytest.mark.parametrize("d", [64, 160, 512])
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("zero", [False, True])
def test_queries_with_wide_dims(dev, tile, d, f16, zero):
    """Dims of a query up to 2^11 times the others, scores in the thousands; or the
    keys are zero there: the digits hold the others to a part of the largest, and
    no worse."""
    rng = np.random.default_rng(d)
    case = Case(rng, [70, 40], head_dim=d, num_kv_heads=1, page_size=32)
    wide = np.arange(0, d, 32) + 2 * rng.integers(0, 16, d // 32)
    if zero:
        case.kc[..., wide] = 0
    case.upload()
    q = rng.standard_normal((50, 3, d)).astype(np.float16 if f16 else np.float32)
    q[..., wide] *= np.exp2(rng.integers(0, 12, q[..., wide].shape)).astype(q.dtype)
    print(f"[wide] d={d} f16={f16}", flush=True)
    got = prompt(case, q, [30, 20], f16=f16)
    want, bound, mass = attention(case, q, [30, 20], d ** -0.5, digits=2.0 ** (-19 if f16 else -24))
    check(got, want, bound, got.dtype, mass if f16 else None)
    if not f16:  # tokens carry each dim with 22 bits of its own
        got = token(case, q[:2])
        check(got, *attention(case, q[:2], [1, 1], d ** -0.5)[:2], got.dtype)


def test_a_prompt_row_equals_its_token(dev):
    """Rows of a prompt are what single tokens at the same lengths are."""
    rng = np.random.default_rng(13)
    case = Case(rng, [90], head_dim=128, num_kv_heads=2, page_size=32)
    case.upload()
    q = rng.standard_normal((90, 4, 128)).astype(np.float32)
    whole = prompt(case, q, [90])
    for n in (1, 2, 33, 64, 90):
        case.lens_dev.upload(np.array([n], np.int32))
        one = token(case, q[n - 1:n])[0]
        assert np.linalg.norm(one - whole[n - 1]) <= 2e-5 * np.linalg.norm(one)


def test_mixed_types(dev):
    """f32 queries with f16 outputs and the other way round."""
    rng = np.random.default_rng(14)
    case = Case(rng, [130, 40], head_dim=128, num_kv_heads=1, page_size=64)
    case.upload()
    for form in ("token", "prompt"):
        rows = [1, 1] if form == "token" else [66, 7]
        for qt, ot in ((np.float32, np.float16), (np.float16, np.float32)):
            q = rng.standard_normal((sum(rows), 3, 128)).astype(qt)
            out = up(np.zeros(q.shape, ot))
            how = dict(num_heads=3, scale=0.09, q_f16=qt == np.float16, out_f16=ot == np.float16)
            if form == "token":
                ws = DeviceBuffer(ops.attention_mx4_workspace(2, 3, 1, 128))
                ops.attention_mx4(case.cache, up(q), out, workspace=ws, **how)
            else:
                ws = DeviceBuffer(ops.attention_mx4_workspace(2, 3, 1, 128, len(q)))
                ops.attention_mx4_prompt(case.cache, up(q), out, len(q), row_starts=up(np.cumsum([0] + rows).astype(np.int32)),
                                         workspace=ws, **how)
            want, bound, mass = attention(case, q, rows, 0.09)
            check(out.download(), want, bound, ot, mass if form == "prompt" and ot == np.float16 else None)


def test_offsets_beyond_32_bits(dev):
    """Pages at the far end of a pool of more than 4 GiB."""
    d, h, ps = 512, 16, 256
    size = mx4.page_bytes(ps, h, d)
    pages = (1 << 32) // size + 5
    rng = np.random.default_rng(15)
    small = Case(rng, [300, 3], head_dim=d, num_kv_heads=h, page_size=ps, spare=0)
    pool = DeviceBuffer(pages * size)
    small_pages = small.pages()
    far = np.arange(pages - small.num_pages, pages, dtype=np.int32)
    for i, page in enumerate(far):
        pool.view(int(page) * size, size).upload(small_pages[i])
    table = up(np.where(small.table >= 0, far[small.table], -1).astype(np.int32))
    lens = up(np.array(small.lens, np.int32))
    cache = ops.Mx4Cache(pool, table, lens, num_pages=pages, page_size=ps, num_kv_heads=h, head_dim=d, batch=2,
                         table_stride=small.stride)
    small.cache = cache
    for rows in ([1, 1], [5, 2]):
        q = rng.standard_normal((sum(rows), h, d)).astype(np.float32)
        want, bound, _ = attention(small, q, rows, d ** -0.5)
        got = token(small, q) if rows == [1, 1] else prompt(small, q, rows)
        check(got, want, bound, got.dtype)
    kv = rng.standard_normal((2, h, d)).astype(np.float32)
    ops.mx4_kv_write(cache, up(kv), up(kv), 2)
    back = [DeviceBuffer.empty(kv.shape, np.float32) for _ in "kv"]
    ops.mx4_kv_read(cache, *back, 2)
    assert all(np.array_equal(b.download(), mx4.dequantise(*mx4.quantise(kv))) for b in back)
    pool.free()


def test_graphs_with_workspaces_of_their_own(dev):
    """Two captured steps on two streams, replayed side by side with growing
    lengths and eager work between: each replay is what the eager call gives."""
    rng = np.random.default_rng(16)
    st = [Stream(), Stream()]
    cases, qs, outs, graphs = [], [], [], []
    for i in range(2):
        case = Case(rng, [3000, 700], head_dim=128, num_kv_heads=2, page_size=64)
        case.upload()
        q, out = up(rng.standard_normal((2, 8, 128)).astype(np.float32)), DeviceBuffer.empty((2, 8, 128), np.float32)
        pq, pout = up(rng.standard_normal((9, 8, 128)).astype(np.float32)), DeviceBuffer.empty((9, 8, 128), np.float32)
        starts = up(np.array([0, 4, 9], np.int32))
        ws = DeviceBuffer(max(ops.attention_mx4_workspace(2, 8, 2, 128), ops.attention_mx4_workspace(2, 8, 2, 128, 9)))

        def step(case=case, q=q, out=out, pq=pq, pout=pout, starts=starts, ws=ws, stream=st[i]):
            ops.attention_mx4(case.cache, q, out, num_heads=8, scale=0.1, workspace=ws, stream=stream)
            ops.attention_mx4_prompt(case.cache, pq, pout, 9, row_starts=starts, num_heads=8, scale=0.1, workspace=ws,
                                     stream=stream)

        graphs.append(Graph.capture(st[i], step))
        cases.append(case)
        qs.append((q, pq, starts))
        outs.append((out, pout))
    for lens in ([3000, 700], [17, 40], [2048, 0], [1, 699], [2999, 64]):
        for case in cases:
            case.lens_dev.upload(np.array(lens, np.int32))
        synchronize()
        for g, s in zip(graphs, st):
            g.launch(s)
        for s in st:
            s.synchronize()
        got = [[o.download() for o in pair] for pair in outs]
        for i, case in enumerate(cases):
            q, pq, starts = qs[i]
            again = [DeviceBuffer.empty(o.shape, np.float32) for o in outs[i]]
            ws = DeviceBuffer(max(ops.attention_mx4_workspace(2, 8, 2, 128), ops.attention_mx4_workspace(2, 8, 2, 128, 9)))
            ops.attention_mx4(case.cache, q, again[0], num_heads=8, scale=0.1, workspace=ws)
            ops.attention_mx4_prompt(case.cache, pq, again[1], 9, row_starts=starts, num_heads=8, scale=0.1, workspace=ws)
            synchronize()
            for a, b in zip(again, got[i]):
                assert np.array_equal(a.download(), b), (lens, i)
    for g in graphs:
        g.destroy()
    for s in st:
        s.destroy()


def test_the_same_call_gives_the_same_bits(dev):
    rng = np.random.default_rng(17)
    case = Case(rng, [4000, 900, 77], head_dim=128, num_kv_heads=2, page_size=64)
    case.upload()
    q = rng.standard_normal((3, 16, 128)).astype(np.float32)
    first = token(case, q)
    assert all(np.array_equal(token(case, q), first) for _ in range(3))
    rows = [50, 20, 7]
    q = rng.standard_normal((77, 16, 128)).astype(np.float32)
    first = prompt(case, q, rows)
    assert all(np.array_equal(prompt(case, q, rows), first) for _ in range(3))
