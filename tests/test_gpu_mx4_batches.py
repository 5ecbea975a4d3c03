"""Attention over the 4-bit cache with more sequences than a wave or the device looks at
once, and prompts of one row a sequence without row_starts, against the formula in 64
bits (tests/mx4_cases.py derives the bounds)."""
import numpy as np
import pytest

from doe_amd import DeviceBuffer, Graph, Stream, mx4, ops, synchronize
from mx4_cases import Case, attention, check
from test_gpu_mx4_attention import prompt, tile, token, up  # noqa: F401  (a fixture among them)

pytestmark = pytest.mark.gpu

# sequences, (share of them, shortest, longest) of their lengths, head_dim, heads, KV heads
MANY = {
    # more rows than workgroups (768 at 64), a few of them split
    "more rows than workgroups": (1000, ((0.97, 0, 60), (0.03, 500, 3000)), 64, 2, 1),
    # the same with few sequences
    "many KV heads": (60, ((0.9, 1, 40), (0.1, 700, 1500)), 64, 16, 16),
    # rows between half and all of the workgroups, half of them split in two: more pieces
    # than workgroups
    "more pieces than workgroups": (150, ((0.5, 1, 31), (0.5, 1450, 1500)), 64, 8, 4),
    "more pieces than workgroups, few sequences": (40, ((0.5, 1, 31), (0.5, 1450, 1500)), 64, 16, 16),
    # more than one search step, every row whole or split
    "sequences beyond a wave": (130, ((0.9, 0, 300), (0.1, 2000, 4000)), 128, 2, 1),
    "head_dim 512": (70, ((0.8, 0, 40), (0.2, 400, 900)), 512, 8, 4),
    "rows of two parts of a head group": (100, ((0.9, 0, 90), (0.1, 600, 2000)), 160, 24, 2),
}


def lengths(rng, batch, shares):
    lens = np.concatenate([rng.integers(lo, hi + 1, int(round(batch * part))) for part, lo, hi in shares])
    return [int(n) for n in rng.permutation(lens)[:batch]]


@pytest.mark.parametrize("name", MANY)
@pytest.mark.parametrize("window", [0, 400])
def test_tokens_of_many_sequences(dev, name, window):
    batch, shares, d, hq, hkv = MANY[name]
    rng = np.random.default_rng(batch)
    case = Case(rng, lengths(rng, batch, shares), head_dim=d, num_kv_heads=hkv, page_size=32)
    case.upload()
    q = rng.standard_normal((case.batch, hq, d)).astype(np.float32)
    print(f"[many] {name} window={window}", flush=True)
    got = token(case, q, sliding_window=window)
    want, bound, _ = attention(case, q, [1] * case.batch, d ** -0.5, 0.0, window)
    check(got, want, bound, got.dtype)
    assert np.array_equal(token(case, q, sliding_window=window), got)


@pytest.mark.parametrize("batch,longest,d,hq,hkv", [
    (3, 3000, 128, 8, 2),      # few rows: keys split
    (150, 90, 128, 8, 2),      # none split
    (5, 500, 64, 80, 2),       # 40 heads a KV head: two tiles of 32 a row
    (40, 60, 64, 160, 1),      # 160: five of 32, two of 128
    (2, 2000, 160, 160, 1),    # and split
    (3, 700, 256, 4, 4), (2, 900, 512, 40, 1)])
@pytest.mark.parametrize("f16", [False, True])
def test_prompts_of_one_row_without_row_starts(dev, tile, batch, longest, d, hq, hkv, f16):  # noqa: F811
    rng = np.random.default_rng(batch + d)
    lens = [longest, 0] + [int(n) for n in rng.integers(1, longest, batch - 2)] if batch > 2 else [longest, 33]
    case = Case(rng, lens, head_dim=d, num_kv_heads=hkv, page_size=32)
    case.upload()
    t = np.float16 if f16 else np.float32
    q = rng.standard_normal((batch, hq, d)).astype(t)
    out = up(np.full(q.shape, 7, t))
    ws = DeviceBuffer(ops.attention_mx4_workspace(batch, hq, hkv, d, batch))
    print(f"[rows] batch={batch} d={d} hq={hq} hkv={hkv} f16={f16}", flush=True)
    ops.attention_mx4_prompt(case.cache, up(q), out, batch, num_heads=hq, scale=d ** -0.5, q_f16=f16, out_f16=f16, workspace=ws)
    want, bound, _ = attention(case, q, [1] * batch, d ** -0.5)
    check(out.download(), want, bound, t)


@pytest.mark.parametrize("batch,most,longest", [(200, 5, 90), (130, 40, 60), (67, 3, 4000)])
def test_many_short_prompts(dev, tile, batch, most, longest):  # noqa: F811
    """Sequences without rows among them, the first 64 all of that kind."""
    rng = np.random.default_rng(batch)
    rows = [0] * 64 + [int(n) for n in rng.integers(0, most + 1, batch - 64)]
    rows[-1], rows[-2] = most, 0
    lens = [n + int(rng.integers(0, longest)) for n in rows]
    case = Case(rng, lens, head_dim=64, num_kv_heads=1, page_size=32)
    case.upload()
    q = rng.standard_normal((sum(rows), 5, 64)).astype(np.float32)
    print(f"[many] batch={batch} rows={sum(rows)}", flush=True)
    got = prompt(case, q, rows, skip=3, behind=2)
    want, bound, _ = attention(case, q, rows, 0.125)
    check(got, want, bound, got.dtype)
    # and the other way round: the last sequences without rows
    case = Case(rng, lens[::-1], head_dim=64, num_kv_heads=1, page_size=32)
    case.upload()
    got = prompt(case, q, rows[::-1], skip=3, behind=2)
    want, bound, _ = attention(case, q, rows[::-1], 0.125)
    check(got, want, bound, got.dtype)


@pytest.mark.parametrize("d,hq,hkv", [(64, 8, 2), (128, 8, 2), (128, 20, 2), (160, 8, 2), (512, 4, 2)])
def test_tokens_that_may_read_past_the_caches(dev, d, hq, hkv):
    """A call that may read more than half the last-level cache gives the bits of one that
    may not, with the same table."""
    rng = np.random.default_rng(d + hq)
    size = mx4.page_bytes(64, hkv, d)
    pages = (150 << 20) // size
    case = Case(rng, [700, 31, 0, 2000], head_dim=d, num_kv_heads=hkv, page_size=64, stride=pages // 4 + 1)
    case.upload()
    q = rng.standard_normal((4, hq, d)).astype(np.float32)
    small = token(case, q)
    check(small, *attention(case, q, [1] * 4, d ** -0.5)[:2], small.dtype)
    pool = DeviceBuffer(pages * size)
    pool.view(0, case.pool.nbytes).upload(case.pages())
    case.cache = ops.Mx4Cache(pool, case.table_dev, case.lens_dev, num_pages=pages, page_size=64, num_kv_heads=hkv,
                              head_dim=d, batch=4, table_stride=case.stride)
    assert np.array_equal(token(case, q), small)
    pool.free()


def guarded(size, fill=0x5a):
    """A workspace of `size` bytes within a buffer that is `fill` around it."""
    buf = up(np.full(size + 8192, fill, np.uint8))
    return buf, buf.view(4096, size)


def intact(buf, size, fill=0x5a):
    host = buf.download()
    return (host[:4096] == fill).all() and (host[4096 + size:] == fill).all()


@pytest.mark.parametrize("d,hq,hkv", [(64, 16, 2), (128, 5, 1), (160, 40, 4), (256, 4, 4), (512, 9, 1)])
@pytest.mark.parametrize("f16", [False, True])
def test_workspaces_and_rows_are_all_that_is_written(dev, d, hq, hkv, f16):
    """Workspaces of the size asked for, queries in the wide rows of a fused projection,
    outputs in rows of another width: what lies around them stays as it was."""
    rng = np.random.default_rng(d + hq)
    rows, lens = [3, 0, 40, 1], [2000, 7, 40, 300]
    case = Case(rng, lens, head_dim=d, num_kv_heads=hkv, page_size=32)
    case.upload()
    t = np.float16 if f16 else np.float32
    how = dict(num_heads=hq, scale=d ** -0.5, q_f16=f16, out_f16=f16)
    print(f"[around] d={d} hq={hq} hkv={hkv} f16={f16}", flush=True)
    q = rng.standard_normal((4, hq, d)).astype(t)
    size = ops.attention_mx4_workspace(4, hq, hkv, d)
    buf, ws = guarded(size)
    out = up(np.full((6, hq * d), 7, t))
    ops.attention_mx4(case.cache, up(q), out.view(hq * d * out.dtype.itemsize, 4 * hq * d * out.dtype.itemsize), workspace=ws, **how)
    got = out.download()
    assert intact(buf, size) and (got[0] == 7).all() and (got[5] == 7).all()
    check(got[1:5].reshape(q.shape), *attention(case, q, [1] * 4, d ** -0.5)[:2], t)
    n, wide, narrow = sum(rows), (hq + 2 * hkv) * d, hq * d + 32
    q = rng.standard_normal((n, hq, d)).astype(t)
    fused = np.full((n, wide), np.nan, t)
    fused[:, :hq * d] = q.reshape(n, -1)
    size = ops.attention_mx4_workspace(4, hq, hkv, d, n)
    buf, ws = guarded(size)
    out = up(np.full((n + 1, narrow), 7, t))
    ops.attention_mx4_prompt(case.cache, up(fused), out, n, row_starts=up(np.cumsum([0] + rows).astype(np.int32)),
                             q_row_stride=wide, out_row_stride=narrow, workspace=ws, **how)
    got = out.download()
    assert intact(buf, size) and (got[n] == 7).all() and (got[:, hq * d:] == 7).all()
    check(got[:n, :hq * d].reshape(q.shape), *attention(case, q, rows, d ** -0.5)[:2], t)


def test_captured_calls_of_many_sequences(dev):
    """More pieces than workgroups, and prompts of one row without row_starts, captured
    and replayed with other lengths: what the eager calls give."""
    rng = np.random.default_rng(21)
    batch, d, hq, hkv = 150, 64, 8, 4
    case = Case(rng, [1500] * batch, head_dim=d, num_kv_heads=hkv, page_size=32)
    case.upload()
    q = up(rng.standard_normal((batch, hq, d)).astype(np.float32))
    size = max(ops.attention_mx4_workspace(batch, hq, hkv, d), ops.attention_mx4_workspace(batch, hq, hkv, d, batch))

    def step(outs, ws, stream=None):
        ops.attention_mx4(case.cache, q, outs[0], num_heads=hq, scale=0.1, workspace=ws, stream=stream)
        ops.attention_mx4_prompt(case.cache, q, outs[1], batch, num_heads=hq, scale=0.1, workspace=ws, stream=stream)

    st, outs, ws = Stream(), [DeviceBuffer.empty((batch, hq, d), np.float32) for _ in "tp"], DeviceBuffer(size)
    graph = Graph.capture(st, lambda: step(outs, ws, st))
    for name in ("more pieces than workgroups", "more rows than workgroups", "sequences beyond a wave"):
        lens = np.minimum(1500, lengths(rng, batch, MANY[name][1])).astype(np.int32)
        case.lens_dev.upload(lens)
        synchronize()
        graph.launch(st)
        st.synchronize()
        got = [o.download() for o in outs]
        again = [DeviceBuffer.empty((batch, hq, d), np.float32) for _ in "tp"]
        other = DeviceBuffer(size)
        step(again, other)
        synchronize()
        for a, b in zip(again, got):
            assert np.array_equal(a.download(), b), name
        # a token is a prompt of one row
        assert np.linalg.norm(got[0] - got[1]) <= 2e-6 * np.linalg.norm(got[0])
    graph.destroy()
    st.destroy()
