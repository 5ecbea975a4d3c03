"""Rows rotated and appended where the angles end inside a page and inside four
positions: those behind append nothing and leave their neighbours' bytes."""
import numpy as np
import pytest

from doe_amd import mx4, ops
from test_gpu_rope_append import Case, rotate

pytestmark = pytest.mark.gpu


def check_mx4(c):
    """Every sequence's positions below the limit as ``mx4.quantise`` codes the rotated rows, all others as before."""
    x = c.qkv[:, :c.width].reshape(c.rows, -1, c.d)
    turned, want_q, kv = x.copy(), c.q.copy(), c.hq
    parts = [p.copy() for p in mx4.unpack_pages(c.pool, c.ps, c.hkv, c.d)]
    for row, pos, page in c.places():
        if 0 <= pos < c.positions:
            turned[row, :kv + c.hkv, :c.rot] = rotate(x[row:row + 1, :kv + c.hkv, :c.rot], c.freq[pos:pos + 1], c.interleaved)[0]
        want_q[row, :kv * c.d] = turned[row, :kv].reshape(-1).astype(want_q.dtype)
        if page >= 0:
            for j, values in enumerate((turned[row, kv:kv + c.hkv], x[row, kv + c.hkv:])):
                codes, scales = mx4.quantise(values)
                parts[2 * j][page, :, pos % c.ps], parts[2 * j + 1][page, :, pos % c.ps] = codes, scales
    assert np.array_equal(c.dq.download(), want_q)
    assert np.array_equal(c.dpools[0].download(), mx4.pack_pages(*parts))


@pytest.mark.parametrize("mx4_cache", [False, True], ids=["f16", "mx4"])
@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "pairs"])
@pytest.mark.parametrize("d", [64, 128, 160, 256, 512])
@pytest.mark.parametrize("positions", [1, 61, 62, 63, 65])
def test_ragged_rows(dev, positions, d, interleaved, mx4_cache):
    lens, counts = [70, 90, 64, 66, 3], [70, 33, 5, 1, 3]
    c = Case(positions, lens, counts, hq=2, hkv=2, d=d, ps=32, positions=positions, interleaved=interleaved, mx4_cache=mx4_cache)
    c.run()
    check_mx4(c) if mx4_cache else c.check()


@pytest.mark.parametrize("mx4_cache", [False, True], ids=["f16", "mx4"])
@pytest.mark.parametrize("d", [64, 160, 256, 512])
@pytest.mark.parametrize("rot", [16, None])
def test_one_row_a_sequence(dev, rot, d, mx4_cache):
    """Sequences that end at every place around the limit."""
    lens = list(range(59, 69)) + [1, 2, 32, 33]
    c = Case(d, lens, [1] * len(lens), hq=2, hkv=1, d=d, ps=32, positions=63, rot=rot, mx4_cache=mx4_cache, starts=False)
    c.run()
    check_mx4(c) if mx4_cache else c.check()


@pytest.mark.parametrize("d", [64, 256])
def test_no_positions_at_all(dev, d):
    """Without a table of angles queries come as they are and nothing is appended."""
    c = Case(d, [40, 7], [9, 7], hq=2, hkv=1, d=d, ps=32, positions=0, mx4_cache=True)
    ops.qkv_rope_append(c.cache, c.dqkv, c.dq, c.rows, num_heads=2, freq_cis=None, max_positions=0, row_starts=c.row_starts)
    check_mx4(c)
