"""The adapters' x and y as columns of the same rows: the bits of buffers of
their own, and nothing else of the rows touched."""
import numpy as np
import pytest

from doe_amd import DeviceBuffer, ops
from test_gpu_lora import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("y_first", [False, True])
@pytest.mark.parametrize("counts,k,slice_n,rank", [([7], 136, [50, 51], 16), ([33, 1, 95], 1032, [300], 128), ([900, 300], 264, [1030, 9], 32), (None, 520, [77], 24)])
def test_in_one_buffer(dev, counts, k, slice_n, rank, y_first):
    rows = sum(counts) + 2 if counts else 40
    c = Case(k, rows, k, slice_n, rank, counts=counts)
    c.run()
    want = c.check()
    n = sum(slice_n)
    x_at = -(-(n + 3) // 4) * 4 if y_first else 4
    y_at = 1 if y_first else 4 + k
    stride = -(-(k + n + 12) // 4) * 4
    whole = np.random.default_rng(0).standard_normal((rows, stride)).astype(np.float32)
    whole[:, x_at:x_at + k], whole[:, y_at:y_at + n] = c.x, c.y
    buf = DeviceBuffer.from_array(whole)
    ops.lora_add(c.lora, c.bufs["adapters"], buf.view(4 * x_at, buf.nbytes - 4 * x_at), buf.view(4 * y_at, buf.nbytes - 4 * y_at), rows,
                 workspace=c.ws, **{**c.how, "x_row_stride": stride, "y_row_stride": stride})
    whole[:, y_at:y_at + n] = want
    assert np.array_equal(buf.download(), whole)
