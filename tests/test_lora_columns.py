"""x and y of the adapters as columns of one buffer: taken where no column is in
both, refused otherwise (CPU only)."""
import pytest

from doe_amd import ops
from test_mx4 import BIG, refused

K, N, STRIDE, ROWS, AT = 64, 40, 112, 5, 1 << 40


def at(ptr, nbytes=1 << 40):
    return type("B", (), dict(nbytes=nbytes, ptr=ptr))()


def add(x, y, x_stride=STRIDE, y_stride=STRIDE, rows=ROWS):
    lora = ops.Lora(BIG, BIG, None, num_adapters=3, rank=16, k=K, slice_n=[N])
    ops.lora_add(lora, BIG, at(AT + 4 * x), at(AT + 4 * y), rows, workspace=at(1 << 50, 16), x_row_stride=x_stride, y_row_stride=y_stride)


@pytest.mark.parametrize("x,y", [(0, K), (0, STRIDE - N), (40, 0), (48, 8), (STRIDE, K), (0, STRIDE + K), (3 * STRIDE + 40, 0), (0, K + 9 * STRIDE),
                                 (48, 1), (0, 4 * STRIDE + K)])
def test_columns_apart_are_taken(x, y):
    """... and then refused for want of a workspace."""
    refused("workspace of", add, x, y)


@pytest.mark.parametrize("x,y,how", [
    (0, 0, {}), (0, K - 1, {}), (0, STRIDE - N + 1, {}), (40, 1, {}), (48, 9, {}), (STRIDE, K - 1, {}), (0, STRIDE, {}), (0, 2 * STRIDE + 5, {}),
    (0, K, dict(y_stride=STRIDE + 4)), (0, K, dict(x_stride=STRIDE + 4)), (40, 0, dict(y_stride=STRIDE - 4)), (0, 1, dict(rows=1)),
])
def test_columns_in_both_are_refused(x, y, how):
    refused("apart", add, x, y, **how)
