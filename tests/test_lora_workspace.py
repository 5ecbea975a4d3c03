"""The adapters' workspace: the copies of t that a call can write, and no more
(CPU only)."""
import pytest

from doe_amd import ops
from test_mx4 import BIG


def size(rows, rank=16, slices=1, k=2304, n=4096):
    lora = ops.Lora(BIG, BIG, None, num_adapters=4, rank=rank, k=k, slice_n=[n // slices] * slices)
    return ops.lora_workspace(lora, rows)


@pytest.mark.parametrize("rows,rank,slices", [(6000, 128, 4), (4799, 128, 4), (100000, 8, 1), (8192, 64, 1), (1024, 256, 4)])
def test_long_prompts_take_one_copy(rows, rank, slices):
    assert size(rows, rank, slices) == 4 * rows * rank * slices


def splits(rows, rank, slices, k, segments):
    """Splits of k that a call in tiles takes: up to eight, two steps of 32 for each of eight
    waves, workgroups for 256 CUs."""
    wgs = (rows // 32 + segments) * -(-rank * slices // 64)
    return max(1, min(8, 256 // wgs, -(-k // 32) // 16))


@pytest.mark.parametrize("rank,slices", [(8, 1), (16, 4), (24, 3), (64, 2), (128, 4), (256, 1), (256, 4)])
@pytest.mark.parametrize("k", [8, 520, 1032, 2304, 21504])
def test_every_split_has_its_place_and_fewer_rows_fit(rank, slices, k):
    last = 0
    for rows in [*range(1, 400), 511, 512, 513, 1000, 2047, 4096, 4097, 8191, 8192, 20000, 1 << 20]:
        now = size(rows, rank, slices, k)
        assert now >= 4 * rows * rank * slices * splits(rows, rank, slices, k, 1)
        assert now >= last  # (a workspace of a program's most rows serves all its calls)
        assert now <= 4 * rank * slices * max(rows, min(8 * rows, 8192 // -(-rank * slices // 64)))
        last = now
