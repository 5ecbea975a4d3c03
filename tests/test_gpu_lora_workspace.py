"""Calls of the adapters in workspaces of just the size that they ask for: what
lies behind stays as it was (bounds as in ``test_gpu_lora``)."""
import numpy as np
import pytest

from doe_amd import ops
from test_gpu_lora import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("counts,k,slice_n,rank", [
    ([1200, 31, 0, 270], 640, [40, 50, 60, 70], 128),  # one copy of t
    ([200, 120], 4224, [300], 64), ([255], 2056, [1200], 64), ([31, 290], 1032, [900, 200], 128),  # two to eight
    ([9, 60, 3], 17504, [700, 300, 41], 32), ([5, 6, 4, 9, 3], 17504, [3000, 2000, 2576], 32),
])
@pytest.mark.parametrize("bf16", [False, True], ids=["f16", "bf16"])
def test_workspaces_to_their_bounds(dev, counts, k, slice_n, rank, bf16):
    print(f"[lora] {counts} {k} {slice_n} {rank}", flush=True)
    c = Case(k, sum(counts), k, slice_n, rank, bf16=bf16, counts=counts)
    c.run()
    c.check()


def test_fewer_rows_in_the_same_workspace(dev):
    """A program's one workspace, of its most rows, under calls that split k further."""
    most = Case(1, 2000, 4224, [500, 600], 64, counts=[2000])
    ws = most.ws
    for rows in (2000, 700, 256, 100, 40, 8):
        c = Case(rows, rows, 4224, [500, 600], 64, counts=[rows])
        assert ops.lora_workspace(c.lora, rows) <= ops.lora_workspace(most.lora, 2000)
        ws.upload(np.full(ws.nbytes, 0xff, np.uint8))
        c.ws = ws
        c.run()
        c.check()
