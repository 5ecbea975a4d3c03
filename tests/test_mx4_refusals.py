"""Arguments of the 4-bit cache's calls at the ends of their ranges (CPU only)."""
import numpy as np
import pytest

from doe_amd import mx4, ops
from test_mx4 import BIG, cache, refused


@pytest.mark.parametrize("bad", [dict(scale=3e38), dict(scale=-3e38), dict(scale=1.0, softcap=3e38)])
def test_factors_that_overflow_in_powers_of_two(bad):
    """scale log2(e) and softcap log2(e) are what the kernels multiply by."""
    c, how = cache(), dict(num_heads=8, scale=0.1, workspace=BIG)
    refused("above 2.35e38", ops.attention_mx4, c, BIG, BIG, **{**how, **bad})
    refused("above 2.35e38", ops.attention_mx4_prompt, c, BIG, BIG, 500, row_starts=BIG, **{**how, **bad})


def test_no_rows_and_no_pages_are_valid():
    codes, scales = mx4.quantise(np.zeros((0, 3, 128), np.float32))
    assert codes.shape == (0, 3, 128) and scales.shape == (0, 3, 4)
    assert mx4.dequantise(codes, scales).shape == (0, 3, 128)
    parts = [np.zeros((0, 2, 32, n), np.uint8) for n in (64, 2, 64, 2)]
    pages = mx4.pack_pages(*parts)
    assert pages.shape == (0, mx4.page_bytes(32, 2, 64))
    assert [p.shape for p in mx4.unpack_pages(pages, 32, 2, 64)] == [p.shape for p in parts]


def test_rows_that_are_no_whole_blocks():
    for d in (0, 31, 48):
        with pytest.raises(ValueError, match="multiple of 32"):
            mx4.quantise(np.zeros((2, d), np.float32))


def test_the_registry_names_every_call_of_the_cache():
    calls = {n for n in vars(ops) if n.startswith(("attention_mx4", "mx4_kv_", "kv_pages_")) and not n.endswith("_workspace")}
    assert len(calls) == 9 and all(ops.OPS[n] is getattr(ops, n) for n in calls)
