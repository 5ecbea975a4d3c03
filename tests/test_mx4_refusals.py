"""Arguments of the 4-bit cache's calls at the ends of their ranges (CPU only)."""
import pytest

from doe_amd import ops
from test_mx4 import BIG, cache, refused


@pytest.mark.parametrize("bad", [dict(scale=3e38), dict(scale=-3e38), dict(scale=1.0, softcap=3e38)])
def test_factors_that_overflow_in_powers_of_two(bad):
    """scale log2(e) and softcap log2(e) are what the kernels multiply by."""
    c, how = cache(), dict(num_heads=8, scale=0.1, workspace=BIG)
    refused("above 2.35e38", ops.attention_mx4, c, BIG, BIG, **{**how, **bad})
    refused("above 2.35e38", ops.attention_mx4_prompt, c, BIG, BIG, 500, row_starts=BIG, **{**how, **bad})
