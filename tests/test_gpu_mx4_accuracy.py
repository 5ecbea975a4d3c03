"""How near the attentions over the 4-bit cache come to the formula in 64 bits where
little but an output's rounding may be lost (tests/mx4_cases.py derives the bounds)."""
import numpy as np
import pytest

from mx4_cases import Case, attention, check
from test_gpu_mx4_attention import prompt, tile  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d,hq,hkv", [(64, 6, 2), (128, 8, 2), (160, 3, 1), (256, 4, 2), (512, 3, 1)])
def test_f16_prompts_lose_their_rounding_only(dev, tile, d, hq, hkv):  # noqa: F811
    """f16 queries and outputs: probabilities keep more bits than the output.  Rows
    that see few positions, of values that nearly cancel, show each of their bits:
    half a step of one f16 is 2^-12 of the values' mass, the bound about 2^-15."""
    rng = np.random.default_rng(d)
    rows, lens = [40, 9, 70], [40, 12, 200]
    case = Case(rng, lens, head_dim=d, num_kv_heads=hkv, page_size=32)
    case.upload()
    q = rng.standard_normal((sum(rows), hq, d)).astype(np.float16)
    print(f"[f16] d={d} hq={hq} hkv={hkv}", flush=True)
    got = prompt(case, q, rows, f16=True)
    want, bound, _ = attention(case, q, rows, d ** -0.5, digits=2.0 ** -24)
    check(got, want, bound, got.dtype)
