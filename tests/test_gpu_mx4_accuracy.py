"""How near the attentions over the 4-bit cache come to the formula in 64 bits where
little but an output's rounding may be lost (tests/mx4_cases.py derives the bounds)."""
import numpy as np
import pytest

from doe_amd import DeviceBuffer, mx4, ops
from mx4_cases import Case, attention, check
from test_gpu_mx4_attention import prompt, tile, token, up  # noqa: F401  (a fixture among them)

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


@pytest.mark.parametrize("d", [64, 128, 160, 256, 512])
@pytest.mark.parametrize("f16", [False, True])
def test_prompt_dims_far_below_the_largest(dev, tile, d, f16):  # noqa: F811
    """Dims of 2^15 (f16: the largest of the type) among normal ones, keys zero there: the
    others make the scores and keep their bits.  f16 queries lose nothing, of f32 ones
    2^-38 of the largest may be lost beside the 2^-22 that the bound counts of each."""
    rng = np.random.default_rng(d)
    rows, lens, hq = [30, 20], [70, 40], 3
    case = Case(rng, lens, head_dim=d, num_kv_heads=1, page_size=32)
    wide = np.arange(0, d, 32) + 2 * rng.integers(0, 16, d // 32)
    case.kc[..., wide] = 0
    case.upload()
    q = rng.standard_normal((sum(rows), hq, d)).astype(np.float16 if f16 else np.float32)
    q[..., wide] = rng.choice([-65504.0, 65504.0] if f16 else [-32768.0, 32768.0], q[..., wide].shape)
    print(f"[far] d={d} f16={f16}", flush=True)
    starts, out = up(np.cumsum([0] + rows).astype(np.int32)), up(np.zeros(q.shape, np.float32))
    ws = DeviceBuffer(ops.attention_mx4_workspace(2, hq, 1, d, len(q)))
    ops.attention_mx4_prompt(case.cache, up(q), out, len(q), row_starts=starts, num_heads=hq, scale=d ** -0.5, q_f16=f16,
                             workspace=ws)
    # (the scores' sum by the dims that the keys have: the others add nothing to it)
    want, bound, mass = attention(case, q * (~np.isin(np.arange(d), wide)), rows, d ** -0.5)
    if not f16:
        keys = np.abs(np.where(case.ks[..., None] == mx4.NAN_SCALE, 0, mx4.dequantise(case.kc, np.minimum(case.ks, 140))
                               .reshape(*case.ks.shape, 32))).sum((-1, -2)).max()
        bound = bound + 2 * 2.0 ** -38 * 32768 * d ** -0.5 * keys * mass
    check(out.download(), want, bound, np.float32)


@pytest.mark.parametrize("d", [64, 160, 512])
@pytest.mark.parametrize("f16", [False, True])
def test_prompt_queries_that_are_no_numbers(dev, tile, d, f16):  # noqa: F811
    """A NaN or an infinity in any dim of a query makes its own output NaN, and no other."""
    rng = np.random.default_rng(d)
    case = Case(rng, [70], head_dim=d, num_kv_heads=1, page_size=32)
    case.upload()
    q = rng.standard_normal((40, 3, d)).astype(np.float16 if f16 else np.float32)
    bad = np.zeros((40, 3), bool)
    for row, head, dim, value in ((0, 0, 0, np.nan), (7, 2, d - 1, np.inf), (20, 1, d // 2 + 3, -np.inf), (39, 0, 37, -np.nan)):
        q[row, head, dim], bad[row, head] = value, True
    got = prompt(case, q, [40], f16=f16)
    assert np.array_equal(np.isnan(got), np.repeat(bad[..., None], d, -1))


@pytest.mark.parametrize("form", ["token", "prompt"])
@pytest.mark.parametrize("d", [64, 160, 512])
def test_queries_at_the_end_of_the_range(dev, form, d):
    """Finite f32 queries up to the type's largest, whatever the scale: scores that f32
    holds are right, also zero ones of a scale that overflows with the query's, and a
    cap holds those that overflow."""
    rng = np.random.default_rng(d)
    case = Case(rng, [300, 40], head_dim=d, num_kv_heads=1, page_size=32)
    case.kc[..., 5] = 0
    case.upload()
    call = token if form == "token" else (lambda c, q, **kw: prompt(c, q, [1, 1], **kw))
    normal = rng.standard_normal((2, 2, d)).astype(np.float32)
    largest = normal.copy()
    largest[..., 5] = np.finfo(np.float32).max
    for name, q, scale, softcap in (("1e36", normal * np.float32(1e36), 1e-37, 0.0), ("1e36", normal * np.float32(1e36), 1e-36, 5.0),
                                    ("1e37", normal * np.float32(3e37), 3e-39, 0.0), ("1e-40", normal * np.float32(1e-40), 1e38, 0.0),
                                    ("largest", largest * np.float32(1), 1e-30, 0.0)):
        print(f"[{form}] d={d} {name} scale={scale} softcap={softcap}", flush=True)
        got = call(case, q, scale=scale, softcap=softcap)
        check(got, *attention(case, q.astype(np.float32) * (name != "largest"), [1, 1], float(np.float32(scale)), softcap)[:2], got.dtype)
    # 2 ds + 2^-16 + 2^-18 of the mass, ds 2^-21 of the cap: no other part of the scores is left
    q = normal * np.float32(1e36)
    got = call(case, q, scale=1e5, softcap=30.0)
    want, _, mass = attention(case, q, [1, 1], 1e5, 30.0)
    check(got, want, (60 * 2.0 ** -21 + 2.0 ** -16 + 2.0 ** -18) * mass + 2.0 ** -32 * 300 * 6, got.dtype)
    case.kc[case.ks[..., None].repeat(32, -1).reshape(case.kc.shape) != mx4.NAN_SCALE] = 0
    case.pool.upload(case.pages())
    for softcap in (0.0, 30.0):
        got = call(case, q, scale=1e5, softcap=softcap)
        check(got, *attention(case, q, [1, 1], 1e5, softcap)[:2], got.dtype)


@pytest.mark.parametrize("d", [64, 160, 512])
@pytest.mark.parametrize("f16", [False, True])
def test_token_queries_that_are_no_numbers(dev, d, f16):
    """A NaN or an infinity in any dim of a query makes its own output NaN, and no other."""
    rng = np.random.default_rng(d)
    case = Case(rng, [70, 1, 900, 0], head_dim=d, num_kv_heads=1, page_size=32)
    case.upload()
    q = rng.standard_normal((4, 12, d)).astype(np.float16 if f16 else np.float32)
    bad = np.zeros((4, 12), bool)
    for row, head, dim, value in ((0, 0, 0, np.nan), (1, 2, d - 1, np.inf), (2, 11, d // 2 + 3, -np.inf), (2, 6, 37, -np.nan)):
        q[row, head, dim], bad[row, head] = value, True
    got = token(case, q, f16=f16)
    assert np.array_equal(np.isnan(got), np.repeat(bad[..., None], d, -1))


@pytest.mark.parametrize("longest", [50, 3000])
@pytest.mark.parametrize("form", ["token", "prompt"])
@pytest.mark.parametrize("d", [64, 160, 512])
@pytest.mark.parametrize("f16,size,factor", [(False, 1e30, 1e12), (False, 1e30, -1e12), (False, 1e36, 1e7), (False, 1e36, -1e7),
                                             (True, 1e3, 1e38), (True, 1e3, -1e38)])
def test_scores_that_overflow_are_no_numbers(dev, tile, form, d, f16, size, factor, longest):  # noqa: F811
    """Uncapped scores beyond f32, of one sign or the other, give NaN and no zeros."""
    rng = np.random.default_rng(d)
    case = Case(rng, [longest, 40, 33], head_dim=d, num_kv_heads=1, page_size=32)
    case.kc &= 7
    case.kc[..., 0] = 4
    case.upload()
    q = (np.abs(rng.standard_normal((3, 2, d))) * size).astype(np.float16 if f16 else np.float32)
    q[..., 0] = size
    got = token(case, q, f16=f16, scale=factor) if form == "token" else prompt(case, q, [1, 1, 1], f16=f16, scale=factor)
    assert np.isnan(got).all()
