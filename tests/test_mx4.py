"""The 4-bit cache's host side and the refusals of its calls (CPU only: every
refusal is made before the device is needed)."""
import ctypes as C
import shutil
import subprocess

import numpy as np
import pytest

from conftest import ROOT
from doe_amd import DoeError, mx4, ops


class FakeBuf:
    def __init__(self, nbytes, ptr=1 << 20):
        self.nbytes, self.ptr = nbytes, ptr


BIG = FakeBuf(1 << 62)


def test_quantise_picks_the_nearest_code():
    """Against a search over all codes in 64 bits, per block."""
    rng = np.random.default_rng(1)
    x = (rng.standard_normal((64, 64)) * np.exp(rng.uniform(-8, 8, (64, 1)))).astype(np.float32)
    codes, scales = mx4.quantise(x)
    assert scales.shape == (64, 2) and codes.max() <= 15
    step = np.ldexp(1.0, scales.astype(int) - 127)[..., None]
    y = x.reshape(64, 2, 32).astype(np.float64) / step
    top = np.abs(y).max(-1)
    assert np.all((top >= 3.5) & (top < 7))  # rounds to 4 or 6
    best = np.abs(np.abs(y)[..., None] - mx4.VALUES.astype(np.float64)).min(-1)
    got = mx4.dequantise(codes, scales).reshape(64, 2, 32) / step
    assert np.array_equal(np.abs(got - y), best)


def test_quantise_borders():
    ties = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], np.float32)
    x = np.zeros((1, 32), np.float32)
    x[0, 0] = 6
    x[0, 1:8], x[0, 8:15] = ties, -ties
    x[0, 15:22] = np.nextafter(ties, np.float32(10))
    x[0, 22:29] = np.nextafter(ties, np.float32(0))
    v = mx4.dequantise(*mx4.quantise(x))[0]
    even, up, down = [0, 1, 1, 2, 2, 4, 4], [0.5, 1, 1.5, 2, 3, 4, 6], [0, 0.5, 1, 1.5, 2, 3, 4]
    assert v[1:8].tolist() == even and v[8:15].tolist() == [-e for e in even]
    assert v[15:22].tolist() == up and v[22:29].tolist() == down
    for top, held in ((6.99, 6), (7, 8), (3.5, 4), (3.49, 3)):
        x = np.zeros((1, 32), np.float32)
        x[0, 3] = top
        assert mx4.dequantise(*mx4.quantise(x))[0, 3] == held


def test_quantise_extremes():
    x = np.zeros((6, 32), np.float32)
    x[1, 5], x[2, 5], x[3, 5], x[4, 5], x[5, 5] = 3e38, np.inf, np.nan, 1e-9, -57344.0
    codes, scales = mx4.quantise(x)
    v = mx4.dequantise(codes, scales)
    assert not v[0].any() and v[1, 5] == 49152 and v[4, 5] == 0 and v[5, 5] == -49152
    assert np.isnan(v[2]).all() and np.isnan(v[3]).all()
    assert np.array_equal(v[[0, 1, 4, 5]].astype(np.float16).astype(np.float32), v[[0, 1, 4, 5]])  # exact in f16


@pytest.mark.parametrize("ps,h,d", [(32, 1, 64), (64, 2, 128), (128, 1, 160), (32, 3, 256), (256, 1, 512)])
def test_pages_round_trip_and_layout(ps, h, d):
    rng = np.random.default_rng(d)
    kc, vc = (rng.integers(0, 16, (2, h, ps, d)).astype(np.uint8) for _ in "kv")
    ks, vs = (rng.integers(104, 141, (2, h, ps, d // 32)).astype(np.uint8) for _ in "kv")
    pages = mx4.pack_pages(kc, ks, vc, vs)
    assert pages.shape == (2, mx4.page_bytes(ps, h, d))
    for got, want in zip(mx4.unpack_pages(pages, ps, h, d), (kc, ks, vc, vs)):
        assert np.array_equal(got, want)
    # single values by the documented places
    slab = ps * (d + d // 16)
    for _ in range(50):
        n, a, x, i = rng.integers(2), rng.integers(h), rng.integers(ps), rng.integers(d)
        base = a * slab
        quarter, place = (x % 32 // 4) % 4, 4 * (x % 32 // 16) + x % 4
        k_at = base + x * d // 2 + i // 2
        column, within = i // (d // 16), i % (d // 16)
        v_at = base + ps * d // 2 + (((x // 32 * 4 + quarter) * 16 + column) * 8 + place) * (d // 32) + within // 2
        assert pages[n, k_at] >> 4 * (i & 1) & 15 == kc[n, a, x, i]
        assert pages[n, v_at] >> 4 * (i & 1) & 15 == vc[n, a, x, i]
        assert pages[n, base + ps * d + x * (d // 32) + i // 32] == ks[n, a, x, i // 32]
        at = base + ps * (d + d // 32) + ((x // 32 * 4 + quarter) * (d // 32) + i // 32) * 8 + place
        assert pages[n, at] == vs[n, a, x, i // 32]


def test_page_bytes_agrees_with_the_library():
    from doe_amd import _lib
    n = C.c_int64()
    _lib.call("doe_mx4_page_bytes", 64, 4, 256, C.byref(n))
    assert n.value == mx4.page_bytes(64, 4, 256) == 64 * 4 * 272
    for bad in ((48, 4, 256), (16, 4, 256), (512, 4, 256), (64, 4, 96), (64, 0, 256)):
        with pytest.raises(ValueError):
            mx4.page_bytes(*bad)
        with pytest.raises(DoeError):
            _lib.call("doe_mx4_page_bytes", *bad, C.byref(n))


@pytest.mark.parametrize("mirror,name", [(ops._Mx4CacheArgs, "doe_mx4_cache"), (ops._KvPagesArgs, "doe_kv_pages")])
def test_struct_layouts_match_the_header(tmp_path, mirror, name):
    if shutil.which("gcc") is None:
        pytest.skip("gcc not available")
    fields = [f[0] for f in mirror._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "doe_mi355x.h"\nint main(void) {\n'
                   + "".join(f'  printf("%zu\\n", offsetof({name}, {f}));\n' for f in fields)
                   + f'  printf("%zu\\n", sizeof({name}));\n  return 0;\n}}\n')
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [getattr(mirror, f).offset for f in fields] + [C.sizeof(mirror)]


def cache(pool=BIG, **change):
    kw = dict(num_pages=10, page_size=64, num_kv_heads=2, head_dim=128, batch=3, table_stride=4) | change
    return ops.Mx4Cache(pool, BIG, BIG, **kw)


def test_cache_checks_its_buffers():
    with pytest.raises(ValueError, match="pool"):
        cache(FakeBuf(10 * 64 * 2 * 136 - 1))
    with pytest.raises(ValueError, match="page_table"):
        ops.Mx4Cache(BIG, FakeBuf(47), BIG, num_pages=10, page_size=64, num_kv_heads=2, head_dim=128, batch=3,
                     table_stride=4)
    with pytest.raises(ValueError, match="kv_lens"):
        ops.Mx4Cache(BIG, BIG, FakeBuf(11), num_pages=10, page_size=64, num_kv_heads=2, head_dim=128, batch=3,
                     table_stride=4)
    for bad in (dict(head_dim=80), dict(page_size=48), dict(num_kv_heads=0)):
        with pytest.raises(ValueError):
            cache(**bad)


def refused(match, call, *args, **kw):
    with pytest.raises(DoeError, match=match) as e:
        call(*args, **kw)
    assert e.value.status in (-1, -4)


def test_cache_calls_refuse_bad_arguments():
    c = cache()
    for call in (ops.mx4_kv_write, ops.mx4_kv_read):
        with pytest.raises(ValueError, match="row_starts"):
            call(c, BIG, BIG, 5)
        with pytest.raises(ValueError, match="row_starts"):
            call(c, BIG, BIG, 5, row_starts=FakeBuf(15))
        with pytest.raises(ValueError, match="k has"):
            call(c, FakeBuf(3 * 256 * 4 - 1), BIG, 3)
        refused("row stride", call, c, BIG, BIG, 3, row_stride=255)
        refused("row stride", call, c, BIG, BIG, 3, row_stride=258)
        refused("aligned", call, c, FakeBuf(1 << 30, 8), BIG, 3)
        refused("null", call, c, BIG, FakeBuf(1 << 30, 0), 3)
        refused("rows", call, c, BIG, BIG, -1, row_starts=BIG)
        refused("2147483647 rows", call, c, BIG, BIG, (1 << 31) - 1, row_starts=BIG)
    refused("row stride", ops.mx4_kv_write, c, BIG, BIG, 3, row_stride=260, in_f16=True)
    refused("pool", ops.mx4_kv_write, cache(FakeBuf(1 << 40, 24)), BIG, BIG, 3)
    for bad, match in ((dict(num_pages=0), "num_pages"), (dict(batch=70000), "batch"), (dict(table_stride=0), "table_stride"),
                       (dict(table_stride=1 << 24), "positions"), (dict(num_kv_heads=2000), "num_kv_heads"),
                       (dict(num_pages=1 << 30), "num_pages")):
        c2 = cache(**bad)
        refused(match, ops.mx4_kv_write, c2, BIG, BIG, c2.batch)


def test_attention_calls_refuse_bad_arguments():
    c = cache()
    token = dict(num_heads=8, scale=0.1, workspace=BIG)
    with pytest.raises(ValueError, match="q has"):
        ops.attention_mx4(c, FakeBuf(3 * 8 * 128 * 4 - 1), BIG, **token)
    with pytest.raises(ValueError, match="output"):
        ops.attention_mx4(c, BIG, FakeBuf(3 * 8 * 128 * 2 - 1), out_f16=True, **token)
    for bad, match in ((dict(num_heads=7), "multiple"), (dict(num_heads=0), "multiple"), (dict(sliding_window=-1), "window"),
                       (dict(sliding_window=1 << 40), "window"), (dict(softcap=-1.0), "softcap"),
                       (dict(softcap=float("nan")), "softcap"), (dict(scale=float("inf")), "scale"),
                       (dict(scale=1e30, softcap=1e-10), "softcap"),
                       (dict(workspace=FakeBuf(8)), "workspace"), (dict(workspace=FakeBuf(1 << 40, 4)), "workspace")):
        refused(match, ops.attention_mx4, c, BIG, BIG, **{**token, **bad})
        refused(match, ops.attention_mx4_prompt, c, BIG, BIG, 500, row_starts=BIG, **{**token, **bad})
    refused("aligned", ops.attention_mx4, c, FakeBuf(1 << 40, 8), BIG, **token)
    refused("null", ops.attention_mx4, c, BIG, FakeBuf(1 << 40, 0), **token)
    with pytest.raises(ValueError, match="row_starts"):
        ops.attention_mx4_prompt(c, BIG, BIG, 5, **token)
    refused("strides", ops.attention_mx4_prompt, c, BIG, BIG, 5, row_starts=BIG, q_row_stride=1023, **token)
    refused("strides", ops.attention_mx4_prompt, c, BIG, BIG, 5, row_starts=BIG, out_row_stride=1026, **token)
    refused("rows", ops.attention_mx4_prompt, c, BIG, BIG, 1 << 40, row_starts=BIG, **token)
    many = cache(batch=65535, num_kv_heads=512)
    refused("KV heads", ops.attention_mx4, many, BIG, BIG, **{**token, "num_heads": 512})
    refused("in one call", ops.attention_mx4_prompt, many, BIG, BIG, 65535, **{**token, "num_heads": 512})
    for f in (lambda: ops.attention_mx4_workspace(3, 7, 2, 128), lambda: ops.attention_mx4_workspace(3, 8, 2, 96),
              lambda: ops.attention_mx4_workspace(-1, 8, 2, 128), lambda: ops.attention_mx4_workspace(3, 8, 2, 128, -1)):
        with pytest.raises(DoeError):
            f()


def test_tile_setting():
    try:
        for v in (32, 128, 0):
            ops.tune("attn_mx4.tile", v)
        for v in (-1, 1, 64, 256):
            refused("attn_mx4.tile", ops.tune, "attn_mx4.tile", v)
    finally:
        ops.tune("attn_mx4.tile", 0)


def test_prompt_workspace_grows_with_the_splits_only():
    # (row, head) pairs times splits; many rows need none
    assert ops.attention_mx4_workspace(1, 8, 2, 128, 1 << 20) == 16
    one = ops.attention_mx4_workspace(1, 8, 2, 128, 17)
    assert one > 16 and one % (17 * 8 * 130 * 4) == 0
    assert ops.attention_mx4_workspace(1, 8, 2, 128, 0) >= 0


def pages(**change):
    kw = dict(max_seqs=6, table_stride=4, num_pages=10, page_size=64, pools=BIG, layers=2, page_bytes=4096) | change
    return ops.KvPages(BIG, BIG, BIG, **kw)


def test_page_calls_refuse_bad_arguments():
    with pytest.raises(ValueError, match="pools"):
        pages(pools=None)
    with pytest.raises(ValueError, match="pools"):
        pages(pools=FakeBuf(2 * 10 * 4096 - 1))
    with pytest.raises(ValueError, match="page_refs"):
        ops.KvPages(BIG, BIG, FakeBuf(39), max_seqs=6, table_stride=4, num_pages=10, page_size=64)
    how = dict(status=BIG, workspace=BIG)
    p = pages()
    for call in (ops.kv_pages_extend, ops.kv_pages_fork):
        with pytest.raises(ValueError):
            call(p, FakeBuf(15), BIG, 4, **how)
        refused("workspace", call, p, BIG, BIG, 4, status=BIG, workspace=FakeBuf(100))
        refused("workspace", call, p, BIG, BIG, 4, status=BIG, workspace=FakeBuf(1 << 30, 8))
        refused("n -1", call, p, BIG, BIG, -1, **how)
        refused("n 16777216", call, p, BIG, BIG, 1 << 24, **how)
        refused("null", call, p, BIG, BIG, 4, status=FakeBuf(4, 0), workspace=BIG)
        refused("null list", call, p, FakeBuf(16, 0), BIG, 4, **how)
        refused("null list", call, p, BIG, FakeBuf(16, 0), 4, **how)
    refused("null list", ops.kv_pages_free, p, FakeBuf(16, 0), 4, status=BIG)
    for bad, match in ((dict(page_bytes=4100), "multiples of 16"), (dict(page_bytes=1 << 32), "page_bytes"), (dict(layer_stride=4096), "layer_stride"),
                       (dict(pools=FakeBuf(1 << 40, 8)), "multiples of 16")):
        refused(match, ops.kv_pages_compact, pages(**bad), **how)
        refused(match, ops.kv_pages_fork, pages(**bad), BIG, BIG, 4, **how)
    for bad, match in ((dict(max_seqs=0), "max_seqs"), (dict(num_pages=0), "num_pages"), (dict(page_size=0), "page_size"),
                       (dict(table_stride=1 << 25), "positions")):
        refused(match, ops.kv_pages_compact, pages(layers=0, **bad), **how)
    copy = dict(layers=2, num_pages=10, page_bytes=4096, status=BIG, workspace=BIG)
    with pytest.raises(ValueError, match="pools"):
        ops.kv_pages_copy(FakeBuf(100), BIG, BIG, 4, **copy)
    refused("multiples of 16", ops.kv_pages_copy, BIG, BIG, BIG, 4, **{**copy, "page_bytes": 4104})
    refused("workspace", ops.kv_pages_copy, BIG, BIG, BIG, 4, **{**copy, "workspace": FakeBuf(16)})
    refused("null list", ops.kv_pages_copy, BIG, FakeBuf(16, 0), BIG, 4, **copy)
    refused("entries of up to", ops.kv_pages_extend, pages(layers=0, max_seqs=1 << 23, table_stride=1 << 10), BIG, BIG,
            1 << 22, **how)
