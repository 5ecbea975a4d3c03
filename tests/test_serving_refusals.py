"""Calls of the adapters, the rotating append and beam search that are refused
on the host (CPU only)."""
import ctypes as C

import numpy as np
import pytest

from doe_amd import DoeError, ops
from test_mx4 import BIG, refused


def f16_cache(**kw):
    how = dict(num_pages=4, page_size=16, num_kv_heads=2, head_dim=64, batch=3, table_stride=2)
    return ops.F16Cache(BIG, BIG, BIG, BIG, **{**how, **kw})


def append(c=None, **kw):
    how = dict(num_heads=4, freq_cis=BIG, max_positions=100, row_starts=BIG)
    rows = kw.pop("rows", 5)
    ops.qkv_rope_append(c or f16_cache(), kw.pop("qkv", BIG), kw.pop("q_out", Apart()), rows, **{**how, **kw})


class Apart:
    """As `BIG`, somewhere else."""
    nbytes = 1 << 40
    ptr = 1 << 50


class Odd:
    nbytes = 1 << 40
    ptr = BIG.ptr + 8


@pytest.mark.parametrize("message,how", [
    ("rotary_dim 60", dict(rotary_dim=60)),
    ("rotary_dim 72", dict(rotary_dim=72)),
    ("row stride 510", dict(row_stride=510)),
    ("row stride 514", dict(row_stride=514)),
    ("q row stride 252", dict(q_row_stride=252)),
    ("q row stride 260", dict(q_row_stride=260, q_f16=True)),
    ("16-byte aligned", dict(qkv=Odd())),
    ("apart from qkv", dict(q_out=BIG, q_row_stride=256)),
    ("apart from qkv", dict(q_out=BIG, q_row_stride=512, q_f16=True)),
    ("max_positions -1", dict(max_positions=-1)),
    ("num_heads -1", dict(num_heads=-1)),
])
def test_append(message, how):
    refused(message, append, **how)
    refused(message, append, ops.Mx4Cache(BIG, BIG, BIG, num_pages=4, page_size=32, num_kv_heads=2, head_dim=64, batch=3,
                                          table_stride=2), **how)


@pytest.mark.parametrize("message,how", [
    ("head_dim 60", dict(head_dim=60)), ("head_dim 2048", dict(head_dim=2048)), ("num_kv_heads 0", dict(num_kv_heads=0)),
    ("num_pages 0", dict(num_pages=0)), ("page_size 0", dict(page_size=0)), ("fewer than 2\\^30", dict(table_stride=1 << 27)),
    ("batch 70000", dict(batch=70000)),
])
def test_f16_cache(message, how):
    c = f16_cache(**how)
    refused(message, append, c, row_stride=8192, q_row_stride=4096, rotary_dim=0, rows=1)


def test_append_buffers_are_checked():
    class Small:
        nbytes, ptr = 64, 16
    for role, how in (("qkv", dict(qkv=Small())), ("q_out", dict(q_out=Small())), ("freq_cis", dict(freq_cis=Small())),
                      ("row_starts", dict(row_starts=type("S", (), dict(nbytes=4, ptr=16))()))):
        with pytest.raises(ValueError, match=role):
            append(**how)
    with pytest.raises(ValueError, match="5 rows without row_starts"):
        append(row_starts=None)
    with pytest.raises(ValueError, match="no q_out"):
        append(q_out=None)
    with pytest.raises(ValueError, match="no freq_cis"):
        append(freq_cis=None)


def lora(**kw):
    how = dict(num_adapters=3, rank=16, k=64, slice_n=[40, 24])
    return ops.Lora(BIG, kw.pop("b", BIG), None, **{**how, **kw})


@pytest.mark.parametrize("message,l,how", [
    ("rank 12", dict(rank=12), {}), ("rank 264", dict(rank=264), {}), ("k 60", dict(k=60), {}),
    ("slice_n\\[1\\] 0", dict(slice_n=[8, 0]), {}), ("num_adapters 0", dict(num_adapters=0), {}),
    ("16-byte aligned", dict(b=Odd()), {}),
    ("x_row_stride 60", {}, dict(x_row_stride=60)), ("x_row_stride 66", {}, dict(x_row_stride=66)),
    ("y_row_stride 63", {}, dict(y_row_stride=63)), ("y_row_stride 67108864", {}, dict(y_row_stride=1 << 26)),
    ("x_row_stride 16777216", {}, dict(x_row_stride=1 << 24)),
    ("4 segments, 5 rows", {}, dict(segments=4)),
    ("workspace of", {}, dict(workspace=type("S", (), dict(nbytes=16, ptr=16))())),
    ("x must be 16-byte", {}, dict(x=Odd())),
    ("apart", {}, dict(y=BIG)),
])
def test_lora(message, l, how):
    x, y = how.pop("x", BIG), how.pop("y", Apart())
    refused(message, ops.lora_add, lora(**l), BIG, x, y, 5, **{**dict(workspace=BIG), **how})


def test_lora_buffers_are_checked():
    for n in (0, 5):
        with pytest.raises(ValueError, match=f"{n} slices"):
            lora(slice_n=[8] * n)
    with pytest.raises(ValueError, match="count of segments"):
        ops.lora_add(lora(), BIG, BIG, Apart(), 5, workspace=BIG, row_starts=BIG)


def at(ptr, nbytes=1 << 40):
    return type("B", (), dict(nbytes=nbytes, ptr=ptr))()


def select(**kw):
    how = dict(batch=2, beams=4, vocab=1000, select=8, parents=Apart(), tokens=Apart(), out_scores=Apart(), workspace=BIG)
    ops.beam_select(kw.pop("logits", BIG), kw.pop("scores", BIG), **{**how, **kw})


@pytest.mark.parametrize("how", [
    dict(out_scores=BIG), dict(out_scores=at(BIG.ptr + 28)), dict(out_scores=at(BIG.ptr - 60)), dict(out_scores=BIG, select=5), dict(parents=BIG),
    dict(tokens=at(BIG.ptr + 4)), dict(out_scores=at(BIG.ptr + 4), select=4), dict(finished=at(1 << 45), out_finished=at(1 << 45), end_token=1),
    dict(finished=at(1 << 45), out_finished=at((1 << 45) + 4), end_token=1, select=4), dict(finished=at(1 << 45), out_scores=at((1 << 45) - 8), end_token=1),
])
def test_select_in_place(how):
    refused("overlap scores or finished", select, **how)


@pytest.mark.parametrize("message,how", [
    ("beams 65", dict(beams=65)), ("beams 0", dict(beams=0)), ("select 0", dict(select=0)), ("select 65", dict(select=65)),
    ("vocab 0", dict(vocab=0)), ("vocab 16777217", dict(vocab=(1 << 24) + 1)), ("row stride 999", dict(row_stride=999)),
    ("inv_temperature 0", dict(inv_temperature=0.0)), ("inv_temperature 1e-20", dict(inv_temperature=1e-20)),
    ("inv_temperature -1", dict(inv_temperature=-1.0)), ("inv_temperature nan", dict(inv_temperature=float("nan"))),
    ("inv_temperature inf", dict(inv_temperature=float("inf"))), ("inv_temperature 3e\\+38", dict(inv_temperature=3e38)),
    ("end_token 1000", dict(end_token=1000)), ("end_token -1", dict(finished=BIG)),
    ("workspace of", dict(workspace=type("S", (), dict(nbytes=16, ptr=16))())),
    ("4-byte aligned", dict(logits=type("S", (), dict(nbytes=1 << 40, ptr=18))())),
])
def test_select(message, how):
    refused(message, select, **how)


def reorder(**kw):
    how = dict(row_bytes=64, layers=2)
    ops.beam_reorder_rows(kw.pop("src", BIG), kw.pop("dst", Apart()), BIG, kw.pop("rows", 6), **{**how, **kw})


@pytest.mark.parametrize("message,how", [
    ("row_bytes 62", dict(row_bytes=62)), ("row_bytes 0", dict(row_bytes=0)), ("layer strides", dict(src_layer_stride=380)),
    ("layer strides", dict(dst_layer_stride=380)), ("layer strides", dict(dst_layer_stride=386)), ("overlap", dict(dst=BIG)),
    ("4-byte aligned", dict(dst=type("S", (), dict(nbytes=1 << 40, ptr=(1 << 50) + 2))())),
])
def test_reorder_rows(message, how):
    refused(message, reorder, **how)


def test_reorder_pages():
    pages = ops.KvPages(BIG, BIG, BIG, max_seqs=8, table_stride=4, num_pages=16, page_size=32)
    refused("n 8193", ops.beam_reorder_pages, ops.KvPages(BIG, BIG, BIG, max_seqs=9000, table_stride=4, num_pages=16, page_size=32),
            BIG, 8193, status=BIG, workspace=BIG)
    refused("9 sequences of 8 slots", ops.beam_reorder_pages, pages, BIG, 9, status=BIG, workspace=BIG)
    refused("workspace of", ops.beam_reorder_pages, pages, BIG, 8, status=BIG,
            workspace=type("S", (), dict(nbytes=16, ptr=16))())
    assert ops.beam_reorder_pages_workspace(16, 8, 8) == 4 * (16 + 16 + 8 + 48)


def test_workspaces_and_registry():
    assert ops.lora_workspace(lora(), 0) == 16
    assert ops.beam_select_workspace(0, 4, 1000, 8) == 16
    for name in ("beam_reorder_pages", "beam_reorder_rows", "beam_select", "lora_add", "qkv_rope_append"):
        assert ops.OPS[name] is getattr(ops, name)
    with pytest.raises(DoeError, match="select 65"):
        ops.beam_select_workspace(1, 4, 1000, 65)


def test_argument_structs_match_the_header(tmp_path):
    import shutil
    import subprocess

    from conftest import ROOT
    if shutil.which("gcc") is None:
        pytest.skip("gcc not available")
    for cls, name in ((ops._F16CacheArgs, "doe_f16_cache"), (ops._LoraArgs, "doe_lora")):
        names = [f[0] for f in cls._fields_]
        src = tmp_path / f"{name}.c"
        src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "doe_mi355x.h"\nint main(void) {\n'
                       + "".join(f'  printf("%zu\\n", offsetof({name}, {n}));\n' for n in names)
                       + f'  printf("%zu\\n", sizeof({name}));\n  return 0;\n}}\n')
        exe = tmp_path / name
        subprocess.run(["gcc", "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
        got = [int(v) for v in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
        assert got == [getattr(cls, n).offset for n in names] + [C.sizeof(cls)]
    assert np.dtype(np.int32).itemsize == 4
