"""Host side of the paged KV cache held in 4 bits: quantisation, pages (numpy).

A value is an E2M1 code times ``2 ** (scale - 127)``, one scale byte for 32
dims of a K or V row; the page layout is the one ``include/doe_mi355x.h``
documents and ``doe_mx4_kv_write`` fills.  These functions make caches on the
host and read them back without the GPU.
"""
from __future__ import annotations

import numpy as np

BLOCK = 32
HEAD_DIMS = (64, 128, 160, 256, 512)
PAGE_SIZES = (32, 64, 128, 256)
VALUES = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], np.float32)
NAN_SCALE = 255
MIN_EXP, MAX_EXP = -23, 13


def page_bytes(page_size: int, num_kv_heads: int, head_dim: int) -> int:
    """Bytes of one layer's page."""
    if head_dim not in HEAD_DIMS:
        raise ValueError(f"head_dim {head_dim} is none of {HEAD_DIMS}")
    if page_size not in PAGE_SIZES:
        raise ValueError(f"page_size {page_size} is none of {PAGE_SIZES}")
    if num_kv_heads <= 0:
        raise ValueError(f"num_kv_heads {num_kv_heads}")
    return page_size * num_kv_heads * (head_dim + head_dim // 16)


def quantise(rows: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """Codes ``[..., D]`` and scale bytes ``[..., D / 32]`` (uint8) of f32 rows."""
    x = np.asarray(rows, np.float32)
    if x.ndim == 0 or x.shape[-1] == 0 or x.shape[-1] % BLOCK:
        raise ValueError(f"rows of shape {x.shape}: the last axis has to be a multiple of {BLOCK}")
    b = x.reshape(*x.shape[:-1], x.shape[-1] // BLOCK, BLOCK)
    top = np.abs(b).max(-1)  # (a NaN is its block's maximum)
    finite = np.isfinite(top)
    bits = np.where(finite, top, 1).astype(np.float32).view(np.uint32)
    e = np.clip(((bits + 0x200000) >> 23).astype(np.int32) - 129, MIN_EXP, MAX_EXP)
    y = np.abs(np.where(finite[..., None], b, 0)) * np.ldexp(np.float32(1), -e)[..., None]
    code = np.zeros(b.shape, np.uint8)
    for at, even in ((0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        code += (y >= at) if even else (y > at)
    code |= np.signbit(b).astype(np.uint8) << 3
    code[~finite] = 0
    scale = np.where(finite, e + 127, NAN_SCALE).astype(np.uint8)
    return code.reshape(x.shape), scale


def dequantise(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    """f32 values ``[..., D]`` of codes and scale bytes."""
    codes = np.asarray(codes)
    v = VALUES[codes & 7] * np.where(codes & 8, np.float32(-1), np.float32(1))
    e = np.asarray(scales).astype(np.int32)
    s = np.where(e == NAN_SCALE, np.float32(np.nan), np.ldexp(np.float32(1), np.where(e == NAN_SCALE, 127, e) - 127))
    return (v.reshape(*s.shape, BLOCK) * s[..., None]).reshape(codes.shape).astype(np.float32)


def _widths(page_size: int, head_dim: int) -> list[int]:
    """Bytes of a slab's K codes, V codes, K scales and V scales."""
    return [page_size * head_dim // 2] * 2 + [page_size * head_dim // BLOCK] * 2


def pack_pages(k_codes, k_scales, v_codes, v_scales) -> np.ndarray:
    """Pages ``[n][page_bytes]`` of codes ``[n][num_kv_heads][page_size][D]``
    and scale bytes ``[n][num_kv_heads][page_size][D / 32]``."""
    n, h, ps, d = k_codes.shape
    size = page_bytes(ps, h, d)

    def two(x):
        return x[..., 0::2] | (x[..., 1::2] << 4)

    vc = v_codes.reshape(n, h, ps // 32, 2, 4, 4, 16, d // 16).transpose(0, 1, 2, 4, 6, 3, 5, 7)
    vs = v_scales.reshape(n, h, ps // 32, 2, 4, 4, d // 32).transpose(0, 1, 2, 4, 6, 3, 5)
    parts = [two(k_codes), two(vc), k_scales, vs]
    slabs = np.concatenate([p.reshape(n, h, w) for p, w in zip(parts, _widths(ps, d))], -1)
    return slabs.reshape(n, size).astype(np.uint8)


def unpack_pages(pages: np.ndarray, page_size: int, num_kv_heads: int, head_dim: int):
    """(k_codes, k_scales, v_codes, v_scales) of pages, as ``pack_pages`` takes them."""
    ps, h, d = page_size, num_kv_heads, head_dim
    if pages.shape[-1] != page_bytes(ps, h, d):
        raise ValueError(f"pages of {pages.shape[-1]} bytes, expected {page_bytes(ps, h, d)}")
    n = pages.shape[0]
    widths = _widths(ps, d)
    kc, vc, ks, vs = np.split(pages.reshape(n, h, sum(widths)), np.cumsum(widths)[:3], axis=-1)

    def two(b):
        return np.stack([b & 15, b >> 4], -1)

    vc = two(vc).reshape(n, h, ps // 32, 4, 16, 2, 4, d // 16).transpose(0, 1, 2, 5, 3, 6, 4, 7)
    vs = vs.reshape(n, h, ps // 32, 4, d // 32, 2, 4).transpose(0, 1, 2, 5, 3, 6, 4)
    return (two(kc).reshape(n, h, ps, d), ks.reshape(n, h, ps, d // 32),
            vc.reshape(n, h, ps, d), vs.reshape(n, h, ps, d // 32))
