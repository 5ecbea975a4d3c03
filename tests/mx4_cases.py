"""Caches of 4-bit pages for tests, and attention over them in 64 bits.

The pages are made on the host (doe_amd.mx4), the reference works on the values
they stand for.  ``bound`` is how far a result may be, element by element:
probabilities carry a relative error of at most 2 ds (numerator and sum), ds
the error of a score, and every output rounding half a step.  ds: the query's
f16 hi + lo parts leave 2^-22 of it (prompts: `attention`'s `digits`), the D products of a score are summed in
f32 in at most D / 16 + 8 steps of 2^-24 each and scaled once, softcap's tanh
is good to 2^-21 of the cap; the exponential, its argument (up to 150, in
steps of 2^-24 of itself) and the sums over positions add 2^-16 and 2^-18.  A
probability is held in f16 parts, where f16 has no steps below 2^-24: at most
2^-25 is lost of each, the largest being 2^7 or more (it lies 2^7 above the
running reference when that is raised, and the reference is only raised), so
2^-32 of |v| summed over the positions whatever they weigh."""
from __future__ import annotations

import numpy as np

from doe_amd import DeviceBuffer, mx4, ops


class Case:
    """Sequences of `lens` positions with scattered pages in a pool whose unused
    bytes are 0xff (NaN scales)."""

    def __init__(self, rng, lens, *, head_dim, num_kv_heads, page_size=32, stride=None, spare=3, k_scale=1.0, v_scale=1.0):
        self.lens, self.d, self.h, self.ps = [int(n) for n in lens], head_dim, num_kv_heads, page_size
        self.batch = len(self.lens)
        held = [-(-n // page_size) for n in self.lens]
        self.stride = stride or max(1, max(held, default=1))
        self.num_pages = sum(held) + spare
        ids = rng.permutation(self.num_pages)
        self.table = np.full((self.batch, self.stride), -1, np.int32)
        at = 0
        for b, n in enumerate(held):
            self.table[b, :n] = ids[at:at + n]
            at += n
        shape = (self.num_pages, num_kv_heads, page_size, head_dim)
        self.kc, self.ks = mx4.quantise(rng.standard_normal(shape).astype(np.float32) * np.float32(k_scale))
        self.vc, self.vs = mx4.quantise(rng.standard_normal(shape).astype(np.float32) * np.float32(v_scale))
        # positions that no sequence has in use
        used = np.zeros((self.num_pages, page_size), bool)
        for b, n in enumerate(self.lens):
            for i in range(held[b]):
                used[self.table[b, i], :min(page_size, n - i * page_size)] = True
        for code, scale in ((self.kc, self.ks), (self.vc, self.vs)):
            code.transpose(0, 2, 1, 3)[~used] = 15
            scale.transpose(0, 2, 1, 3)[~used] = mx4.NAN_SCALE

    def pages(self):
        return mx4.pack_pages(self.kc, self.ks, self.vc, self.vs)

    def upload(self):
        self.pool = DeviceBuffer.from_array(self.pages())
        self.table_dev = DeviceBuffer.from_array(self.table)
        self.lens_dev = DeviceBuffer.from_array(np.array(self.lens, np.int32))
        self.cache = ops.Mx4Cache(self.pool, self.table_dev, self.lens_dev, num_pages=self.num_pages, page_size=self.ps,
                                  num_kv_heads=self.h, head_dim=self.d, batch=self.batch, table_stride=self.stride)
        return self.cache

    def values(self, b, n):
        """K and V [n][h][D] in 64 bits of sequence b, and which positions have a page."""
        k, v = np.zeros((n, self.h, self.d)), np.zeros((n, self.h, self.d))
        has = np.zeros(n, bool)
        for p in range(0, n, self.ps):
            page, e = self.table[b, p // self.ps], min(self.ps, n - p)
            if 0 <= page < self.num_pages:
                for out, code, scale in ((k, self.kc, self.ks), (v, self.vc, self.vs)):
                    out[p:p + e] = mx4.dequantise(code[page], scale[page]).transpose(1, 0, 2)[:e]
                has[p:p + e] = True
        return k, v, has


def attention(case, q, rows, scale, softcap=0.0, window=0, digits=None):
    """(out, bound, mass) [total rows][heads][D] in 64 bits: q the rows of
    sequence 0, 1, ..., rows[b] of them each, at its last positions; mass is
    sum p |v|.  `digits` (prompts whose dims differ widely): what the queries'
    digits leave of the largest of each 32 dims, 2^-24 or 2^-19 of it."""
    q = np.asarray(q, np.float64)
    hq, g = q.shape[1], q.shape[1] // case.h
    out, bound, mass = np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape)
    at = 0
    for b, n in enumerate(rows):
        room = case.stride * case.ps
        length = max(0, min(case.lens[b], room))
        k, v, has = case.values(b, length)
        for i in range(n):
            pos = length - n + i
            key = np.arange(length)
            see = has & (key <= pos)
            if window:
                see &= key > pos - window
            if pos < 0 or not see.any():
                continue
            for head in range(hq):
                kk, vv = k[see, head // g], v[see, head // g]
                s = kk @ q[at + i, head] * scale
                big = np.max(np.abs(kk) @ np.abs(q[at + i, head])) * abs(scale)
                ds = big * (2.0 ** -22 + (case.d / 16 + 9) * 2.0 ** -24)
                if digits:
                    top = np.abs(q[at + i, head]).reshape(-1, 32).max(1)
                    ds += digits * abs(scale) * np.max(np.abs(kk).reshape(len(kk), -1, 32).sum(2) @ top)
                if softcap:
                    s = np.tanh(s / softcap) * softcap
                    ds += softcap * 2.0 ** -21
                p = np.exp(s - s.max())
                p /= p.sum()
                out[at + i, head], mass[at + i, head] = p @ vv, p @ np.abs(vv)
                bound[at + i, head] = (2 * ds + 2.0 ** -16 + 2.0 ** -18) * mass[at + i, head] + 2.0 ** -32 * np.abs(vv).sum(0)
        at += n
    return out, bound, mass


def check(got, want, bound, dtype, mass=None):
    """Every element within the bound and the output's rounding; with `mass`
    probabilities may be held in f16 (half a step each, 2^-11, and as much
    for what f16 loses of small ones)."""
    got = np.asarray(got, np.float64)
    tol = bound + float(np.finfo(dtype).eps) / 2 * np.abs(want) + (2.0 ** -25 if dtype == np.float16 else 0)
    if mass is not None:
        tol = tol + 2.0 ** -10 * mass
    rel = np.linalg.norm(got - want) / max(np.linalg.norm(want), 1e-300)
    worst = np.max(np.abs(got - want) / np.maximum(tol, 1e-300), initial=0.0)
    print(f"  rel {rel:.2e} of 64 bits, at most {worst:.2f} of the bound", flush=True)
    assert np.all(np.abs(got - want) <= tol), (rel, worst)
