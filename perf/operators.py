"""Performance cases of the paged KV cache held in 4 bits.

Each case is one pass that a serving program makes: writing K / V rows into
the cache (and reading them back), attention of single tokens or of prompts
over it, and the handling of its pages.  ``run`` computes a pass in plain torch
where ``own`` is false and through ``doe_amd.ops`` where it is true.

The cache.  A pool of pages, ``page_size`` positions each.  A page holds one
slab for each KV head, of page_size * (D + D / 16) bytes:

  K codes   [page_size][D / 2]           two values a byte, the even dim low
  V codes   [page_size / 32][4][16][8][D / 32]
  K scales  [page_size][D / 32]
  V scales  [page_size / 32][4][D / 32][8]

Position x of 32 has its V at [(x / 4) % 4][.][4 (x / 16) + x % 4]; the 16
columns hold D / 16 dims each.  A value is a 4-bit float (sign, two exponent
bits, one mantissa bit) times 2^(scale - 127), one scale for 32 dims; 255 says
that the block is not a number.  ``page_table`` [sequences][stride] holds page
ids, ``kv_lens`` the positions in use.  Row i of the n rows that a call brings
for a sequence is at position kv_len - n + i.

Kinds
  write    K / V rows of a step or of prompts into the cache, and back
  token    attention of one query token a sequence
  prompt   causal attention of a prompt's rows, or a chunk of them
  extend   pages for the next tokens of some sequences, and freeing of others
  fork     sequences that go on as several (beams, samples of one prompt)
  compact  the pages in use moved to the front of the pool
  copy     pages copied to others, in every layer
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
I32, F32 = torch.int32, torch.float32


class Buf:
    """A torch tensor as an operator's argument (its address and its bytes)."""

    def __init__(self, t: torch.Tensor):
        self.t = t
        self.ptr = t.data_ptr()
        self.nbytes = t.numel() * t.element_size()


# ---- the cases -----------------------------------------------------------------

def listed() -> list[dict]:
    return [
        # one decode step's K / V row of the 2B-class decoder: the smallest call
        dict(name="write_token", kind="write", batch=1, hkv=4, d=256, n=1, past=700, f16=False, page=64),
        # eight prompts of up to 4000 tokens, ragged, into caches that hold something already
        dict(name="write_prompts", kind="write", batch=8, hkv=8, d=128, n=4000, past=500, f16=False, page=64),
        # one token against a 4096-token context, batch 1: the 2B-class decoder's head layout
        dict(name="token_4096", kind="token", batch=1, hq=8, hkv=4, d=256, kv=4096, f16=False, page=64, window=0,
             softcap=0.0),
        # eight sequences of up to 32768 tokens, f16 queries
        dict(name="token_32k_b8", kind="token", batch=8, hq=64, hkv=8, d=128, kv=32768, f16=True, page=64, window=0,
             softcap=0.0, even=True),
        # a serving batch of sequences of 1 to 12000 tokens
        dict(name="token_ragged_b48", kind="token", batch=48, hq=16, hkv=2, d=128, kv=12000, f16=False, page=32,
             window=0, softcap=0.0),
        # 31B-class heads of 160, a sliding window and capped scores
        dict(name="token_window_b5", kind="token", batch=5, hq=32, hkv=16, d=160, kv=9001, f16=True, page=128,
             window=1024, softcap=50.0),
        # a 1000-token prompt of the 2B-class decoder
        dict(name="prompt_1000", kind="prompt", batch=1, hq=8, hkv=4, d=256, n=1000, past=0, f16=False, page=64,
             window=0, softcap=0.0),
        # 2048 tokens of a long prompt behind 8192 that are in the cache already
        dict(name="prompt_chunk_2048", kind="prompt", batch=1, hq=32, hkv=8, d=128, n=2048, past=8192, f16=True,
             page=64, window=0, softcap=0.0),
        # a batch of ragged prompts, one KV head, sliding window, capped scores
        dict(name="prompt_ragged_b12", kind="prompt", batch=12, hq=8, hkv=1, d=64, n=777, past=1500, f16=False,
             page=32, window=512, softcap=30.0),
        # a serving step's page bookkeeping: 192 sequences grow, 40 end
        dict(name="extend_free_256", kind="extend", seqs=256, grow=192, end=40, kv=6000, add=100, pages=40000,
             page=64),
        # twelve prompts that go on as eight samples each; the last page of each is copied in every layer
        dict(name="fork_12x8", kind="fork", seqs=12, forks=8, kv=1900, layers=26, hkv=4, d=256, page=64),
        # half of a pool in use, scattered: its pages are moved to the front in every layer
        dict(name="compact_900", kind="compact", seqs=20, kv=1900, pages=900, layers=26, hkv=4, d=256, page=64),
    ]


def _log(rng, lo, hi) -> int:
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    kind = rng.choice(["write", "token", "token", "token", "prompt", "prompt", "extend", "fork", "compact", "copy"])
    page = rng.choice([32, 64, 128, 256])
    d, hkv = rng.choice([64, 128, 128, 160, 256, 512]), rng.choice([1, 2, 4, 8, 16])
    hq = hkv * rng.choice([1, 2, 3, 4, 6, 8, 12, 16])
    f16, window, softcap = rng.random() < 0.5, rng.choice([0, 0, 100, 1024]), rng.choice([0.0, 0.0, 30.0])
    if kind == "write":
        batch = _log(rng, 1, 64)
        n = rng.choice([1, _log(rng, 2, 8000)])
        return dict(kind=kind, batch=batch, hkv=hkv, d=d, n=max(1, min(n, 16_000_000 // (batch * hkv * d))),
                    past=rng.randint(0, 900), f16=f16, page=page)
    if kind == "token":
        batch = _log(rng, 1, 64)
        kv = _log(rng, 20, min(60000, 260_000_000 // (batch * hkv * d)))
        return dict(kind=kind, batch=batch, hq=hq, hkv=hkv, d=d, kv=kv, f16=f16, page=page, window=window,
                    softcap=softcap, even=rng.random() < 0.3)
    if kind == "prompt":
        batch, n = _log(rng, 1, 16), _log(rng, 3, 2000)
        hq, hkv = min(hq, 32), min(hkv, hq, 8)
        hq -= hq % hkv
        past = rng.choice([0, 0, _log(rng, 10, 9000)])
        while batch * n * (past + n) * hq * d > 2 ** 36:
            n, past = max(3, n * 3 // 4), past * 3 // 4
        return dict(kind=kind, batch=batch, hq=hq, hkv=hkv, d=d, n=n, past=past, f16=f16, page=page, window=window,
                    softcap=softcap)
    if kind == "extend":
        seqs = _log(rng, 4, 512)
        grow = rng.randint(1, seqs - 1)
        kv, add = _log(rng, 50, 8000), _log(rng, 1, 3000)
        return dict(kind=kind, seqs=seqs, grow=grow, end=rng.randint(1, seqs - grow), kv=kv, add=add,
                    pages=seqs * (kv // page + 2) + grow * (add // page + 2) + rng.randint(0, 5000), page=page)
    layers, d, hkv = rng.randint(1, 26), rng.choice([64, 128, 256]), rng.choice([1, 2, 4])
    page = rng.choice([32, 64])
    if kind == "fork":
        return dict(kind=kind, seqs=rng.randint(1, 12), forks=rng.randint(1, 8), kv=_log(rng, 20, 1900),
                    layers=layers, hkv=hkv, d=d, page=page)
    if kind == "copy":
        return dict(kind=kind, count=_log(rng, 1, 200), pages=900, layers=layers, hkv=hkv, d=d, page=page)
    seqs, kv = rng.randint(1, 20), _log(rng, 20, 1500 if page == 64 else 700)
    pages = seqs * -(-kv // page) + rng.randint(10, 400)
    return dict(kind=kind, seqs=seqs, kv=kv, pages=pages, layers=layers, hkv=hkv, d=d, page=page)


# ---- sizes ---------------------------------------------------------------------

def _spread(count: int, most: int, shift: float) -> list[int]:
    """`count` whole numbers over [min(1, most), most], the first of them `most`."""
    least = min(1, most)
    return [most if i == 0 else least + int((most - least) * math.modf(i * 0.6180339887 + shift)[0])
            for i in range(count)]


def _rows(c: dict) -> list[int]:
    """Rows that the call brings for each sequence."""
    if c["kind"] == "token" or c["n"] == 1:
        return [1] * c["batch"]
    return _spread(c["batch"], c["n"], 0.13)


def _lens(c: dict) -> list[int]:
    """Positions in use of each sequence, the call's own rows among them."""
    if c["kind"] == "token":
        return [c["kv"]] * c["batch"] if c.get("even") else _spread(c["batch"], c["kv"], 0.37)
    if c["kind"] in ("extend", "fork", "compact"):
        return _spread(c["seqs"], c["kv"], 0.37)
    return [n + p for n, p in zip(_rows(c), _spread(c["batch"], c["past"], 0.37))]


def _page_bytes(c: dict) -> int:
    return c["page"] * c["hkv"] * (c["d"] + c["d"] // 16)


def _moved(c: dict) -> tuple[int, int]:
    """(pages copied, table entries written) by a pass over the pages."""
    ps = c["page"]
    lens = _lens(c) if c["kind"] != "copy" else []
    if c["kind"] == "copy":
        return c["count"], 2 * c["count"]
    if c["kind"] == "fork":
        return sum(c["forks"] for n in lens if n % ps), c["forks"] * sum(-(-n // ps) for n in lens)
    live = sum(-(-n // ps) for n in lens)
    if c["kind"] == "compact":
        return int(live * (1 - live / c["pages"])), live
    return 0, c["grow"] * (c["add"] // ps + 1)


def work(case: dict) -> dict:
    c = case
    if c["kind"] in ("extend", "fork", "compact", "copy"):
        moved, entries = _moved(c)
        data = 2 * moved * c.get("layers", 0) * (_page_bytes(c) if "d" in c else 0)
        return {"bytes": data + 8 * entries + 4 * c.get("pages", entries), "flops": 0}
    rows, lens, d = _rows(c), _lens(c), c["d"]
    size = 2 if c["f16"] else 4
    cell = c["hkv"] * 2 * (d // 2 + d // 32)
    if c["kind"] == "write":
        values = sum(rows) * c["hkv"] * d * 2
        return {"bytes": values * (size + 4) + 2 * sum(rows) * cell, "flops": 4 * values}
    reach = [min(m, c["window"] + n - 1) if c["window"] else m for n, m in zip(rows, lens)]
    seen = sum(sum(min(m - n + i + 1, c["window"] or m) for i in range(n)) for n, m in zip(rows, lens))
    return {"bytes": sum(reach) * cell + 2 * sum(rows) * c["hq"] * d * size, "flops": 4 * seen * c["hq"] * d}


# ---- inputs ----------------------------------------------------------------------

def _gen(seed: int) -> torch.Generator:
    return torch.Generator(DEV).manual_seed(seed)


def _kv_values(g, shape) -> torch.Tensor:
    """Rows as a model's projections give them: normal, some channels wider."""
    wide = 1 + 4 * (torch.rand(shape[-1], generator=g, device=DEV) < 0.04)
    return torch.randn(shape, generator=g, device=DEV) * wide


def _tables(g, lens, page, pages, stride) -> torch.Tensor:
    """A page table whose sequences hold scattered pages of their own."""
    need = [-(-n // page) for n in lens]
    ids = torch.randperm(pages, generator=g, device=DEV).int()
    table = torch.full((len(lens), stride), -1, dtype=I32, device=DEV)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = ids[at:at + n]
        at += n
    return table


def _prepare_pages(c: dict, seed: int) -> dict:
    g, kind, ps = _gen(seed), c["kind"], c["page"]
    st = {"case": c, "status": torch.zeros(1, dtype=I32, device=DEV)}
    if kind == "copy":
        ids = torch.randperm(c["pages"], generator=g, device=DEV).int()
        st["src"], st["dst"] = ids[:c["count"]].contiguous(), ids[c["count"]:2 * c["count"]].contiguous()
        pages = c["pages"]
    else:
        lens = _lens(c)
        live = sum(-(-n // ps) for n in lens)
        slots = len(lens) * (1 + c.get("forks", 0))
        stride = -(-(c["kv"] + c.get("add", 0)) // ps) + 1
        pages = c.get("pages") or live + len(lens) * c["forks"] + 16
        # page_table, kv_lens and page_refs in one piece, so that a pass starts
        # from the same state with one copy
        meta = torch.zeros(slots * stride + slots + pages, dtype=I32, device=DEV)
        table, kv_lens = meta[:slots * stride].view(slots, stride), meta[slots * stride:slots * stride + slots]
        refs = meta[slots * stride + slots:]
        table.fill_(-1)
        table[:len(lens)] = _tables(g, lens, ps, pages, stride)
        kv_lens[:len(lens)] = torch.tensor(lens, dtype=I32, device=DEV)
        refs[table[table >= 0].long()] = 1
        st |= {"meta": meta, "saved": meta.clone(), "table": table, "kv_lens": kv_lens, "refs": refs}
        if kind == "fork":
            who = torch.arange(slots - len(lens), device=DEV, dtype=I32)
            st["src"], st["dst"] = who % len(lens), who + len(lens)
        if kind == "extend":
            who = torch.randperm(len(lens), generator=g, device=DEV).int()
            st["src"], st["dst"] = who[:c["grow"]].contiguous(), who[c["grow"]:c["grow"] + c["end"]].contiguous()
            st["add"] = torch.randint(1, c["add"] + 1, (c["grow"],), generator=g, device=DEV, dtype=I32)
    if "layers" in c:
        st["pool"] = torch.randint(0, 256, (c["layers"], pages, _page_bytes(c)), generator=g, device=DEV,
                                   dtype=torch.uint8)
    st["scratch"] = torch.zeros(1 << 22, dtype=I32, device=DEV)
    return st


def prepare(case: dict, seed: int) -> dict:
    c = case
    if c["kind"] in ("extend", "fork", "compact", "copy"):
        st = _prepare_pages(c, seed)
    else:
        g, ps, d = _gen(seed), c["page"], c["d"]
        rows, lens = _rows(c), _lens(c)
        stride = -(-max(lens) // ps)
        pages = sum(-(-n // ps) for n in lens) + 3
        starts = [sum(rows[:b]) for b in range(len(rows) + 1)]
        dtype = torch.float16 if c["f16"] else F32
        st = {"case": c, "table": _tables(g, lens, ps, pages, stride),
              "kv_lens": torch.tensor(lens, dtype=I32, device=DEV), "starts": torch.tensor(starts, dtype=I32, device=DEV),
              "scratch": torch.empty(1 << 28, dtype=torch.uint8, device=DEV)}
        if c["kind"] == "write":
            st["pool"] = torch.zeros((pages, _page_bytes(c)), dtype=torch.uint8, device=DEV)
            for name in ("k", "v"):
                st[name] = _kv_values(g, (starts[-1], c["hkv"], d)).to(dtype)
                st[name + "_back"] = torch.zeros((starts[-1], c["hkv"], d), device=DEV)
        else:
            parts = [_quantise(_kv_values(g, (pages, c["hkv"], ps, d))) for _ in "kv"]
            st["pool"] = _pack(c, *parts[0], *parts[1])
            st["q"] = torch.randn((starts[-1], c["hq"], d), generator=g, device=DEV).to(dtype)
            st["out"] = torch.zeros_like(st["q"])
    st["buf"] = {k: Buf(t) for k, t in st.items() if isinstance(t, torch.Tensor)}
    return st


# ---- the plain form ----------------------------------------------------------------

VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _quantise(x: torch.Tensor):
    """(codes, scale bytes) of f32 rows [..., D]: blocks of 32, a power of two
    so that the largest value, rounded to a power of two from 1.75 on, is at
    4, values to the nearest of VALUES, ties to the even code."""
    b = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    top = b.abs().amax(-1, keepdim=True)
    e = (((top.view(I32) + 0x200000) >> 23) - 129).clamp(-23, 13)
    y = (b * torch.ldexp(torch.ones_like(top), -e)).abs()
    code = (y > 0.25).to(torch.uint8)
    for at, even in ((0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        code += (y >= at) if even else (y > at)
    code += 8 * torch.signbit(b).to(torch.uint8)
    scale = torch.where(top < math.inf, e + 127, 255).to(torch.uint8)
    return code.reshape(x.shape), scale.squeeze(-1)


def _values(code: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """f32 values [..., D] of codes [..., D] and scale bytes [..., D / 32]."""
    table = torch.tensor(VALUES + tuple(-v for v in VALUES), device=code.device)
    s = torch.where(scale == 255, math.nan, torch.ldexp(torch.ones(1, device=code.device), scale.int() - 127))
    v = table[code.int()]
    return (v.view(*scale.shape, 32) * s.unsqueeze(-1)).view(code.shape)


def _pack(c: dict, kc, ks, vc, vs) -> torch.Tensor:
    """Pages [n][bytes] of codes [n][hkv][page_size][D] and their scales."""
    n, h, ps, d = kc.shape
    two = lambda x: x[..., 0::2] | (x[..., 1::2] << 4)  # noqa: E731
    vt = vc.view(n, h, ps // 32, 2, 4, 4, 16, d // 16).permute(0, 1, 2, 4, 6, 3, 5, 7)
    st = vs.view(n, h, ps // 32, 2, 4, 4, d // 32).permute(0, 1, 2, 4, 6, 3, 5)
    return torch.cat([p.reshape(n, h, -1) for p in (two(kc), two(vt.contiguous()), ks, st)], -1).view(n, -1)


def _unpack(c: dict, pages: torch.Tensor):
    """K and V values [n][hkv][page_size][D] of pages [n][bytes]."""
    n, h, ps, d = pages.shape[0], c["hkv"], c["page"], c["d"]
    x = pages.view(n, h, -1)
    kc, vc, ks, vs = x.split([ps * d // 2, ps * d // 2, ps * d // 32, ps * d // 32], -1)
    two = lambda b: torch.stack([b & 15, b >> 4], -1)  # noqa: E731
    vc = two(vc).view(n, h, ps // 32, 4, 16, 2, 4, d // 16).permute(0, 1, 2, 5, 3, 6, 4, 7)
    vs = vs.reshape(n, h, ps // 32, 4, d // 32, 2, 4).permute(0, 1, 2, 5, 3, 6, 4)
    return (_values(two(kc).view(n, h, ps, d), ks.reshape(n, h, ps, d // 32)),
            _values(vc.reshape(n, h, ps, d), vs.reshape(n, h, ps, d // 32)))


def _where(st: dict):
    """Sequence and position of each row of the call."""
    starts = st["starts"].long()
    row = torch.arange(int(st["rows"]), device=DEV)
    b = torch.searchsorted(starts[1:], row, right=True)
    return b, row - starts[1:][b] + st["kv_lens"].long()[b]


def _plain_write(st: dict):
    c = st["case"]
    h, ps, d, pool = c["hkv"], c["page"], c["d"], st["pool"].view(-1)
    b, pos = _where(st)
    slab = _page_bytes(c) // h
    x = (pos % ps).view(-1, 1, 1)
    base = (st["table"].long()[b, pos // ps].view(-1, 1, 1) * h + torch.arange(h, device=DEV).view(1, -1, 1)) * slab
    block, g, j = x // 32, (x // 4) % 4, (x % 32) // 16 * 4 + x % 4
    byte, group = torch.arange(d // 2, device=DEV), torch.arange(d // 32, device=DEV)
    column, within = byte // (d // 32), byte % (d // 32)
    at = {"k": base + x * (d // 2) + byte,
          "v": base + ps * d // 2 + (((block * 4 + g) * 16 + column) * 8 + j) * (d // 32) + within,
          "ks": base + ps * d + x * (d // 32) + group,
          "vs": base + ps * (d + d // 32) + ((block * 4 + g) * (d // 32) + group) * 8 + j}
    for name in "kv":
        code, scale = _quantise(st[name].float())
        pool[at[name]] = code[..., 0::2] | (code[..., 1::2] << 4)
        pool[at[name + "s"]] = scale
    back = []
    for name in "kv":
        two = pool[at[name]]
        back.append(_values(torch.stack([two & 15, two >> 4], -1).flatten(-2), pool[at[name + "s"]]))
    return back


def _plain_attention(st: dict) -> torch.Tensor:
    c = st["case"]
    table, lens = st["table"], st["kv_lens"].long()
    batch, width = table.shape
    h, d, ps, g = c["hkv"], c["d"], c["page"], c["hq"] // c["hkv"]
    n, kv = max(_rows(c)), width * ps
    k, v = (t.view(batch, width, h, ps, d).transpose(1, 2).reshape(batch, h, kv, d)
            for t in _unpack(c, st["pool"][table.clamp(min=0).long().view(-1)]))
    key = torch.arange(kv, device=DEV)
    held = (key < lens.view(-1, 1)).view(batch, 1, kv, 1)
    k, v = torch.where(held, k, 0.0), torch.where(held, v, 0.0)
    # rows of a sequence side by side, the last of them at its end
    count = (st["starts"][1:] - st["starts"][:-1]).long()
    i = torch.arange(n, device=DEV)
    real = i < count.view(-1, 1)
    at = (st["starts"][:-1].long().view(-1, 1) + i).clamp(max=st["q"].shape[0] - 1)
    pos = (lens - count).view(-1, 1) + i
    q = st["q"].float()[at.view(-1)].view(batch, n, h, g, d).permute(0, 2, 3, 1, 4).reshape(batch * h, g * n, d)
    s = torch.bmm(q, k.transpose(2, 3).reshape(batch * h, d, kv).contiguous()).view(batch, h, g, n, kv) * (1 / math.sqrt(d))
    if c["softcap"]:
        s = torch.tanh(s / c["softcap"]) * c["softcap"]
    see = (key <= pos.unsqueeze(-1)) & (key < lens.view(-1, 1, 1))
    if c["window"]:
        see &= key > pos.unsqueeze(-1) - c["window"]
    s = torch.where(see.view(batch, 1, 1, n, kv), s, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = torch.bmm(p.reshape(batch * h, g * n, kv), v.reshape(batch * h, kv, d)).view(batch, h, g, n, d)
    o = torch.where(total > 0, o / total, 0.0).permute(0, 3, 1, 2, 4).reshape(batch, n, c["hq"], d)
    out = torch.zeros((st["q"].shape[0] + 1, c["hq"], d), device=DEV)
    out[torch.where(real, at, st["q"].shape[0]).view(-1)] = o.reshape(-1, c["hq"], d)
    return out[:-1].to(st["q"].dtype)


def _plain_take(refs: torch.Tensor, rank: torch.Tensor) -> torch.Tensor:
    """The rank-th free page (no sequence holds it), from 0, in the order of the ids."""
    return torch.searchsorted((refs == 0).cumsum(0), rank + 1).int()


def _plain_pages(st: dict) -> None:
    c = st["case"]
    if c["kind"] == "copy":
        st["pool"][:, st["dst"].long()] = st["pool"][:, st["src"].long()]
        st["status"].zero_()
        return
    ps, table, lens, refs = c["page"], st["table"], st["kv_lens"], st["refs"]
    st["meta"].copy_(st["saved"])
    col = torch.arange(table.shape[1], device=DEV)
    if c["kind"] == "extend":
        src, dst = st["src"].long(), st["dst"].long()
        n = lens[src]
        old, new = (n + ps - 1) // ps, (n + st["add"] + ps - 1) // ps
        first = (new - old).cumsum(0) - (new - old)
        fresh = (col >= old.view(-1, 1)) & (col < new.view(-1, 1))
        ids = _plain_take(refs, first.view(-1, 1) + col - old.view(-1, 1))
        table[src] = torch.where(fresh, ids, table[src])
        refs.index_add_(0, torch.where(fresh, ids, 0).view(-1), fresh.int().view(-1))
        lens[src] = n + st["add"]
        held = col < ((lens[dst] + ps - 1) // ps).view(-1, 1)
        refs.index_add_(0, torch.where(held, table[dst], 0).view(-1), -held.int().view(-1))
        table[dst] = -1
        lens[dst] = 0
    elif c["kind"] == "fork":
        src, dst, pool = st["src"].long(), st["dst"].long(), st["pool"]
        n = lens[src]
        full, part = (n // ps).view(-1, 1), (n % ps > 0).view(-1, 1)
        fresh = _plain_take(refs, part.view(-1).cumsum(0) - 1).view(-1, 1)
        rows = table[src]
        last = rows.gather(1, full.long().clamp(max=table.shape[1] - 1))
        mine = torch.where(col < full, rows, torch.where((col == full) & part, fresh, -1))
        table[dst] = mine
        refs.index_add_(0, mine.clamp(min=0).view(-1), (mine >= 0).int().view(-1))
        lens[dst] = n
        frm, to = torch.where(part, last, rows[:, :1]).view(-1), torch.where(part, fresh, rows[:, :1]).view(-1)
        pool[:, to.long()] = pool[:, frm.long()]
    else:
        ids, live = torch.arange(refs.numel(), device=DEV), refs > 0
        count = live.sum()
        high, low = live & (ids >= count), ~live & (ids < count)
        to = torch.searchsorted(low.cumsum(0), high.cumsum(0))
        remap = torch.where(high, to, ids).int()
        frm = high.nonzero().view(-1)
        st["pool"][:, remap[frm].long()] = st["pool"][:, frm]
        held = col < ((lens + ps - 1) // ps).view(-1, 1)
        table.copy_(torch.where(held, remap[table.clamp(min=0).long()], table))
        moved = torch.zeros_like(refs)
        moved.index_add_(0, remap, torch.where(live, refs, 0))
        refs.copy_(moved)
    st["status"].zero_()


# ---- a pass ------------------------------------------------------------------------

def _cache(st: dict):
    """The cache as the framework takes it; a program keeps it."""
    from doe_amd import ops
    if "cache" not in st:
        c, b = st["case"], st["buf"]
        st["cache"] = ops.Mx4Cache(b["pool"], b["table"], b["kv_lens"], page_size=c["page"], num_kv_heads=c["hkv"],
                                   head_dim=c["d"], num_pages=st["pool"].shape[0], batch=c["batch"],
                                   table_stride=st["table"].shape[1])
    return st["cache"]


def _pages(st: dict):
    from doe_amd import ops
    if "pages" not in st:
        c, b = st["case"], st["buf"]
        pool = dict(layers=c["layers"], page_bytes=_page_bytes(c)) if "pool" in st else {}
        st["pages"] = ops.KvPages(b["table"], b["kv_lens"], b["refs"], page_size=c["page"],
                                  num_pages=st["refs"].numel(), max_seqs=st["table"].shape[0],
                                  table_stride=st["table"].shape[1], pools=b.get("pool"), **pool)
    return st["pages"]


def _own(st: dict):
    import doe_amd
    from doe_amd import ops
    doe_amd.init(0)
    c, b, kind = st["case"], st["buf"], st["case"]["kind"]
    rows = st["rows"]
    if kind == "write":
        ops.mx4_kv_write(_cache(st), b["k"], b["v"], rows, row_starts=b["starts"], in_f16=c["f16"])
        ops.mx4_kv_read(_cache(st), b["k_back"], b["v_back"], rows, row_starts=b["starts"])
        return
    if kind in ("token", "prompt"):
        how = dict(num_heads=c["hq"], scale=1 / math.sqrt(c["d"]), q_f16=c["f16"], out_f16=c["f16"],
                   softcap=c["softcap"], sliding_window=c["window"], workspace=b["scratch"])
        if kind == "token":
            ops.attention_mx4(_cache(st), b["q"], b["out"], **how)
        else:
            ops.attention_mx4_prompt(_cache(st), b["q"], b["out"], rows, row_starts=b["starts"], **how)
        return
    if kind == "copy":
        ops.kv_pages_copy(b["pool"], b["src"], b["dst"], c["count"], layers=c["layers"], num_pages=c["pages"],
                          page_bytes=_page_bytes(c), status=b["status"], workspace=b["scratch"])
        return
    st["meta"].copy_(st["saved"])
    if kind == "extend":
        ops.kv_pages_extend(_pages(st), b["src"], b["add"], c["grow"], status=b["status"], workspace=b["scratch"])
        ops.kv_pages_free(_pages(st), b["dst"], c["end"], status=b["status"], workspace=b["scratch"])
    elif kind == "fork":
        ops.kv_pages_fork(_pages(st), b["src"], b["dst"], st["src"].numel(), status=b["status"],
                          workspace=b["scratch"])
    else:
        ops.kv_pages_compact(_pages(st), status=b["status"], workspace=b["scratch"])


def run(state: dict):
    st, kind = state, state["case"]["kind"]
    if "rows" not in st:
        st["rows"] = sum(_rows(st["case"])) if "n" in st["case"] or kind == "token" else 0
    if own:
        _own(st)
    if kind == "write":
        k, v = (st["k_back"], st["v_back"]) if own else _plain_write(st)
        return {"k": k, "v": v}
    if kind in ("token", "prompt"):
        return st["out"] if own else _plain_attention(st)
    if not own:
        _plain_pages(st)
    return {name: st[name] for name in ("meta", "pool", "status") if name in st}


# ---- the operators in 64 bits, from their definition ----------------------------------

def _exact_round(x: torch.Tensor) -> torch.Tensor:
    """The values that rows [..., D] are held as."""
    b = x.double().view(*x.shape[:-1], -1, 32)
    top = b.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(top)  # top = m 2^e, m in [0.5, 1)
    e = torch.where(top > 0, e - 3 + (m >= 0.875).int(), -23).clamp(-23, 13)
    y = (b / torch.exp2(e.double())).unsqueeze(-1).abs()
    grid = torch.tensor(VALUES, dtype=torch.float64, device=x.device)
    off = (y - grid).abs()
    # the even code of two that are as near
    off = off + 1e-12 * (torch.arange(8, device=x.device) % 2) * (off > 0)
    v = grid[off.argmin(-1)] * torch.sign(b) * torch.exp2(e.double())
    return v.view(x.shape)


def _exact_cells(c: dict, pool: torch.Tensor, table: torch.Tensor, n: int, head: int):
    """K and V [n][D] in 64 bits of one head of a sequence: each value from its own nibble."""
    d, ps = c["d"], c["page"]
    pos = torch.arange(n, device=DEV).view(-1, 1)
    dim = torch.arange(d, device=DEV).view(1, -1)
    x, slab = pos % ps, ps * (d + d // 16)
    base = table.long()[pos // ps] * (slab * c["hkv"]) + head * slab
    x32, col = x % 32, dim // (d // 16)
    j = (x32 // 16) * 4 + x32 % 4
    quad = x // 32 * 4 + (x32 // 4) % 4
    places = ((x * (d // 2) + dim // 2, ps * d + x * (d // 32) + dim // 32),
              (ps * d // 2 + ((quad * 16 + col) * 8 + j) * (d // 32) + dim % (d // 16) // 2,
               ps * d + ps * (d // 32) + (quad * (d // 32) + dim // 32) * 8 + j))
    grid = torch.tensor(VALUES, dtype=torch.float64, device=DEV)
    flat, out = pool.view(-1), []
    for code_at, scale_at in places:
        byte = flat[base + code_at].long()
        code = torch.where(dim % 2 == 0, byte % 16, byte // 16)
        out.append(grid[code % 8] * (1 - 2 * (code // 8)) * torch.exp2(flat[base + scale_at].double() - 127))
    return out


def exact(case: dict, seed: int):
    c = case
    if c["kind"] in ("extend", "fork", "compact", "copy"):
        return None
    st = prepare(case, seed)
    if c["kind"] == "write":
        return {"k": _exact_round(st["k"]), "v": _exact_round(st["v"])}
    rows, lens, g = _rows(c), _lens(c), c["hq"] // c["hkv"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
    at = 0
    for b, (n, m) in enumerate(zip(rows, lens)):
        pos = torch.arange(m - n, m, device=DEV).view(-1, 1)
        key = torch.arange(m, device=DEV).view(1, -1)
        hide = key > pos
        if c["window"]:
            hide = hide | (key < pos - c["window"] + 1)
        for h in range(c["hkv"]):
            k, v = _exact_cells(c, st["pool"], st["table"][b], m, h)
            for head in range(h * g, (h + 1) * g):
                s = st["q"][at:at + n, head].double() @ k.t().contiguous() / math.sqrt(c["d"])
                if c["softcap"]:
                    s = c["softcap"] * torch.tanh(s / c["softcap"])
                out[at:at + n, head] = torch.softmax(s.masked_fill(hide, -math.inf), -1) @ v
        at += n
    return out
