"""Performance cases of a serving step of many requests: low-rank adapters
beside a shared projection, rotation and appending of rows to a paged cache,
and beam search with the states that follow it.

Each case is one pass that a serving program makes.  ``run`` computes it in
plain torch where ``own`` is false and through ``doe_amd.ops`` where it is true.

Kinds
  lora    y[r] += scale_a B_a (A_a x[r]) for the adapter a of each row's request;
          A [adapters][slices * rank][k], B [adapters][n][rank], the columns of
          slice s take rows s * rank .. of A; an id outside the adapters is none
  append  rows [q heads | k heads | v heads] of ragged requests: q and k rotated
          at each row's position, q out, k and v into their pages; f16 pages
          [page_size][kv heads][head_dim], or the 4-bit pages of
          ``doe_mx4_kv_write`` (their values are read back)
  beam    the best `select` of beams x vocabulary by score + log_softmax(logits *
          inv_temperature), ties to the lowest beam, then token; a finished beam
          offers its end token at its score, a beam of score -inf nothing
  pages   the page tables of sequences in the order of their parents: whole
          pages shared, a partly filled last one copied for all heirs but one
          (the parent's own slot, else the first), in every layer
  rows    dense states of every layer in the order of their parents
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
        # one token of one request beside the 2B-class decoder's o_proj: the smallest call
        dict(name="lora_token", kind="lora", rows=1, segments=0, adapters=4, rank=16, k=2048, n=2304, slices=1, bf16=False),
        # a decode step of 64 requests with adapters of their own, q/k/v projection of the 2B-class decoder
        dict(name="lora_tokens_b64", kind="lora", rows=64, segments=0, adapters=48, rank=16, k=2304, n=4096, slices=3,
             bf16=True),
        # ragged prompts of twelve requests, gate and up projections of the 2B-class decoder
        dict(name="lora_prompts_b12", kind="lora", rows=4096, segments=12, adapters=10, rank=32, k=2304, n=18432, slices=2,
             bf16=False),
        # long prompts of four requests, 31B-class up projection, wide adapters
        dict(name="lora_prompts_wide", kind="lora", rows=2048, segments=4, adapters=4, rank=64, k=5376, n=21504, slices=1,
             bf16=True),
        # one decode step's row of the 2B-class decoder
        dict(name="append_token", kind="append", batch=1, hq=8, hkv=4, d=256, n=1, past=700, rot=256, pairs=False, f16=False,
             page=64, mx4=False),
        # eight prompts of up to 2000 tokens behind what is cached, partly rotated heads, f16 queries
        dict(name="append_prompts_b8", kind="append", batch=8, hq=32, hkv=8, d=128, n=2000, past=900, rot=64, pairs=True,
             f16=True, page=16, mx4=False),
        # the same kind of batch into the cache held in 4 bits, 31B-class heads
        dict(name="append_mx4_b5", kind="append", batch=5, hq=32, hkv=16, d=256, n=700, past=300, rot=256, pairs=False,
             f16=False, page=64, mx4=True),
        # four beams of one request over the 2B-class vocabulary
        dict(name="beam_4", kind="beam", batch=1, beams=4, vocab=256000, select=4, inv_temperature=1.0, ended=False),
        # a batch of sixteen requests of eight beams, twice as many candidates, odd vocabulary
        dict(name="beam_16x8", kind="beam", batch=16, beams=8, vocab=248321, select=16, inv_temperature=1.25, ended=True),
        # twelve requests of eight beams: page tables and last pages of 26 layers of f16 K and V
        dict(name="pages_12x8", kind="pages", groups=12, beams=8, kv=1900, layers=52, hkv=4, d=256, page=32),
        # three requests of four beams
        dict(name="pages_3x4", kind="pages", groups=3, beams=4, kv=300, layers=8, hkv=1, d=64, page=16),
        # recurrent states of 48 linear-attention layers, twelve sequences
        dict(name="rows_states", kind="rows", groups=3, beams=4, layers=48, row=16 * 128 * 128),
    ]


def _log(rng, lo, hi) -> int:
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    kind = rng.choice(["lora", "lora", "lora", "append", "append", "beam", "beam", "pages", "rows"])
    if kind == "lora":
        rows, rank = _log(rng, 1, 6000), rng.choice([8, 16, 16, 24, 32, 64, 128])
        k, slices = 8 * _log(rng, 16, 2688), rng.choice([1, 1, 2, 3, 4])
        n = _log(rng, 33, 20000) + slices
        adapters = max(1, min(_log(rng, 1, 64), 2 ** 26 // (rank * (slices * k + n))))
        segments = rng.choice([0, _log(rng, 1, 32)]) if rows < 300 else _log(rng, 1, 32)
        while rows * (k + 2 * n) > 60_000_000 or rows * adapters * rank * (slices * k + n) > 2 ** 38:
            rows = max(1, rows * 3 // 4)
        return dict(kind=kind, rows=rows, segments=min(segments, rows), adapters=adapters, rank=rank, k=k, n=n, slices=slices,
                    bf16=rng.random() < 0.5)
    if kind == "append":
        mx4 = rng.random() < 0.3
        d = rng.choice([64, 128, 160, 256, 512] if mx4 else [48, 64, 80, 128, 160, 256, 512])
        batch, hkv = _log(rng, 1, 96), rng.choice([1, 2, 4, 8, 16])
        hq = hkv * rng.choice([1, 2, 3, 4, 8])
        n = rng.choice([1, _log(rng, 2, 4000)])
        rot = rng.choice([d, d, 8 * rng.randint(1, d // 8)])
        return dict(kind=kind, batch=batch, hq=hq, hkv=hkv, d=d, n=max(1, min(n, 50_000_000 // (batch * (hq + 2 * hkv) * d))),
                    past=rng.randint(0, 900), rot=rot, pairs=rng.random() < 0.4, f16=rng.random() < 0.5,
                    page=rng.choice([32, 64, 128, 256] if mx4 else [16, 32, 48, 64, 128]), mx4=mx4)
    if kind == "beam":
        beams, vocab = _log(rng, 1, 32), _log(rng, 300, 262144)
        batch = max(1, min(_log(rng, 1, 32), 30_000_000 // (beams * vocab)))
        return dict(kind=kind, batch=batch, beams=beams, vocab=vocab, select=min(64, beams * rng.choice([1, 1, 2])),
                    inv_temperature=rng.choice([1.0, 1.0, 0.7, 1.5]), ended=rng.random() < 0.5)
    layers = rng.randint(1, 52)
    groups, beams = _log(rng, 1, 12), _log(rng, 2, 8)
    if kind == "rows":
        row = _log(rng, 4, 260_000)
        return dict(kind=kind, groups=groups, beams=beams, layers=max(1, min(layers, 150_000_000 // (groups * beams * row))), row=row)
    return dict(kind=kind, groups=groups, beams=beams, kv=_log(rng, 20, 1900), layers=layers, hkv=rng.choice([1, 2, 4]),
                d=rng.choice([64, 128, 256]), page=rng.choice([16, 32]))


# ---- sizes ---------------------------------------------------------------------

def _spread(count: int, most: int, shift: float) -> list[int]:
    """`count` whole numbers over [min(1, most), most], the first of them `most`."""
    least = min(1, most)
    return [most if i == 0 else least + int((most - least) * math.modf(i * 0.6180339887 + shift)[0]) for i in range(count)]


def _segments(c: dict) -> list[int]:
    """Rows of each request of an adapter call."""
    if not c["segments"]:
        return [1] * c["rows"]
    parts = _spread(c["segments"], 1000, 0.29)
    cut = [c["rows"] * sum(parts[:i]) // sum(parts) for i in range(len(parts) + 1)]
    return [b - a for a, b in zip(cut, cut[1:])]


def _slices(c: dict) -> list[int]:
    """Columns of each projection that shares the input: the first half of them for q beside k and v, else even."""
    s, n = c["slices"], c["n"]
    first = n // 2 if s == 3 else n // s
    rest = [(n - first) * i // max(1, s - 1) for i in range(s)]
    return [first] + [b - a for a, b in zip(rest, rest[1:])] if s > 1 else [n]


def _rows(c: dict) -> list[int]:
    """Rows that an append brings for each sequence."""
    return [1] * c["batch"] if c["n"] == 1 else _spread(c["batch"], c["n"], 0.13)


def _lens(c: dict) -> list[int]:
    """Positions in use of each sequence, the call's own rows among them."""
    if c["kind"] == "pages":
        return [n for n in _spread(c["groups"], c["kv"], 0.37) for _ in range(c["beams"])]
    return [n + p for n, p in zip(_rows(c), _spread(c["batch"], c["past"], 0.37))]


def _mx4_page_bytes(c: dict) -> int:
    return c["page"] * c["hkv"] * (c["d"] + c["d"] // 16)


def _page_bytes(c: dict) -> int:
    """Of the pages that a reordering copies: f16 K or V of one layer."""
    return c["page"] * c["hkv"] * c["d"] * 2


def work(case: dict) -> dict:
    c = case
    if c["kind"] == "lora":
        used = min(c["adapters"], c["segments"] or c["rows"])
        weights = used * c["rank"] * (c["slices"] * c["k"] + c["n"])
        return {"bytes": 2 * weights + 4 * c["rows"] * (c["k"] + 2 * c["n"]),
                "flops": 2 * c["rows"] * c["rank"] * (c["slices"] * c["k"] + c["n"])}
    if c["kind"] == "append":
        rows, q, kv = sum(_rows(c)), c["hq"] * c["d"], c["hkv"] * c["d"]
        held = kv * 2 * 17 // 32 if c["mx4"] else kv * 4
        back = held + kv * 8 if c["mx4"] else 0
        return {"bytes": rows * (4 * (q + 2 * kv) + (2 if c["f16"] else 4) * q + held + back + 4 * c["rot"]),
                "flops": 3 * rows * c["rot"] * (c["hq"] + c["hkv"])}
    if c["kind"] == "beam":
        values = c["batch"] * c["beams"] * c["vocab"]
        return {"bytes": 4 * values, "flops": 4 * values}
    if c["kind"] == "rows":
        return {"bytes": 8 * c["groups"] * c["beams"] * c["layers"] * c["row"], "flops": 0}
    # about a third of the beams go on as copies of others
    lens = _lens(c)
    copies = sum(n % c["page"] > 0 for n in lens) // 3
    entries = sum(-(-n // c["page"]) for n in lens)
    return {"bytes": 2 * copies * c["layers"] * _page_bytes(c) + 16 * entries, "flops": 0}


# ---- inputs ----------------------------------------------------------------------

def _gen(seed: int) -> torch.Generator:
    return torch.Generator(DEV).manual_seed(seed)


def _ints(values) -> torch.Tensor:
    return torch.tensor(values, dtype=I32, device=DEV)


def _starts(counts) -> torch.Tensor:
    return _ints([sum(counts[:b]) for b in range(len(counts) + 1)])


def _wide(g, shape) -> torch.Tensor:
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


def _parents(g, groups: int, beams: int) -> torch.Tensor:
    """Each request's beams go on from beams of its own, the better ones more often."""
    u = torch.rand(groups, beams, generator=g, device=DEV)
    mine = (u * u * beams).int().clamp(max=beams - 1)
    return (mine + beams * torch.arange(groups, device=DEV, dtype=I32).view(-1, 1)).view(-1).contiguous()


def _prepare_lora(c: dict, g, st: dict) -> None:
    dtype = torch.bfloat16 if c["bf16"] else torch.float16
    a, r, s = c["adapters"], c["rank"], c["slices"]
    counts = _segments(c)
    st["a"] = (torch.randn(a, s * r, c["k"], generator=g, device=DEV) / math.sqrt(c["k"])).to(dtype)
    st["b"] = (torch.randn(a, c["n"], r, generator=g, device=DEV) / math.sqrt(r)).to(dtype)
    st["scales"] = 0.25 + torch.rand(a, generator=g, device=DEV)
    # a request in ten or so without an adapter
    st["ids"] = torch.randint(-1 if len(counts) > 8 else 0, a, (len(counts),), generator=g, device=DEV, dtype=I32)
    st["starts"] = _starts(counts)
    st["x"] = _wide(g, (c["rows"], c["k"]))
    st["y"] = torch.randn(c["rows"], c["n"], generator=g, device=DEV)
    st["scratch"] = torch.empty(1 << 26, dtype=torch.uint8, device=DEV)


def _prepare_append(c: dict, g, st: dict) -> None:
    rows, lens, ps = _rows(c), _lens(c), c["page"]
    total, stride = sum(rows), -(-max(lens) // ps)
    pages = sum(-(-n // ps) for n in lens) + 3
    st["qkv"] = _wide(g, (total, (c["hq"] + 2 * c["hkv"]) * c["d"]))
    st["q"] = torch.zeros((total, c["hq"], c["d"]), dtype=torch.float16 if c["f16"] else F32, device=DEV)
    angle = torch.arange(max(lens), device=DEV, dtype=torch.float64).view(-1, 1) * torch.pow(
        torch.tensor(10000.0, dtype=torch.float64, device=DEV), -torch.arange(0, c["rot"], 2, device=DEV) / c["rot"])
    st["freq"] = torch.stack([torch.cos(angle), torch.sin(angle)], -1).float().contiguous()
    st["table"], st["kv_lens"], st["starts"] = _tables(g, lens, ps, pages, stride), _ints(lens), _starts(rows)
    if c["mx4"]:
        st["pool"] = torch.zeros((pages, _mx4_page_bytes(c)), dtype=torch.uint8, device=DEV)
        for name in ("k_back", "v_back"):
            st[name] = torch.zeros((total, c["hkv"], c["d"]), device=DEV)
    else:
        for name in ("k_pool", "v_pool"):
            st[name] = torch.randn((pages, ps, c["hkv"], c["d"]), generator=g, device=DEV).half()


def _prepare_beam(c: dict, g, st: dict) -> None:
    rows, k = c["batch"] * c["beams"], c["beams"]
    st["logits"] = 2.5 * torch.randn(rows, c["vocab"], generator=g, device=DEV)
    # running scores a few nats apart; now and then a request's first step, with one beam
    st["scores"] = -20 - 6 * torch.rand(c["batch"], k, generator=g, device=DEV)
    first = torch.rand(c["batch"], 1, generator=g, device=DEV) < 0.15
    st["scores"][first & (torch.arange(k, device=DEV) > 0)] = -math.inf
    st["finished"] = (torch.rand(c["batch"], k, generator=g, device=DEV) < (0.15 if c["ended"] else 0)).int()
    for name in ("parents", "tokens", "ended"):
        st[name] = torch.zeros(c["batch"], c["select"], dtype=I32, device=DEV)
    st["best"] = torch.zeros(c["batch"], c["select"], device=DEV)
    st["scratch"] = torch.empty(1 << 27, dtype=torch.uint8, device=DEV)


def _prepare_pages(c: dict, g, st: dict) -> None:
    lens, ps = _lens(c), c["page"]
    n, stride = len(lens), -(-c["kv"] // ps) + 1
    pages = sum(-(-x // ps) for x in lens) + n + 16
    # page_table, kv_lens and page_refs in one piece, so that a pass starts from
    # the same state with one copy
    meta = torch.zeros(n * stride + n + pages, dtype=I32, device=DEV)
    table, kv_lens, refs = meta[:n * stride].view(n, stride), meta[n * stride:n * stride + n], meta[n * stride + n:]
    table.copy_(_tables(g, lens, ps, pages, stride))
    kv_lens.copy_(_ints(lens))
    # beams of a request share the pages of their common prompt
    col = torch.arange(stride, device=DEV)
    common = (kv_lens * 7 // 10 // ps).view(-1, 1)
    head = torch.arange(n, device=DEV) // c["beams"] * c["beams"]
    table.copy_(torch.where(col < common, table[head], table))
    refs.index_add_(0, table.clamp(min=0).view(-1), (table >= 0).int().view(-1))
    st |= {"meta": meta, "saved": meta.clone(), "table": table, "kv_lens": kv_lens, "refs": refs,
           "parents": _parents(g, c["groups"], c["beams"]), "status": torch.zeros(1, dtype=I32, device=DEV),
           "pool": torch.randint(0, 256, (c["layers"], pages, _page_bytes(c)), generator=g, device=DEV, dtype=torch.uint8),
           "scratch": torch.zeros(1 << 22, dtype=I32, device=DEV)}


def _prepare_rows(c: dict, g, st: dict) -> None:
    n = c["groups"] * c["beams"]
    st["src"] = torch.randn(c["layers"], n, c["row"], generator=g, device=DEV)
    st["dst"] = torch.zeros_like(st["src"])
    st["parents"] = _parents(g, c["groups"], c["beams"])


def prepare(case: dict, seed: int) -> dict:
    st = {"case": case}
    {"lora": _prepare_lora, "append": _prepare_append, "beam": _prepare_beam, "pages": _prepare_pages,
     "rows": _prepare_rows}[case["kind"]](case, _gen(seed), st)
    st["buf"] = {k: Buf(t) for k, t in st.items() if isinstance(t, torch.Tensor)}
    return st


# ---- the plain form ----------------------------------------------------------------

def _where(starts: torch.Tensor, rows: int):
    """Sequence of each row of a call, and its number in the sequence."""
    starts = starts.long()
    row = torch.arange(rows, device=DEV)
    b = torch.searchsorted(starts[1:], row, right=True)
    return b, row - starts[b]


def _plain_lora(st: dict) -> torch.Tensor:
    c = st["case"]
    a, r, s, rows = c["adapters"], c["rank"], c["slices"], c["rows"]
    mine = st["ids"][_where(st["starts"], rows)[0]]
    t = (st["x"] @ st["a"].float().view(a * s * r, c["k"]).t()).view(rows, a, s, r)
    t = torch.where((mine.view(-1, 1) == torch.arange(a, device=DEV)).view(rows, a, 1, 1), t, 0.0) * st["scales"].view(1, a, 1, 1)
    b = st["b"].float().split(_slices(c), 1)
    delta = [t[:, :, i].reshape(rows, a * r) @ b[i].transpose(1, 2).reshape(a * r, -1) for i in range(s)]
    return st["y"].add_(torch.cat(delta, 1))


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
    return code.reshape(x.shape), (e + 127).to(torch.uint8).squeeze(-1)


def _values(code: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """f32 values [..., D] of codes [..., D] and scale bytes [..., D / 32]."""
    table = torch.tensor(VALUES + tuple(-v for v in VALUES), device=code.device)
    s = torch.ldexp(torch.ones(1, device=code.device), scale.int() - 127)
    return (table[code.int()].view(*scale.shape, 32) * s.unsqueeze(-1)).view(code.shape)


def _plain_append(st: dict) -> dict:
    c = st["case"]
    hq, h, d, ps, half = c["hq"], c["hkv"], c["d"], c["page"], c["rot"] // 2
    rows = st["qkv"].shape[0]
    b, i = _where(st["starts"], rows)
    count = (st["starts"][1:] - st["starts"][:-1]).long()
    pos = st["kv_lens"].long()[b] - count[b] + i
    x = st["qkv"].view(rows, hq + 2 * h, d)
    cos, sin = st["freq"][pos].unsqueeze(1).unbind(-1)
    qk = x[:, :hq + h]
    if c["pairs"]:
        x0, x1 = qk[..., 0:2 * half:2], qk[..., 1:2 * half:2]
        turned = torch.stack([x0 * cos - x1 * sin, x0 * sin + x1 * cos], -1).flatten(-2)
    else:
        x0, x1 = qk[..., :half], qk[..., half:2 * half]
        turned = torch.cat([x0 * cos - x1 * sin, x0 * sin + x1 * cos], -1)
    qk = torch.cat([turned, qk[..., 2 * half:]], -1)
    st["q"].copy_(qk[:, :hq])
    page = st["table"].long()[b, pos // ps]
    if not c["mx4"]:
        for name, v in (("k_pool", qk[:, hq:]), ("v_pool", x[:, hq + h:])):
            st[name].view(-1, h, d)[page * ps + pos % ps] = v.half()
        return {name: st[name] for name in ("q", "k_pool", "v_pool")}
    pool, slab = st["pool"].view(-1), _mx4_page_bytes(c) // h
    at_x = (pos % ps).view(-1, 1, 1)
    base = (page.view(-1, 1, 1) * h + torch.arange(h, device=DEV).view(1, -1, 1)) * slab
    block, g, j = at_x // 32, (at_x // 4) % 4, (at_x % 32) // 16 * 4 + at_x % 4
    byte, group = torch.arange(d // 2, device=DEV), torch.arange(d // 32, device=DEV)
    column, within = byte // (d // 32), byte % (d // 32)
    at = {"k": base + at_x * (d // 2) + byte,
          "v": base + ps * d // 2 + (((block * 4 + g) * 16 + column) * 8 + j) * (d // 32) + within,
          "ks": base + ps * d + at_x * (d // 32) + group,
          "vs": base + ps * (d + d // 32) + ((block * 4 + g) * (d // 32) + group) * 8 + j}
    back = {}
    for name, v in (("k", qk[:, hq:].contiguous()), ("v", x[:, hq + h:].contiguous())):
        code, scale = _quantise(v)
        pool[at[name]] = code[..., 0::2] | (code[..., 1::2] << 4)
        pool[at[name + "s"]] = scale
        two = pool[at[name]]
        back[name] = _values(torch.stack([two & 15, two >> 4], -1).flatten(-2), pool[at[name + "s"]])
    return {"q": st["q"], **back}


END = 1  # the end token


def _plain_beam(st: dict) -> dict:
    c = st["case"]
    batch, k, vocab, select = c["batch"], c["beams"], c["vocab"], c["select"]
    logits, scores = st["logits"], st["scores"].double()
    x = logits.double() * c["inv_temperature"]
    top = x.amax(-1, keepdim=True)
    lse = (torch.exp(x - top).sum(-1, keepdim=True).log() + top).view(batch, k, 1)
    # the best of each row, whole numbers in the order of (logit, lowest token)
    bits = logits.view(I32).long()
    key = torch.where(bits < 0, -(bits & 0x7fffffff), bits) * 2 ** 24 + (2 ** 24 - 1 - torch.arange(vocab, device=DEV))
    few = min(select, vocab)
    token = (2 ** 24 - 1 - (torch.topk(key, few, -1).values & (2 ** 24 - 1))).view(batch, k, few)
    logit = logits.view(batch, k, vocab).gather(2, token).double() * c["inv_temperature"]
    cand = scores.unsqueeze(-1) + logit - lse
    done = st["finished"].bool().unsqueeze(-1)
    first = torch.arange(few, device=DEV) == 0
    cand = torch.where(done, torch.where(first, scores.unsqueeze(-1), -math.inf), cand).view(batch, -1)
    token = torch.where(done, END, token).view(batch, -1)
    beam = torch.arange(k, device=DEV).view(1, -1, 1).expand(batch, k, few).reshape(batch, -1)
    # ties to the lowest beam, then token
    order = torch.argsort(beam * vocab + token, dim=1, stable=True)
    order = order.gather(1, torch.argsort(cand.gather(1, order), dim=1, stable=True, descending=True))[:, :select]
    best, token, beam = (v.gather(1, order) for v in (cand, token, beam))
    full = best > -math.inf
    parent = beam + k * torch.arange(batch, device=DEV).view(-1, 1)
    ended = (done.view(batch, k).gather(1, beam) | (token == END)).int()
    short = select - best.shape[1]
    out = {"parents": torch.where(full, parent, -1).int(), "tokens": torch.where(full, token, -1).int(),
           "best": best.float(), "ended": torch.where(full, ended, 0)}
    fill = {"parents": -1, "tokens": -1, "best": -math.inf, "ended": 0}
    return {name: torch.nn.functional.pad(v, (0, short), value=fill[name]) for name, v in out.items()}


def _plain_pages(st: dict) -> None:
    c = st["case"]
    ps, table, lens, refs = c["page"], st["table"], st["kv_lens"], st["refs"]
    st["meta"].copy_(st["saved"])
    par = st["parents"].long()
    n = par.numel()
    i, col = torch.arange(n, device=DEV), torch.arange(table.shape[1], device=DEV)
    heirs = torch.zeros_like(lens).index_add_(0, par, torch.ones_like(lens))
    # the heir that keeps a parent's last page: its own slot, else the first
    first = torch.full_like(i, n).scatter_reduce(0, par, i, "amin")
    keeper = torch.where(par == i, i, first)
    old, old_lens = table.clone(), lens.clone()
    held = col < ((old_lens + ps - 1) // ps).view(-1, 1)
    whole = col < (old_lens // ps).view(-1, 1)
    part = held & ~whole
    # pages free before the call, the lowest first, in the order of the sequences
    fresh = (keeper[par] != i) & (old_lens[par] % ps > 0)
    ids = torch.searchsorted((refs == 0).cumsum(0), fresh.cumsum(0)).int()
    rows, mine = old[par], part[par]
    last = torch.where(mine, rows, -1).amax(1)
    table.copy_(torch.where(held[par], torch.where(mine & fresh.view(-1, 1), ids.view(-1, 1), rows), -1))
    lens.copy_(old_lens[par])
    gone = torch.where(whole, heirs.view(-1, 1) - 1, torch.where(part & (heirs == 0).view(-1, 1), -1, 0)).int()
    refs.index_add_(0, old.clamp(min=0).view(-1), gone.view(-1))
    refs.index_add_(0, torch.where(fresh, ids, 0), fresh.int())
    to, frm = ids[fresh].long(), last[fresh].long()
    st["pool"][:, to] = st["pool"][:, frm]
    st["status"].zero_()


# ---- a pass ------------------------------------------------------------------------

def _handle(st: dict, make):
    """What a program keeps beside its buffers."""
    if "handle" not in st:
        import doe_amd
        doe_amd.init(0)
        st["handle"] = make()
    return st["handle"]


def _own_lora(st: dict) -> torch.Tensor:
    from doe_amd import ops
    c, b = st["case"], st["buf"]
    lora = _handle(st, lambda: ops.Lora(b["a"], b["b"], b["scales"], num_adapters=c["adapters"], rank=c["rank"], k=c["k"],
                                        slice_n=_slices(c), bf16=c["bf16"]))
    if c["segments"]:
        ops.lora_add(lora, b["ids"], b["x"], b["y"], c["rows"], row_starts=b["starts"], segments=c["segments"],
                     workspace=b["scratch"])
    else:
        ops.lora_add(lora, b["ids"], b["x"], b["y"], c["rows"], workspace=b["scratch"])
    return st["y"]


def _own_append(st: dict) -> dict:
    from doe_amd import ops
    c, b = st["case"], st["buf"]

    def make():
        how = dict(page_size=c["page"], num_kv_heads=c["hkv"], head_dim=c["d"], num_pages=st["pool" if c["mx4"] else "k_pool"].shape[0],
                   batch=c["batch"], table_stride=st["table"].shape[1])
        if c["mx4"]:
            return ops.Mx4Cache(b["pool"], b["table"], b["kv_lens"], **how)
        return ops.F16Cache(b["k_pool"], b["v_pool"], b["table"], b["kv_lens"], **how)

    cache, rows = _handle(st, make), st["qkv"].shape[0]
    ops.qkv_rope_append(cache, b["qkv"], b["q"], rows, num_heads=c["hq"], freq_cis=b["freq"], max_positions=st["freq"].shape[0],
                        rotary_dim=c["rot"], interleaved=c["pairs"], q_f16=c["f16"], row_starts=b["starts"])
    if not c["mx4"]:
        return {name: st[name] for name in ("q", "k_pool", "v_pool")}
    ops.mx4_kv_read(cache, b["k_back"], b["v_back"], rows, row_starts=b["starts"])
    return {"q": st["q"], "k": st["k_back"], "v": st["v_back"]}


def _own_beam(st: dict) -> dict:
    import doe_amd
    from doe_amd import ops
    doe_amd.init(0)
    c, b = st["case"], st["buf"]
    ops.beam_select(b["logits"], b["scores"], batch=c["batch"], beams=c["beams"], vocab=c["vocab"], select=c["select"],
                    parents=b["parents"], tokens=b["tokens"], out_scores=b["best"], inv_temperature=c["inv_temperature"],
                    finished=b["finished"], out_finished=b["ended"], end_token=END, workspace=b["scratch"])
    return {name: st[name] for name in ("parents", "tokens", "best", "ended")}


def _own_pages(st: dict) -> None:
    from doe_amd import ops
    c, b = st["case"], st["buf"]
    pages = _handle(st, lambda: ops.KvPages(b["table"], b["kv_lens"], b["refs"], page_size=c["page"], layers=c["layers"],
                                            num_pages=st["refs"].numel(), max_seqs=st["table"].shape[0], pools=b["pool"],
                                            table_stride=st["table"].shape[1], page_bytes=_page_bytes(c)))
    st["meta"].copy_(st["saved"])
    ops.beam_reorder_pages(pages, b["parents"], st["parents"].numel(), status=b["status"], workspace=b["scratch"])


def run(state: dict):
    st, kind = state, state["case"]["kind"]
    if kind == "lora":
        return _own_lora(st) if own else _plain_lora(st)
    if kind == "append":
        return _own_append(st) if own else _plain_append(st)
    if kind == "beam":
        return _own_beam(st) if own else _plain_beam(st)
    if kind == "pages":
        if own:
            _own_pages(st)
        else:
            _plain_pages(st)
        return {name: st[name] for name in ("meta", "pool", "status")}
    if own:
        import doe_amd
        from doe_amd import ops
        doe_amd.init(0)
        c, b = st["case"], st["buf"]
        ops.beam_reorder_rows(b["src"], b["dst"], b["parents"], st["parents"].numel(), row_bytes=4 * c["row"], layers=c["layers"])
    else:
        torch.index_select(st["src"], 1, st["parents"], out=st["dst"])
    return st["dst"]


# ---- the operators in 64 bits, from their definition ----------------------------------

def _exact_lora(c: dict, st: dict) -> torch.Tensor:
    out, at, r = st["y"].double(), 0, c["rank"]
    for n, a in zip(_segments(c), st["ids"].tolist()):
        if 0 <= a < c["adapters"] and n:
            t = st["x"][at:at + n].double() @ st["a"][a].double().t().contiguous()
            col = 0
            for s, width in enumerate(_slices(c)):
                b = st["b"][a, col:col + width].double().t().contiguous()
                out[at:at + n, col:col + width] += float(st["scales"][a]) * (t[:, s * r:(s + 1) * r].contiguous() @ b)
                col += width
        at += n
    return out


def _exact_round(x: torch.Tensor) -> torch.Tensor:
    """The values that f32 rows [..., D] are held as in 4 bits."""
    b = x.double().reshape(*x.shape[:-1], -1, 32)
    top = b.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(top)  # top = m 2^e, m in [0.5, 1)
    e = torch.where(top > 0, e - 3 + (m >= 0.875).int(), -23).clamp(-23, 13)
    y = (b / torch.exp2(e.double())).unsqueeze(-1).abs()
    grid = torch.tensor(VALUES, dtype=torch.float64, device=x.device)
    off = (y - grid).abs()
    off = off + 1e-12 * (torch.arange(8, device=x.device) % 2) * (off > 0)  # the even code of two that are as near
    return (grid[off.argmin(-1)] * torch.sign(b) * torch.exp2(e.double())).view(x.shape)


def _exact_append(c: dict, st: dict) -> dict:
    hq, h, d, ps, rot = c["hq"], c["hkv"], c["d"], c["page"], c["rot"]
    rows, lens = _rows(c), _lens(c)
    x = st["qkv"].view(-1, hq + 2 * h, d)
    # what is held in 4 bits is the f32 rotation, rounded at each product and sum
    wide = F32 if c["mx4"] else torch.float64
    dim = torch.arange(rot, device=DEV)
    pair = dim // 2 if c["pairs"] else dim % (rot // 2)
    low = dim % 2 == 0 if c["pairs"] else dim < rot // 2
    other = torch.where(low, dim + (1 if c["pairs"] else rot // 2), dim - (1 if c["pairs"] else rot // 2))
    out = {"q": torch.zeros(x.shape[0], hq, d, dtype=torch.float64, device=DEV)}
    for name in ("k_pool", "v_pool"):
        if not c["mx4"]:
            out[name] = st[name].double()
    keys, at = [], 0
    for b, (n, m) in enumerate(zip(rows, lens)):
        angle = st["freq"][m - n:m, pair].to(wide).unsqueeze(1)
        one = x[at:at + n].to(wide)
        turned = one[:, :hq + h].clone()
        own_part, their_part = turned[..., :rot] * angle[..., 0], turned[..., other] * angle[..., 1]
        turned[..., :rot] = torch.where(low, own_part - their_part, their_part + own_part)
        out["q"][at:at + n] = turned[:, :hq].double()
        keys.append(turned[:, hq:])
        for p in range(m - n, m) if not c["mx4"] else ():
            page = int(st["table"][b, p // ps]) if p % ps == 0 or p == m - n else page
            if p % ps == 0 or p == m - n:
                stop = min(m, (p // ps + 1) * ps)
                here = slice(p % ps, p % ps + stop - p)
                out["k_pool"][page, here] = turned[p - m + n:stop - m + n, hq:]
                out["v_pool"][page, here] = one[p - m + n:stop - m + n, hq + h:]
        at += n
    if c["mx4"]:
        return {"q": out["q"], "k": _exact_round(torch.cat(keys)), "v": _exact_round(x[:, hq + h:])}
    return out


def _exact_beam(c: dict, st: dict) -> dict:
    best = torch.full((c["batch"], c["select"]), -math.inf, dtype=torch.float64, device=DEV)
    for b in range(c["batch"]):
        offers = []
        for k in range(c["beams"]):
            score = float(st["scores"][b, k])
            if score == -math.inf:
                continue
            if int(st["finished"][b, k]):
                offers.append(torch.tensor([score], dtype=torch.float64, device=DEV))
                continue
            row = torch.log_softmax(st["logits"][b * c["beams"] + k].double() * c["inv_temperature"], 0)
            offers.append(score + row.sort(descending=True).values[:c["select"]])
        found = torch.cat(offers).sort(descending=True).values[:c["select"]] if offers else best[b, :0]
        best[b, :found.numel()] = found
    return {"parents": None, "tokens": None, "best": best, "ended": None}


def exact(case: dict, seed: int):
    c = case
    if c["kind"] == "pages":
        return None
    st = prepare(case, seed)
    if c["kind"] == "rows":
        return torch.stack([st["src"][:, p] for p in st["parents"].tolist()], 1).double()
    return {"lora": _exact_lora, "append": _exact_append, "beam": _exact_beam}[c["kind"]](c, st)
