"""A serving program's steps of many requests with adapters and beams, as the
calls are used together: a quantized projection with each request's adapter
beside it, rotation and appending to the paged cache, attention over it, logits,
the choice of beams, and pages, states and records in the order of the parents.
Every step against the host, which keeps each sequence by itself."""
import numpy as np
import pytest

from doe_amd import DeviceBuffer, Graph, Stream, mx4, ops, q4k, synchronize
from test_gpu_beam import oracle
from test_gpu_rope_append import rotate

pytestmark = pytest.mark.gpu

up = DeviceBuffer.from_array
i32 = lambda x: np.asarray(x, np.int32)  # noqa: E731

HQ, HKV, D, K, PS, VOCAB, RANK, ADAPTERS = 4, 2, 64, 256, 32, 700, 16, 3
WIDTH = (HQ + 2 * HKV) * D


class Program:
    """Device buffers of `batch` requests of `beams` sequences, and the step's calls."""

    def __init__(self, seed, batch, beams, prompt, steps):
        rng = np.random.default_rng(seed)
        self.rng, self.batch, self.beams, self.n = rng, batch, beams, batch * beams
        n, self.stride, self.pages = self.n, -(-(max(prompt) + steps + 1) // PS), 80
        self.w = q4k.random_q4k(rng, WIDTH, K)
        self.wdq = DeviceBuffer.empty((WIDTH, K), np.float32)
        self.dw = up(self.w)
        ops.dequant_q4k(self.dw, self.wdq, WIDTH, K)
        self.weights = self.wdq.download().astype(np.float64)
        self.embed = rng.standard_normal((VOCAB, K)).astype(np.float32) * 3
        self.head = (rng.standard_normal((VOCAB, HQ * D)) / 8).astype(np.float16)
        self.a = (rng.standard_normal((ADAPTERS, 3 * RANK, K)) / 16).astype(np.float16)
        self.b = rng.standard_normal((ADAPTERS, WIDTH, RANK)).astype(np.float16)
        self.scales = rng.uniform(0.1, 0.3, ADAPTERS).astype(np.float32) * np.float32(np.abs(self.weights).mean())
        self.slices = [HQ * D, HKV * D, HKV * D]
        self.lora = ops.Lora(up(self.a), up(self.b), up(self.scales), num_adapters=ADAPTERS, rank=RANK, k=K, slice_n=self.slices)
        self.request_adapter = rng.integers(-1, ADAPTERS, batch)
        self.ids = up(i32(np.repeat(self.request_adapter, beams)))
        angle = rng.uniform(-np.pi, np.pi, (self.stride * PS, D // 2))
        self.freq = np.stack([np.cos(angle), np.sin(angle)], -1).astype(np.float32)
        self.dfreq, self.dhead, self.dembed = up(self.freq), up(self.head), up(self.embed)
        self.table, self.lens, self.refs = up(np.full((n, self.stride), -1, np.int32)), up(np.zeros(n, np.int32)), up(np.zeros(self.pages, np.int32))
        self.page_bytes = mx4.page_bytes(PS, HKV, D)
        self.pool = up(rng.integers(0, 256, self.pages * self.page_bytes).astype(np.uint8))
        self.kv = ops.KvPages(self.table, self.lens, self.refs, max_seqs=n, table_stride=self.stride, num_pages=self.pages, page_size=PS,
                              pools=self.pool, layers=1, page_bytes=self.page_bytes)
        self.cache = ops.Mx4Cache(self.pool, self.table, self.lens, num_pages=self.pages, page_size=PS, num_kv_heads=HKV, head_dim=D,
                                  batch=n, table_stride=self.stride)
        self.all, self.ones, self.status = up(i32(range(n))), up(i32([1] * n)), up(i32([7]))
        self.status2 = up(i32([7]))
        self.ws = DeviceBuffer(max(ops.kv_pages_workspace(self.pages, n, n), ops.attention_mx4_workspace(n, HQ, HKV, D),
                                   ops.lora_workspace(self.lora, 256), ops.beam_select_workspace(batch, beams, VOCAB, beams),
                                   ops.attention_mx4_workspace(n, HQ, HKV, D, n), ops.attention_mx4_workspace(n, HQ, HKV, D, sum(prompt)), ops.beam_reorder_pages_workspace(self.pages, n, n)))
        self.x, self.qkv = DeviceBuffer.empty((n, K), np.float32), DeviceBuffer.empty((n, WIDTH), np.float32)
        self.out, self.logits = DeviceBuffer.empty((n, HQ * D), np.float32), DeviceBuffer.empty((n, VOCAB), np.float32)
        self.tokens, self.parents = up(i32(rng.integers(0, VOCAB, n))), up(np.zeros(n, np.int32))
        first = np.full((batch, beams), -np.inf, np.float32)
        first[:, 0] = 0
        self.scores, self.finished = [up(first), up(first)], [up(np.zeros(n, np.int32)) for _ in range(2)]
        # what else a program keeps of every sequence (here its number, to see it move)
        self.record = [up(i32(np.arange(n)[:, None] * [1, 100, 10000])) for _ in range(2)]

    def project(self, rows, x, qkv, ids, stream=None, **segments):
        ops.matmul_q4k_gemm_f32(x, self.dw, qkv, rows, WIDTH, K, stream=stream)
        ops.lora_add(self.lora, ids, x, qkv, rows, workspace=self.ws, stream=stream, **segments)

    def step(self, turn, stream=None):
        """One step: the sequences' tokens in, their successors out."""
        n, old, new = self.n, turn & 1, ~turn & 1
        ops.embed(self.dembed16, self.tokens, self.x, n, VOCAB, K, stream=stream)
        ops.kv_pages_extend(self.kv, self.all, self.ones, n, status=self.status, workspace=self.ws, stream=stream)
        self.project(n, self.x, self.qkv, self.ids, stream=stream)
        ops.qkv_rope_append(self.cache, self.qkv, self.qkv, n, num_heads=HQ, freq_cis=self.dfreq, max_positions=len(self.freq), stream=stream)
        # (the queries lie in rows of the projection)
        ops.attention_mx4_prompt(self.cache, self.qkv, self.out, n, num_heads=HQ, scale=0.125, workspace=self.ws, q_row_stride=WIDTH,
                                 stream=stream)
        ops.lm_head_gemv(self.out, self.dhead, self.logits, n, VOCAB, HQ * D, stream=stream)
        ops.beam_select(self.logits, self.scores[old], batch=self.batch, beams=self.beams, vocab=VOCAB, select=self.beams,
                        parents=self.parents, tokens=self.tokens, out_scores=self.scores[new], finished=self.finished[old],
                        out_finished=self.finished[new], end_token=3, workspace=self.ws, stream=stream)
        ops.beam_reorder_pages(self.kv, self.parents, n, status=self.status2, workspace=self.ws, stream=stream)
        ops.beam_reorder_rows(self.record[old], self.record[new], self.parents, n, row_bytes=12, stream=stream)


class Host:
    """The same sequences, each by itself."""

    def __init__(self, p):
        self.p = p
        self.k, self.v = [[] for _ in range(p.n)], [[] for _ in range(p.n)]
        self.record = [p.record[i].download() for i in range(2)]

    def row(self, x, adapter):
        """The projection's row with its adapter, in 64 bits."""
        p = self.p
        y = x.astype(np.float64) @ p.weights.T
        if 0 <= adapter < ADAPTERS:
            t, col = x.astype(np.float64) @ p.a[adapter].astype(np.float64).T, 0
            for i, w in enumerate(p.slices):
                y[col:col + w] += float(p.scales[adapter]) * p.b[adapter, col:col + w].astype(np.float64) @ t[i * RANK:(i + 1) * RANK]
                col += w
        return y

    def append(self, s, row):
        """A row of the device's projection into sequence s, as the cache holds it; its query."""
        pos = len(self.k[s])
        heads = row.reshape(1, -1, D).astype(np.float32)
        turned = rotate(heads[:, :HQ + HKV], self.p.freq[pos:pos + 1], False)
        k, v = turned[0, HQ:], heads[0, HQ + HKV:]
        self.k[s].append(mx4.dequantise(*mx4.quantise(k)).astype(np.float64))
        self.v[s].append(mx4.dequantise(*mx4.quantise(v)).astype(np.float64))
        return turned[0, :HQ].astype(np.float64)

    def attend(self, s, q):
        k, v = np.stack(self.k[s]), np.stack(self.v[s])
        out = np.zeros((HQ, D))
        for h in range(HQ):
            w = k[:, h * HKV // HQ] @ q[h] * 0.125
            w = np.exp(w - w.max())
            out[h] = w / w.sum() @ v[:, h * HKV // HQ]
        return out.reshape(-1)

    def reorder(self, parents):
        for name in ("k", "v"):
            old = getattr(self, name)
            setattr(self, name, [list(old[q]) if q >= 0 else [] for q in parents])


def near(got, want, tol):
    off = np.linalg.norm(np.asarray(got, np.float64) - want) / max(np.linalg.norm(want), 1e-30)
    assert off <= tol, off


@pytest.mark.parametrize("captured", [False, True], ids=["calls", "graph"])
def test_steps_of_beams_with_adapters(dev, captured):
    prompt, steps, batch, beams = [41, 3, 70], 6, 3, 4
    p = Program(11, batch, beams, prompt, steps)
    p.dembed16 = up(p.embed.astype(np.float16))
    embed = p.embed.astype(np.float16).astype(np.float32)
    # the prompts: rows of three requests in one call, into the requests' first sequences
    tokens = [p.rng.integers(0, VOCAB, n) for n in prompt]
    flat = np.concatenate(tokens)
    starts = np.zeros(p.n + 1, np.int64)
    for r in range(batch):
        starts[r * beams + 1:] += prompt[r]
    rows = len(flat)
    x, qkv, out = up(embed[flat]), DeviceBuffer.empty((rows, WIDTH), np.float32), DeviceBuffer.empty((rows, HQ * D), np.float32)
    ops.kv_pages_extend(p.kv, up(i32(range(0, p.n, beams))), up(i32(prompt)), batch, status=p.status, workspace=p.ws)
    p.project(rows, x, qkv, up(i32(p.request_adapter)), row_starts=up(i32(starts[::beams])), segments=batch)
    projected = qkv.download()
    ops.qkv_rope_append(p.cache, qkv, qkv, rows, num_heads=HQ, freq_cis=p.dfreq, max_positions=len(p.freq), row_starts=up(i32(starts)))
    ops.attention_mx4_prompt(p.cache, qkv, out, rows, num_heads=HQ, scale=0.125, workspace=p.ws, row_starts=up(i32(starts)), q_row_stride=WIDTH)
    assert p.status.download()[0] == 0
    h = Host(p)
    got, at = out.download(), 0
    for r in range(batch):
        for i in range(prompt[r]):
            near(projected[at], h.row(embed[flat[at]], p.request_adapter[r]), 2e-6)
            q = h.append(r * beams, projected[at])
            near(got[at], h.attend(r * beams, q), 2e-6)
            at += 1
    # its sequences go on as beams: all of a request from the first
    p.parents.upload(i32([s // beams * beams for s in range(p.n)]))
    ops.beam_reorder_pages(p.kv, p.parents, p.n, status=p.status, workspace=p.ws)
    assert p.status.download()[0] == 0
    h.reorder([s // beams * beams for s in range(p.n)])
    s = Stream() if captured else None
    synchronize()
    graphs = [Graph.capture(s, lambda t=t: p.step(t, s)) for t in range(2)] if captured else None
    for turn in range(steps):
        old, new = turn & 1, ~turn & 1
        took, scores, finished = p.tokens.download(), p.scores[old].download(), p.finished[old].download()
        if captured:
            graphs[old].launch(s)
            s.synchronize()
        else:
            p.step(turn)
        assert p.status.download()[0] == 0 and p.status2.download()[0] == 0
        out, logits = p.out.download(), p.logits.download()
        qkv = p.qkv.download()
        for q in range(p.n):
            want = h.row(embed[took[q]], p.request_adapter[q // beams])
            near(qkv[q, HQ * D:], want[HQ * D:], 2e-6)
            row = np.concatenate([want[:HQ * D], qkv[q, HQ * D:]])  # (the queries were rotated where they lay)
            near(qkv[q, :HQ * D], h.append(q, row).reshape(-1), 2e-6)
            near(out[q], h.attend(q, qkv[q, :HQ * D].reshape(HQ, D).astype(np.float64)), 2e-6)
            near(logits[q], p.head.astype(np.float64) @ out[q].astype(np.float64), 1e-6)
        want, _ = oracle(logits.reshape(batch, beams, VOCAB), scores.reshape(batch, beams), finished.reshape(batch, beams), beams, 1.0, 3)
        parents, chosen = p.parents.download(), p.tokens.download()
        assert np.array_equal(parents, want[0].reshape(-1)) and np.array_equal(chosen, want[1].reshape(-1))
        assert np.array_equal(p.finished[new].download(), want[3].reshape(-1))
        h.reorder(parents)
        h.record[new] = np.where(parents[:, None] >= 0, h.record[old][parents], h.record[new])
        assert np.array_equal(p.record[new].download(), h.record[new])
        lens = p.lens.download()
        assert [len(k) for k in h.k] == lens.tolist()
        # no page is lost or held twice over: the counts are those of the tables
        table, refs = p.table.download(), p.refs.download()
        held = np.bincount(table[table >= 0], minlength=p.pages)
        assert np.array_equal(held, refs)
    if captured:
        for g in graphs:
            g.destroy()
        s.destroy()
