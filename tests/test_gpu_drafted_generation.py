"""The head norms, the 8-bit cache and the verification as they are used together:
examples/drafted_generation.py step by step against float64 restatements of each
call on what the step before left, and a step captured into a graph."""
import importlib.util
from pathlib import Path

import numpy as np
import pytest
import torch

from ouroboros_amd import ops
from ouroboros_amd.kvcache import KVCache8, attend8_workspace_bytes

from test_gpu_kv8_attend import U
from test_gpu_kv8_attend import plain as attention
from test_gpu_kv8_cache import Cache8
from test_gpu_qk_rope import plain as rotated
from test_gpu_verify import plain as judged

pytestmark = pytest.mark.gpu


def example():
    path = Path(__file__).resolve().parents[1] / "examples" / "drafted_generation.py"
    spec = importlib.util.spec_from_file_location("drafted_generation", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


@pytest.mark.parametrize("seqs,text,steps,drafts,window,temperature", [(3, 37, 8, 4, 0, 1.0), (2, 20, 6, 2, 24, 0.7), (2, 50, 5, 3, 0, 0.0), (1, 5, 4, 0, 0, 1.0)])
def test_example(gpu, seqs, text, steps, drafts, window, temperature):
    """Bars as of each call's own test: the rotated rows are within those of
    test_gpu_qk_rope; codes and scales follow from the device's own rows bit for bit, so
    that attention is held to its bar on them; the verdicts are equal."""
    m = example()
    w = m.weights(5)
    first = np.random.default_rng(6).integers(0, m.VOCAB, (seqs, text)).astype(np.int32)
    r = m.run(w, first, steps, drafts, window, temperature, 7)
    assert len(r["steps"]) == steps + 1
    most = text + (steps + 1) * (drafts + 1)
    t = Cache8(0, seqs, most, m.N_HEAD_KV, m.HEAD_DIM, m.PAGE, m.BLOCK)
    t.table, t.n_pages = r["table"], r["table"].size
    d, kv, hq = m.HEAD_DIM, m.N_HEAD_KV, m.N_HEAD
    before = np.zeros(seqs, np.int64)
    for i, s in enumerate(r["steps"]):
        n = s["fed"].shape[1]
        rows = seqs * n
        assert np.array_equal(s["lens"], before + n)
        pos = (s["lens"][:, None] - n + np.arange(n)).reshape(1, -1)
        for raw, got, gain, h in ((s["raw"][0], s["q"], w["q_gain"], hq), (s["raw"][1], s["k"], w["k_gain"], kv)):
            want, size = rotated(raw.astype(np.float64).reshape(rows, h, d), gain, pos, np.zeros(m.N_ROT // 2, int), w["freq"], False, 1e-6)
            assert (np.abs(got.reshape(rows, h, d) - want) <= 32 * U * size).all(), i
        t.write([s[x].astype(np.float64).reshape(rows, kv, d) for x in ("k", "v")], s["lens"], [n] * seqs, np.arange(seqs) * n)
        for b in range(seqs):
            L = int(s["lens"][b])
            k, v, _ = t.values(b, 0, L)
            for x in range(n):
                at, j = L - n + x, np.arange(L)
                seen = (j <= at) & ((at - j < window) | (j < m.SINKS) if window else True)
                o, _, size, spread = attention(s["q"].reshape(seqs, n, hq, d)[b, x].astype(np.float64), k, v, seen, d ** -0.5)
                bar = (16 * U * size[:, None] + 600 * U) * spread + L * 2.0 ** -39 * np.abs(v).max()
                assert (np.abs(s["out"].reshape(seqs, n, hq, d)[b, x] - o) <= bar).all(), (i, b, x)
            logits = s["logits"].reshape(seqs, n, m.VOCAB)[b].astype(np.float64)
            heat = float(np.float32(temperature))
            if i == 0:
                a, token, margin = judged(logits[-1:], None, s["fed"][b, -1:], heat, s["u"][b], float(s["u_next"][b]))
            else:
                a, token, margin = judged(logits, s["guesses"][b].astype(np.float64) if drafts else None, s["fed"][b], heat,
                                          s["u"][b].astype(np.float64), float(s["u_next"][b]))
            assert margin > 1e-10
            assert (a, token) == (s["accepted"][b], s["next"][b]), (i, b)
            assert s["lens_out"][b] == L - (0 if i == 0 else n - 1 - a)
        before = s["lens_out"].astype(np.int64)
    for b, answer in enumerate(r["answers"]):
        assert len(answer) == 1 + sum(int(s["accepted"][b]) + 1 for s in r["steps"][1:])


class Step:
    """Rotation, write, attention and verification of three sequences with their own buffers."""
    B, T, HQ, KV, D, PAGE, N = 3, 4, 8, 2, 64, 32, 512

    def __init__(self):
        g = torch.Generator().manual_seed(3)
        B, T, HQ, KV, D, PAGE, N = self.B, self.T, self.HQ, self.KV, self.D, self.PAGE, self.N
        pages, rows = 40, B * T
        new = lambda *s: torch.randn(*s, generator=g).cuda()
        self.codes = [torch.zeros(B * pages, PAGE, KV, D, dtype=torch.int8).cuda() for _ in range(2)]
        self.scales = [torch.zeros(B * pages, PAGE // 16, KV).cuda() for _ in range(2)]
        self.table = torch.randperm(B * pages, generator=g).int().reshape(B, pages).cuda()
        self.q, self.k, self.v, self.x, self.y = new(rows, HQ, D), new(rows, KV, D), new(rows, KV, D), 2 * new(rows, N), 2 * new(rows, N)
        self.qr, self.kr, self.out = (torch.zeros_like(t) for t in (self.q, self.k, self.q))
        self.lse = torch.zeros(rows, HQ).cuda()
        self.gain, self.freq = torch.rand(D, generator=g).cuda(), torch.rand(D // 2, generator=g).cuda()
        self.lens, self.lens_out = torch.tensor([900, 40, 600]).int().cuda(), torch.zeros(B).int().cuda()
        self.cu = torch.tensor([0, 4, 7, 11]).int().cuda()  # ragged, the last row nobody's
        self.pos = torch.zeros(rows).int().cuda()
        self.tokens = torch.randint(0, N, (rows,), generator=g).int().cuda()
        self.u, self.un = torch.rand(rows, generator=g).cuda(), torch.rand(B, generator=g).cuda()
        self.said = [torch.zeros(B).int().cuda() for _ in range(2)]
        self.scratch = [torch.zeros(max(n, 16), dtype=torch.uint8).cuda() for n in (
            attend8_workspace_bytes(B, rows, T, HQ, KV, D, pages * PAGE), ops.verify_workspace_bytes(B, rows, N))]
        p = lambda t: t.data_ptr()
        self.cache = KVCache8(*map(p, self.codes), *map(p, self.scales), p(self.table), n_pages=B * pages, max_pages=pages, page_tokens=PAGE,
                              block_tokens=16, n_head_kv=KV, head_dim=D)
        self.slots = pages * PAGE
        held = torch.randn(900 * B, KV, D, generator=g).cuda()
        full = torch.full((B,), 900).int().cuda()
        self.cache.write(p(held), p(held), p(full), B, 900 * B, 900)
        torch.cuda.synchronize()

    def step(self, stream):
        p = lambda t: t.data_ptr()
        B, T, rows = self.B, self.T, self.B * self.T
        ops.qk_norm_rope(p(self.q), p(self.k), p(self.qr), p(self.kr), p(self.pos), p(self.freq), rows=rows, n_head=self.HQ, n_head_kv=self.KV,
                         head_dim=self.D, n_rot=self.D, q_gain=p(self.gain), k_gain=p(self.gain), stream=stream)
        self.cache.write(p(self.kr), p(self.v), p(self.lens), B, rows, T, cu=p(self.cu), stream=stream)
        self.cache.attend(p(self.qr), p(self.out), p(self.lens), B, rows, T, self.slots, self.HQ, cu=p(self.cu), lse=p(self.lse),
                          workspace=p(self.scratch[0]), stream=stream)
        ops.verify_drafts(p(self.x), p(self.tokens), p(self.u), p(self.un), p(self.said[0]), p(self.said[1]), seqs=B, rows=rows, max_new=T,
                          n=self.N, cu=p(self.cu), draft=p(self.y), lens=p(self.lens), lens_out=p(self.lens_out), workspace=p(self.scratch[1]),
                          stream=stream)

    def next(self, i):
        """The next step's inputs, in place: the refused rows are taken back, four, three and four slots come."""
        self.lens.copy_(self.lens_out + torch.tensor([4, 3, 4]).int().cuda())
        for t, f in ((self.q, 0.9), (self.k, -1.2), (self.v, 1.1), (self.x, 0.97), (self.y, 0.95)):
            t.copy_(t.flip(0) * f)
        for t in (self.u, self.un):
            t.copy_((t * 7.3 + 0.1 * i) % 1.0)
        self.tokens.copy_((self.tokens * 5 + i) % self.N)
        self.pos.add_(17)

    def all(self):
        return [t.cpu().numpy() for t in (*self.codes, *self.scales, self.qr, self.kr, self.out, self.lse, *self.said, self.lens_out)]


def test_captured_step(gpu):
    plain, captured = Step(), Step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        plain.step(s.cuda_stream)  # a first call outside any capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        captured.step(torch.cuda.current_stream().cuda_stream)
    for i in range(5):
        graph.replay()
        torch.cuda.synchronize()
        for n, (a, b) in enumerate(zip(plain.all(), captured.all())):
            assert np.array_equal(a.view(np.uint8), b.view(np.uint8)), (i, n)
        for x in (plain, captured):
            x.next(i + 1)
        torch.cuda.synchronize()
        plain.step(None)
        torch.cuda.synchronize()
