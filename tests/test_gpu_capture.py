"""A decode step over a paged cache, captured once and replayed: attention that
writes the new token and adds to the history, eviction back to the budget, log
probabilities of the outputs taken as logits.  With workspaces of their own the
calls allocate nothing and clear no memory outside their kernels, so every
replay equals, bit for bit, the same calls made one by one on a copy."""
import numpy as np
import pytest
import torch

from ouroboros_amd import _lib, kvcache, ops
from ouroboros_amd.kvcache import History, KVCache

pytestmark = pytest.mark.gpu
SEQS, HEADS, KV, D, PAGE, KEEP = 3, 8, 2, 64, 16, 400


class State:
    def __init__(self):
        g = torch.Generator().manual_seed(7)
        pages = -(-(KEEP + 1) // PAGE)
        new = lambda *s: torch.randn(*s, generator=g).cuda()
        self.k, self.v = (new(SEQS * pages, PAGE, KV, D).bfloat16() for _ in range(2))
        self.pages = torch.randperm(SEQS * pages, generator=g).int().reshape(SEQS, pages).cuda()
        self.q, self.kn, self.vn = new(SEQS, HEADS, D), new(SEQS, KV, D), new(SEQS, KV, D)
        self.weight = torch.rand(SEQS, KV, KEEP + 1, generator=g).cuda()
        self.pos = torch.arange(KEEP + 1).int().expand(SEQS, KV, KEEP + 1).contiguous().cuda()
        self.pos_new = torch.full((SEQS,), KEEP).int().cuda()
        self.lens, self.left = torch.full((SEQS,), KEEP + 1).int().cuda(), torch.zeros(SEQS).int().cuda()
        self.out = torch.zeros(SEQS, HEADS, D).cuda()
        self.src = torch.zeros(SEQS, KV, KEEP).int().cuda()
        self.targets = torch.tensor([3, 511, -1]).int().cuda()
        self.said = {n: torch.zeros(SEQS, *s).to(t).cuda() for n, t, s in (
            ("logprob", torch.float32, ()), ("rank", torch.int32, ()), ("entropy", torch.float32, ()), ("lse", torch.float32, ()),
            ("top_id", torch.int32, (4,)), ("top_logprob", torch.float32, (4,)))}
        self.scratch = [torch.zeros(max(n, 16), dtype=torch.uint8).cuda() for n in (
            kvcache.attend_workspace_bytes(SEQS, HEADS, D, KEEP + 1, True), kvcache.evict_workspace_bytes(SEQS, KV, KEEP + 1, KEEP),
            int(_lib.lib().ouro_token_logprobs_workspace_bytes(SEQS, HEADS * D, 4)))]
        p = lambda t: t.data_ptr()
        self.cache = KVCache(p(self.k), p(self.v), p(self.pages), n_pages=SEQS * pages, max_pages=pages, page_tokens=PAGE,
                             n_head_kv=KV, head_dim=D)
        self.history = History(p(self.weight), p(self.pos), KV, KEEP + 1)

    def step(self, stream):
        p = lambda t: t.data_ptr()
        self.cache.attend(p(self.q), p(self.out), p(self.lens), SEQS, KEEP + 1, HEADS, k_new=p(self.kn), v_new=p(self.vn),
                          pos_new=p(self.pos_new), history=self.history, workspace=p(self.scratch[0]), stream=stream)
        self.cache.evict(self.history, p(self.lens), SEQS, KEEP + 1, KEEP, 20, p(self.left), slot_from=p(self.src),
                         workspace=p(self.scratch[1]), stream=stream)
        ops.token_logprobs(p(self.out), SEQS, HEADS * D, targets=p(self.targets), k=4, workspace=p(self.scratch[2]), stream=stream,
                           **{n: p(t) for n, t in self.said.items()})

    def next(self, i):
        """The next step's inputs, in place."""
        for t, x in ((self.q, 0.9), (self.kn, -1.1), (self.vn, 1.05)):
            t.copy_(t.flip(0) * x)
        self.pos_new.fill_(KEEP + i)

    def all(self):
        return {n: t.cpu().numpy() for n, t in (("k", self.k.view(torch.int16)), ("v", self.v.view(torch.int16)), ("weight", self.weight),
                ("pos", self.pos), ("left", self.left), ("out", self.out), ("src", self.src), *self.said.items())}


def test_captured_step(gpu):
    plain, captured = State(), State()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        plain.step(s.cuda_stream)  # a first call outside any capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        captured.step(torch.cuda.current_stream().cuda_stream)
    for i in range(4):
        graph.replay()
        torch.cuda.synchronize()
        a, b = plain.all(), captured.all()
        for name in a:
            assert np.array_equal(a[name].view(np.uint8), b[name].view(np.uint8)), (i, name)
        for x in (plain, captured):
            x.next(i + 1)
        torch.cuda.synchronize()
        plain.step(None)
        torch.cuda.synchronize()
