"""A captured attention call whose kernel takes more than 64 KiB of LDS (an fp32
cache of heads wider than 128): replays equal the same calls made one by one,
also where the kernel's first call is the captured one."""
import numpy as np
import pytest
import torch

from ouroboros_amd.kvcache import KVCache, attend_workspace_bytes

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page", [8, 16])
@pytest.mark.parametrize("io", ["f32", "bf16"])
def test_captured_wide_heads(gpu, page, io):
    seqs, heads, d, n = 2, 3, 256, 300
    g = torch.Generator().manual_seed(page)
    new = lambda *s: torch.randn(*s, generator=g).cuda()
    pages = -(-n // page)
    k, v = new(seqs * pages, page, 1, d), new(seqs * pages, page, 1, d)
    table = torch.randperm(seqs * pages, generator=g).int().cuda()
    lens = torch.tensor([n, 17]).int().cuda()
    q = new(seqs, heads, d).to(torch.float32 if io == "f32" else torch.bfloat16)
    c = KVCache(k.data_ptr(), v.data_ptr(), table.data_ptr(), n_pages=seqs * pages, max_pages=pages, page_tokens=page, n_head_kv=1,
                head_dim=d, dtype="f32")
    outs = [torch.zeros_like(q) for _ in range(2)]
    scratch = [torch.zeros(attend_workspace_bytes(seqs, heads, d, n), dtype=torch.uint8).cuda() for _ in range(2)]

    def call(i, stream):
        c.attend(q.data_ptr(), outs[i].data_ptr(), lens.data_ptr(), seqs, n, heads, dtype=io, workspace=scratch[i].data_ptr(), stream=stream)

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        call(0, torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        call(1, None)
        torch.cuda.synchronize()
        a, b = (o.float().cpu().numpy() for o in outs)
        assert np.array_equal(a, b) and (a != 0).all()
        q.copy_(q.flip(0) * -1.1)
        torch.cuda.synchronize()
