"""ouro_qk_norm_rope at the most rows that it takes, where a workgroup a token would be 2^32 threads."""
import numpy as np
import pytest
import torch

from ouroboros_amd import ops

from test_gpu_qk_rope import U, plain

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d,n_rot", [(8, 4), (8, 8), (16, 12)])
def test_most_rows(gpu, d, n_rot):
    """Rows at both ends, around the middle and spread over all; the bar of test_gpu_qk_rope.py."""
    rows, half = 1 << 24, n_rot // 2
    g = torch.Generator(device="cuda").manual_seed(d + n_rot)
    q = 3 * torch.randn(rows, d, generator=g, device="cuda")
    pos = torch.randint(0, 5000, (rows,), generator=g, device="cuda", dtype=torch.int32)
    freq = (1e4 ** -(torch.arange(half) / half)).float().cuda()
    gain = 1 + 0.3 * torch.randn(d, generator=g, device="cuda")
    out = torch.full((rows, d), 77.0, device="cuda")
    torch.cuda.synchronize()
    ops.qk_norm_rope(q.data_ptr(), None, out.data_ptr(), None, pos.data_ptr(), freq.data_ptr(), rows=rows, n_head=1, n_head_kv=0, head_dim=d,
                     n_rot=n_rot, q_gain=gain.data_ptr())
    torch.cuda.synchronize()
    at = torch.tensor(sorted({0, 1, 2, 3, rows // 2 - 1, rows // 2, rows // 2 + 1, rows - 4, rows - 3, rows - 2, rows - 1} |
                             set(range(7, rows, 104729))), device="cuda")
    x, y, p = q[at].cpu().numpy().astype(np.float64)[:, None], out[at].cpu().numpy(), pos[at].cpu().numpy()[None]
    want, size = plain(x, gain.cpu().numpy(), p, np.zeros(half, int), freq.cpu().numpy(), False, 1e-6)
    assert (np.abs(y[:, None] - want) <= 32 * U * size).all()
    assert not (out == 77.0).all(1).any()  # every row was written
