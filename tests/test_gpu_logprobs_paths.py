"""Token log probabilities (ouro_token_logprobs) where a call takes more than
one launch of rows (over 65535), and where more segments hold a logit than the
choice of alternatives lists."""
import numpy as np
import pytest
import torch

from ouroboros_amd import ops
from ouroboros_amd.device import DeviceBuffer

from test_gpu_logprobs import check, logits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,k", [(33, 3), (500, 0), (8200, 0)])
def test_more_rows_than_a_grid(gpu, n, k):
    """Rows 0 .. 9, around 65535 and the last have the bits of calls of their own on the same memory."""
    rows = 65535 + 40
    g = torch.Generator(device="cuda").manual_seed(n)
    x = torch.randn(rows, n, generator=g, device="cuda").bfloat16()
    t = torch.randint(0, n, (rows,), generator=g, device="cuda", dtype=torch.int32)
    torch.cuda.synchronize()

    def call(first, count):
        out = {name: DeviceBuffer((count,), np.float32, zero=True) for name in ("logprob", "entropy", "lse")}
        out["rank"] = DeviceBuffer((count,), np.int32, zero=True)
        if k:
            out.update(top_id=DeviceBuffer((count, k), np.int32, zero=True), top_logprob=DeviceBuffer((count, k), np.float32, zero=True))
        ops.token_logprobs(x.data_ptr() + 2 * n * first, count, n, dtype="bf16", targets=t.data_ptr() + 4 * first, k=k, **out)
        return {name: b.download() for name, b in out.items()}

    got = call(0, rows)
    assert all((got[name] != 0).all() for name in ("entropy", "lse"))
    for a, b in ((0, 10), (65525, 65545), (rows - 10, rows)):
        for name, want in call(a, b - a).items():
            assert np.array_equal(got[name][a:b], want), (name, a)
        want = check(x[a:b].float().cpu().numpy(), t[a:b].cpu().numpy(), k, bf16=True)
        for name in set(got) & {"rank", "top_id"}:
            assert np.array_equal(got[name][a:b], want[name]), (name, a)


@pytest.mark.parametrize("groups", [40, 63])
def test_logits_in_few_groups_of_many_segments(gpu, groups):
    """All but some segments ruled out, those of fewer groups than alternatives are asked for: no bound from
    the groups, and thousands of segments with a logit (a segment: 16 lanes' vectors of a part of 8192)."""
    n = 6_000_000
    i = np.arange(n)
    segment = i // 8192 * 16 + i // 4 % 256 // 16
    x = logits(groups, 1, n)
    x[0, segment % 256 >= groups] = -np.inf
    assert (len(np.unique(segment[x[0] > -np.inf])) > 2048) == (groups > 45)
    check(x, [int(np.flatnonzero(x[0] > -np.inf)[77])], 64)
    x[0, x[0] > -np.inf] = 1.5  # ties alone
    check(x, [0], 64)
