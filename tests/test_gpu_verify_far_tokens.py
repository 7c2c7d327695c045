"""ouro_verify_drafts: a probability below 2^-1000 of the likeliest's counts as 0 in
what is left of p - q and in every sum, as it does where a draft is judged."""
import numpy as np
import pytest

from test_gpu_verify import Case, enc

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("far", [-692.0, -696.0, -740.0])
def test_far_tokens(gpu, bf16, far):
    """p and q agree but for a token that p has at e^far (2^-998, 2^-1004, 2^-1068): drafted it is kept
    above 2^-1000; below, it is refused, nothing is left of p - q and the next is p's other token."""
    c = Case(51, [2, 2], 3000, bf16=bf16)
    c.logits[:, :], c.draft[:, :] = enc(np.float32([-np.inf]), bf16)[0], enc(np.float32([-np.inf]), bf16)[0]
    c.logits[:, 40], c.draft[:, 40] = 0, 0
    c.logits[:, 2500] = enc(np.float32([far]), bf16)[0]
    c.tokens[[1, 3]] = 2500, 40
    c.u_accept[:] = 0.5
    got = c.check()
    assert got[0].tolist() == [1 if far > -693 else 0, 1] and (got[1] == 40).all()
