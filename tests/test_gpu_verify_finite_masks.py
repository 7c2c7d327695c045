"""ouro_verify_drafts where logits are masked with large finite numbers, a token is
forced by one, or the temperature is tiny: the restatement and the margins of
test_gpu_verify.py."""
import numpy as np
import pytest

from test_gpu_verify import Case, enc

pytestmark = pytest.mark.gpu
LOWEST = {False: -3.4028234663852886e38, True: -3.3895313892515355e38}  # f32, bf16


def masked(seed, bf16, draft, value, heat, n=20001):
    """Two stretches of `value`, of whole segments of 2048 each, in the target's rows and others in the drafter's."""
    c = Case(seed, [4, 1, 3, 5, 2, 6], n, bf16=bf16, draft=draft, heat=heat)
    low = enc(np.float32([LOWEST[bf16] if value is None else value]), bf16)[0]
    c.logits[:, 1500:9000] = low
    c.logits[:, 14000:n] = low
    if draft:
        c.draft[:, 3000:11000] = low
    return c


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("value", [None, -1e30, -1e20, -1e9])
def test_finite_masks(gpu, bf16, draft, value):
    masked(31, bf16, draft, value, [1.0, 0.8, 0.7, 0.6, 0.5, 1.3]).check()


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("draft", [False, True])
def test_rows_of_the_lowest_number_alone(gpu, bf16, draft):
    """All tokens alike, whatever the number: p is flat."""
    c = masked(32, bf16, draft, None, [1.0, 0.8, 0.7, 0.6, 0.5, 0.0])
    c.logits[:, :c.n] = c.logits[0, 2000]
    c.check()


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("value", [1e9, 1e30, 3e38])
def test_forced_tokens(gpu, bf16, value):
    """One token of a large finite logit has all of the mass, two share it."""
    for draft in (False, True):
        c = Case(33, [2, 3, 4, 1], 9001, bf16=bf16, draft=draft, heat=[1.0, 0.7, 1.9, 0.6])
        big = enc(np.float32([value]), bf16)[0]
        c.logits[:, 7000] = big
        c.logits[5:, 11] = big
        if draft:
            c.draft[3, 7000] = big
        got = c.check()
        assert (got[1, :2] == 7000).all() and np.isin(got[1], (11, 7000)).all()


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("heat", [1e-3, 1e-6, 1e-10, 1e-18, 1e-20, 1e-30, 1e-38])
def test_tiny_temperatures(gpu, bf16, heat):
    """As near to the likeliest token as the formula has it; equal logits share the mass at any temperature."""
    for draft in (False, True):
        c = Case(34, [3, 4, 1, 2], 5000, bf16=bf16, draft=draft, heat=[heat, 1.7 * heat, heat, 3.1 * heat])
        c.logits[5:, 123] = c.logits[5:, 4321] = enc(np.float32([30.0]), bf16)[0]
        c.check()
