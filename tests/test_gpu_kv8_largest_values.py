"""Attention over the 8-bit cache where values come near the largest fp32: an average of
them is one of fp32 too, in whatever splits its sums were made.  The bar of
test_gpu_kv8_value_scales.py."""
import numpy as np
import pytest

from test_gpu_kv8_attend import U, plain
from test_gpu_kv8_cache import Cache8
from test_gpu_kv8_value_scales import FORMS, attend, put

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,count,hq,hkv", [*FORMS, (20000, 1, 4, 2), (20000, 6, 8, 2)])
@pytest.mark.parametrize("exponent", [112, 118, 121])
def test_largest_values(gpu, n, count, hq, hkv, exponent):
    """Codes of 100 to 127 of either sign a dim, V's scales up to 2^121, weights flat: sums of n values are past fp32, averages are not."""
    t = Cache8(n + exponent, 1, n, hkv, 64, 64, 16)
    t.fill([n])
    sign = np.where(np.arange(64) % 3 == 0, -1, 1)
    for j in range(0, n, 16):
        p, tok = t.at(0, j)
        t.view(t.codes[1])[p, tok:tok + 16] = sign * t.rng.integers(100, 128, (16, hkv, 64))
        put(t, j, 1, 2.0 ** exponent)
    q = (0.1 * t.rng.standard_normal((count, hq, 64))).astype(np.float32)
    out, _ = attend(t, q, n)
    assert np.isfinite(out).all()
    k, v, _ = t.values(0, 0, n)
    for i in sorted({0, count // 2, count - 1}):
        o, _, size, spread = plain(q[i].astype(np.float64), k, v, np.arange(n) <= n - count + i, 0.125, count * (hq // hkv) > 256)
        bar = (16 * U * size[:, None] + 600 * U) * spread + 2.0 ** (exponent - 24)
        assert (np.abs(out[i] - o) <= bar).all(), float((np.abs(out[i] - o) / bar).max())
