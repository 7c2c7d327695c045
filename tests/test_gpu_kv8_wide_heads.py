"""Attention over the 8-bit cache with heads of 144 and 192 dims, whose lanes take 12
codes of a row each: the last row of the pools is the last slot, the last head's codes
their last bytes, and many splits are joined.  Bars as of test_gpu_kv8_attend.py."""
import numpy as np
import pytest

from ouroboros_amd.device import DeviceBuffer

from test_gpu_kv8_attend import U, check, plain
from test_gpu_kv8_cache import Cache8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [144, 192])
@pytest.mark.parametrize("layout", ["token", "head"])
@pytest.mark.parametrize("count,hq", [(1, 4), (9, 4)])
def test_last_row_of_the_pools(gpu, d, layout, count, hq):
    n, page = 64, 16
    t = Cache8(d, 1, n, 2, d, page, 16, layout, spare=0)
    t.table[0] = [2, 0, 1, 3]  # the last page is the last slots'
    t.fill([n])
    q = t.rng.standard_normal((count, hq, d)).astype(np.float32)
    out = DeviceBuffer((count, hq, d), np.float32)
    t.open().attend(DeviceBuffer.from_host(q), out, DeviceBuffer.from_host(np.array([n], np.int32)), 1, count, count, n, hq)
    k, v, _ = t.values(0, 0, n)
    for i in range(count):
        seen = np.arange(n) <= n - count + i
        o, _, size, spread = plain(q[i].astype(np.float64), k, v, seen, d ** -0.5)
        bar = (16 * U * size[:, None] + 600 * U) * spread + n * 2.0 ** -39 * np.abs(v[seen]).max()
        assert (np.abs(out.download()[i] - o) <= bar).all()


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("d", [144, 192])
def test_many_splits(gpu, bf16, d):
    """Two splits, up to sixteen, and more: the forms of the join, of which 192 dims leave threads without work."""
    for n in (1500, 9000, 30000):
        check(d, (n, 700), (1, 1), 4, 2, d, 256, 64, bf16=bf16, gate=True)
        check(d + 1, (n, 700), (5, 3), 4, 1, d, 256, 256, bf16=bf16)
