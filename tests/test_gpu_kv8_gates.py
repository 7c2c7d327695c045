"""Attention over the 8-bit cache with gates that are not numbers: rows that see nothing
are 0 whatever their gate, others what the formula gives, and no row touches another."""
import numpy as np
import pytest

from ouroboros_amd.device import DeviceBuffer

from test_gpu_kv8_cache import Cache8, dec, enc, name

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("n,count,hq,hkv,d", [(200, 4, 4, 2, 64), (200, 12, 4, 1, 128), (3000, 4, 4, 2, 64), (3000, 90, 4, 1, 64), (200, 90, 4, 1, 128),
                                              (3000, 10, 4, 1, 192)])
def test_gates(gpu, bf16, n, count, hq, hkv, d):
    """Sequence 0 is all padding but for the last rows' own slots, sequence 1 sees all."""
    t = Cache8(n + d, 2, n, hkv, d, 64, 16)
    t.fill([n, n])
    mask = np.ones((2, n), np.uint8)
    mask[0, :n - 2] = 0  # all but the last two rows see nothing
    q = enc(t.rng.standard_normal((2 * count, hq, d)), bf16)
    gate = enc(t.rng.standard_normal((2 * count, hq, d)), bf16)
    spoilt = enc(dec(gate), bf16)
    odd = enc(np.float32([np.nan, np.inf, -np.inf]), bf16)
    spoilt[0, :, :3], spoilt[count, :, :3], spoilt[2 * count - 1, 1, 5:8] = odd, odd, odd
    got = []
    for g in (gate, spoilt):
        out, lse = DeviceBuffer((2 * count, hq, d), q.dtype), DeviceBuffer((2 * count, hq), np.float32)
        t.open().attend(DeviceBuffer.from_host(q), out, DeviceBuffer.from_host(np.array([n, n], np.int32)), 2, 2 * count, count, n, hq,
                        dtype=name(bf16), mask=DeviceBuffer.from_host(mask), gate=DeviceBuffer.from_host(g), lse=lse)
        got.append((dec(out.download()), lse.download()))
    (o, l), (p, k) = got
    assert np.array_equal(l, k) and np.isneginf(l[:count - 2]).all()
    assert not o[:count - 2].any() and not p[:count - 2].any() and not np.isnan(p[:count - 2]).any()
    changed = np.zeros(o.shape, bool)
    changed[count, :, :3], changed[2 * count - 1, 1, 5:8] = True, True
    assert np.array_equal(o[~changed], p[~changed])
    for row in (p[count, :, :3], p[2 * count - 1, 1, None, 5:8]):
        assert np.isnan(row[:, 0]).all() and (row[:, 1] != 0).all() and np.isfinite(row[:, 1]).all() and (row[:, 2] == 0).all()
