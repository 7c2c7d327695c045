"""Eviction (ouro_kv_evict) without slot_from, and with a budget far above every
length: its work and its scratch go by the slots in use, not by the budget."""
import numpy as np
import pytest

from ouroboros_amd.device import DeviceBuffer
from ouroboros_amd.kvcache import History

from test_gpu_kv_cache import Setup

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("apart", [False, True])
def test_budget_far_above_every_length(gpu, apart):
    """2^30 slots a head for 64 sequences of 4 heads: a terabyte, were any of it asked for."""
    B, H, n = 64, 4, 40
    lens = [1 + i % n for i in range(B)]
    lens[7] = n
    t = Setup(3, lens, H, 16, 16, True)
    w, pos = t.rng.random((B, H, n)).astype(np.float32), t.rng.integers(0, 99, (B, H, n)).astype(np.int32)
    hist = History(DeviceBuffer.from_host(w), DeviceBuffer.from_host(pos), H, n)
    out = History(DeviceBuffer((B, H, n), np.float32, zero=True), DeviceBuffer((B, H, n), np.int32, zero=True), H, n) if apart else None
    c, left = t.open(), DeviceBuffer((B,), np.int32)
    c.evict(hist, DeviceBuffer.from_host(t.lens), B, n, 1 << 30, 8, left, out=out)
    assert np.array_equal(left.download(), t.lens)
    assert np.array_equal(hist.weight.download(), w) and np.array_equal(hist.pos.download(), pos)
    assert np.array_equal(t.kb.download(), t.k) and np.array_equal(t.vb.download(), t.v)
    if apart:
        live = np.arange(n) < t.lens[:, None, None]
        assert np.array_equal(out.weight.download(), np.where(live, w, 0)) and np.array_equal(out.pos.download(), np.where(live, pos, 0))


@pytest.mark.parametrize("lens,keep", [((300, 40, 0), 64), ((300, 299), 299), ((2000, 1500), 900), ((16385,), 3000)], ids=str)
@pytest.mark.parametrize("heads", [1, 2])
def test_without_slot_from(gpu, lens, keep, heads):
    """The same cache, history and lengths are left whether slot_from is asked for or not."""
    left = []
    for asked in (True, False):
        t = Setup(5, lens, 2, 16, 16, True)
        B, n = len(lens), t.max_len
        w = np.exp(t.rng.standard_normal((B, heads, n))).astype(np.float32)
        pos = np.broadcast_to(np.arange(n, dtype=np.int32), w.shape)
        hist = History(DeviceBuffer.from_host(w), DeviceBuffer.from_host(pos), heads, n)
        c, lens_out = t.open(), DeviceBuffer((B,), np.int32)
        c.evict(hist, DeviceBuffer.from_host(t.lens), B, n, keep, 20, lens_out, slot_from=DeviceBuffer((B, heads, keep), np.int32) if asked else None)
        left.append([b.download() for b in (lens_out, hist.weight, hist.pos, t.kb, t.vb)])
    for a, b in zip(*left):
        assert np.array_equal(a.view(np.uint8), b.view(np.uint8))
