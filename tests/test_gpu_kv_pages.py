"""Pages that a caller gave up, and eviction (ouro_kv_evict), which asks for a
page under every slot in use: the table is closed up first, the sequence's last
whole page with its history taking the freed place.  Every slot that eviction
then reports as kept holds the key and value that slot_from names, bit for bit,
and attention over what is left sees exactly the slots kept."""
import numpy as np
import pytest

from ouroboros_amd.device import DeviceBuffer
from ouroboros_amd.kvcache import History

from test_gpu_kv_cache import U, Setup, dec

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cache", [True, False])
@pytest.mark.parametrize("heads", [1, 2])
@pytest.mark.parametrize("gone", [[1], [0, 2], [3, 8]], ids=str)
def test_pages_given_up(gpu, gone, heads, cache):
    hkv, d, page, n, keep, recent = 2, 64, 16, 160, 70, 8
    t = Setup(len(gone), (n,), hkv, d, page, cache)
    w = np.exp(2 * t.rng.standard_normal((1, heads, n))).astype(np.float32)
    pos = np.broadcast_to(np.arange(n, dtype=np.int32), w.shape).copy()
    # close the table up: the last whole page in use into each place, from the lowest on
    pages, used = t.table[0], n // page
    for g in gone:
        used -= 1
        if g < used:
            pages[g] = pages[used]
            for x in (w, pos):
                x[..., g * page:(g + 1) * page] = x[..., used * page:(used + 1) * page]
        pages[used] = -1
    n = used * page
    t.lens[0] = n
    c = t.open()
    before = [dec(t.view(p)[pages[:used]].reshape(n, hkv, d)).copy() for p in (t.k, t.v)]
    hist = History(DeviceBuffer.from_host(w), DeviceBuffer.from_host(pos), heads, w.shape[2])
    lens, left, src_b = DeviceBuffer.from_host(t.lens), DeviceBuffer((1,), np.int32), DeviceBuffer((1, heads, keep), np.int32)
    c.evict(hist, lens, 1, n, keep, recent, left, slot_from=src_b)
    src = src_b.download()[0]
    assert left.download()[0] == keep
    for h in range(hkv):
        s = src[h % heads]
        assert len(set(s.tolist())) == keep and s.min() >= 0 and s.max() < n
        new = pos[0, h % heads, :n] > pos[0, h % heads, :n].max() - recent
        order = sorted(range(n), key=lambda j: (not new[j], -w[0, h % heads, j], j))[:keep]
        assert sorted(s.tolist()) == sorted(order)
        for buf, was in zip((t.kb, t.vb), before):
            pool = buf.download()
            held = dec(t.view(pool)[pages[np.arange(keep) // page], np.arange(keep) % page])
            assert np.array_equal(held[:, h], was[s, h])
    q = t.rng.standard_normal((1, hkv, d)).astype(np.float32)
    out = DeviceBuffer((1, hkv, d), np.float32)
    c.attend(DeviceBuffer.from_host(q), out, left, 1, keep, hkv)
    for h in range(hkv):
        k, v = (x[src[h % heads], h].astype(np.float64) for x in before)
        z = k @ q[0, h] / 8.0
        p = np.exp(z - z.max())
        p /= p.sum()
        S = (np.abs(k) @ np.abs(q[0, h])).max() / 8.0
        assert (np.abs(out.download()[0, h] - p @ v) <= (136 * U * S + 600 * U) * (p @ np.abs(v))).all()
