"""Attention over the 8-bit cache where blocks' scales are far apart.

A block that a row does not see changes none of its bits, whatever other rows of the
call see of it.  What a row sees is held to test_gpu_kv8_attend.py's bar with its last
term by what counts: a weight times its scale is held to half of 2^-24 at a power of two
that takes 2^8 times the largest of them to 2^15 at most, and to 2^14 at least, so to
2^-25 2^-14 2^8 = 2^-31 of the largest; one below 2^-112 may be held to less than it is (its scale times the
row's power of two is no more than 2^127, where weights come to 2^15 at most), so that n
slots of |v| <= 128 scale add n 2^-24 max p scale + n 2^-112 max |v|; outputs are rounded
to 2^-149 at least."""
import numpy as np
import pytest

from ouroboros_amd.device import DeviceBuffer

from test_gpu_kv8_attend import U, plain
from test_gpu_kv8_cache import Cache8, dec, enc, name

pytestmark = pytest.mark.gpu
# slots, new rows, query heads, kv heads: 16 rows of a kv head at most, 32 a workgroup, the kernel for many rows; one split and several
FORMS = [(197, 8, 2, 1), (3013, 7, 4, 2), (213, 22, 4, 1), (3013, 30, 8, 1), (709, 70, 8, 1), (5013, 90, 8, 2)]


def attend(t, q, n, bf16=False, **more):
    count, hq = q.shape[:2]
    out, lse = DeviceBuffer(q.shape, q.dtype), DeviceBuffer((count, hq), np.float32)
    t.open().attend(DeviceBuffer.from_host(q), out, DeviceBuffer.from_host(np.array([n], np.int32)), 1, count, count, n, hq, dtype=name(bf16),
                    lse=lse, **more)
    return dec(out.download()), lse.download().astype(np.float64)


def put(t, j, which, scale):
    p, tok = t.at(0, j)
    t.scales[which][p, tok // t.block] = scale


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("n,count,hq,hkv", FORMS)
def test_blocks_out_of_a_rows_sight(gpu, bf16, d, n, count, hq, hkv):
    """The last block, which only the last rows see; with a window the first one of the first row's sight too."""
    t = Cache8(d + n, 1, n, hkv, d, 64, 16)
    t.fill([n])
    q = enc(t.rng.standard_normal((count, hq, d)), bf16)
    at = n - count + np.arange(count)
    window = next(w for w in range(40, 80) if (at[0] - w + 1) % 16 == 13)  # three slots of that block
    for more, block in ((dict(), n // 16), (dict(window=window, sinks=2), n // 16), (dict(window=window), (at[0] - window + 1) // 16)):
        sees = at >= 16 * block
        if more:
            sees &= at - 16 * block - 15 < window
        assert sees.any() and not sees.all()
        got = []
        for which, scale in ((1, 2.0 ** -6), (1, 2.0 ** 25), (1, 3.7e9), (1, 2.0 ** 45), (1, 2.0 ** 110), (0, 2.0 ** 70), (0, 1e30)):
            put(t, 16 * block, which, scale)
            got.append(attend(t, q, n, bf16, **more))
            put(t, 16 * block, which, 2.0 ** -6)
        for o, l in got[1:]:
            assert np.array_equal(o[~sees], got[0][0][~sees]) and np.array_equal(l[~sees], got[0][1][~sees])
        assert not np.array_equal(got[3][0][sees], got[0][0][sees])


@pytest.mark.parametrize("n,count,hq,hkv", FORMS)
@pytest.mark.parametrize("far", [0, 5, 20, 45, 70])
def test_large_scales_of_little_weight(gpu, n, count, hq, hkv, far):
    """A block of scale 2^far 2^10 whose keys score some far ln 2 below the others', first, in the middle and last."""
    d = 64
    for where in (0, n // 2 // 16, (n - count) // 16 - 1):
        t = Cache8(n + far, 1, n, hkv, d, 64, 16)
        t.fill([n])
        for j in range(0, n, 16):
            put(t, j, 0, 2.0 ** -8)
            put(t, j, 1, 2.0 ** -7)
            p, tok = t.at(0, j)
            t.view(t.codes[0])[p, tok:tok + 16, :, 0] = 0
        put(t, 16 * where, 0, 2.0 ** -4)
        put(t, 16 * where, 1, 2.0 ** (far + 3))
        p, tok = t.at(0, 16 * where)
        t.view(t.codes[0])[p, tok:tok + 16] = 0
        t.view(t.codes[0])[p, tok:tok + 16, :, 0] = -100
        q = t.rng.standard_normal((count, hq, d)).astype(np.float32)
        q[..., 0] = far * np.log(2) / (100 * 2.0 ** -4 * 0.125)
        out, lse = attend(t, q, n)
        k, v, _ = t.values(0, 0, n)
        scales = np.array([t.scales[1][t.at(0, j)[0], t.at(0, j)[1] // 16] for j in range(n)], np.float64)  # [n][hkv]
        for i in range(count):
            seen = np.arange(n) <= n - count + i
            o, l, size, spread = plain(q[i].astype(np.float64), k, v, seen, 0.125, count * (hq // hkv) > 256)
            ds = 8 * U * size
            for h in range(hq):
                g = h // (hq // hkv)
                s = 0.125 * (k[seen, g] @ q[i, h].astype(np.float64))
                most = (np.exp(s - l[h]) * scales[seen, g]).max()
                bar = (2 * ds[h] + 600 * U) * spread[h] + n * (2.0 ** -24 * most + 2.0 ** -112 * np.abs(v[seen, g]).max())
                assert (np.abs(out[i, h] - o[h]) <= bar).all(), (where, i, h)
                assert abs(lse[i, h] - l[h]) <= ds[h] + 600 * U + 2 * U * abs(l[h])


@pytest.mark.parametrize("n,count,hq,hkv", FORMS)
def test_scales_at_both_ends(gpu, n, count, hq, hkv):
    """V's scales of 2^-126 where the weight is, and one block of 2^100 whose weights are 0: it leaves nothing, not a NaN."""
    t = Cache8(n, 1, n, hkv, 64, 64, 16)
    t.fill([n])
    where = 16 * (n // 3 // 16)
    for j in range(0, n, 16):
        put(t, j, 0, 2.0 ** -8)
        put(t, j, 1, 2.0 ** 100 if j == where else 2.0 ** -126)
        p, tok = t.at(0, j)
        t.view(t.codes[0])[p, tok:tok + 16, :, 0] = -100 if j == where else 0
    q = (0.1 * t.rng.standard_normal((count, hq, 64))).astype(np.float32)
    q[..., 0] = 4000  # scores of -195 there: e^-195 < 2^-126
    out, _ = attend(t, q, n, scale=0.125)
    k, v, _ = t.values(0, 0, n)
    for i in range(count):
        seen = np.arange(n) <= n - count + i
        seen[where:where + 16] = False
        o, _, size, spread = plain(q[i].astype(np.float64), k, v, seen, 0.125, count * (hq // hkv) > 256)
        bar = (16 * U * size[:, None] + 600 * U) * spread + n * 2.0 ** (-126 - 24) + 2.0 ** -148
        assert (np.abs(out[i] - o) <= bar).all()


@pytest.mark.parametrize("n,count,hq,hkv", FORMS)
@pytest.mark.parametrize("exponent", [-126, -121, -112])
def test_tiny_values(gpu, n, count, hq, hkv, exponent):
    """V's scales at the ends of fp32, weights flat."""
    t = Cache8(n - exponent, 1, n, hkv, 64, 64, 16)
    t.fill([n])
    for j in range(0, n, 16):
        put(t, j, 1, 2.0 ** exponent)
    q = (0.1 * t.rng.standard_normal((count, hq, 64))).astype(np.float32)
    out, _ = attend(t, q, n)
    k, v, _ = t.values(0, 0, n)
    for i in range(count):
        o, _, size, spread = plain(q[i].astype(np.float64), k, v, np.arange(n) <= n - count + i, 0.125, count * (hq // hkv) > 256)
        bar = (16 * U * size[:, None] + 600 * U) * spread + n * 2.0 ** (exponent - 24) / n + 2.0 ** -148
        assert (np.abs(out[i] - o) <= bar).all(), float((np.abs(out[i] - o) / bar).max())
