"""Attention over the 8-bit cache with scores so large that the softmax is one slot's,
and past fp32.

Large: keys are 0 but for the first dim of one slot, of two equal ones, or of one of the
other sign, so that a score is X there and 0 elsewhere.  The weight of the largest is 1
but for some e^-X, so that its value comes out within 600 U |v| + n 2^-39 max |v|, as
test_gpu_kv8_attend.py derives it, and lse is X within 8 U X + 600 U + 2 U X.

Past fp32: a score of +inf makes out and lse NaN, one of -inf weighs nothing."""
import numpy as np
import pytest

from ouroboros_amd.device import DeviceBuffer

from test_gpu_kv8_attend import U
from test_gpu_kv8_cache import Cache8, dec, enc, name

pytestmark = pytest.mark.gpu
# one split of a sequence, several, and the kernel for many rows of a kv head (one split, several)
FORMS = [(200, 1, 4, 1), (3000, 2, 4, 1), (3000, 5, 8, 1), (700, 80, 8, 2), (6000, 150, 4, 2)]


def run(n, count, hq, hkv, d, bf16, size, codes, ks=1.0, scale=None, seed=0):
    """(out, lse, v [n][hkv][d]): keys codes[slot] * ks in dim 0, queries `size` there and small elsewhere."""
    t = Cache8(seed, 1, n, hkv, d, 64, 32)
    t.fill([n])
    for j in range(n):
        p, tok = t.at(0, j)
        k = t.view(t.codes[0])[p, tok]
        k[:] = 0
        k[:, 0] = codes[j]
        t.scales[0][p, tok // 32] = ks
    q = 0.5 * t.rng.standard_normal((count, hq, d))
    q[..., 0] = size
    q = enc(q, bf16)
    out, lse = DeviceBuffer((count, hq, d), q.dtype), DeviceBuffer((count, hq), np.float32)
    t.open().attend(DeviceBuffer.from_host(q), out, DeviceBuffer.from_host(np.array([n], np.int32)), 1, count, count, n, hq, dtype=name(bf16),
                    lse=lse, scale=scale)
    return dec(out.download()), lse.download().astype(np.float64), t.values(0, 0, n)[1], float(dec(q)[0, 0, 0])


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("n,count,hq,hkv", FORMS)
@pytest.mark.parametrize("d", [64, 192])
@pytest.mark.parametrize("exponent", [4, 13, 17, 19, 20, 22, 24, 27, 33, 50, 90, 118])
def test_one_slot_has_all(gpu, bf16, n, count, hq, hkv, d, exponent):
    """The largest score from some hundred to 2^125, of an odd multiple so that its product rounds."""
    codes = np.zeros(n, np.int64)
    at = n - count - 7  # seen by every row
    codes[at] = 127
    codes[3] = -127
    X = 1.2345 * 2.0 ** exponent
    out, lse, v, x = run(n, count, hq, hkv, d, bf16, X, codes, scale=0.9173)
    s = float(np.float32(0.9173)) * x * 127
    G = hq // hkv
    want = np.stack([v[at, h // G] for h in range(hq)])[None]
    bar = 600 * U * np.abs(want) + n * 2.0 ** -39 * np.abs(v).max() + (2.0 ** -8 * np.abs(want) if bf16 else 0)
    assert (np.abs(out - want) <= bar).all()
    assert (np.abs(lse - s) <= 8 * U * s + 600 * U + 2 * U * s).all()


@pytest.mark.parametrize("n,count,hq,hkv", FORMS)
def test_two_slots_share(gpu, n, count, hq, hkv):
    """Equal large scores in two tiles, of a negative scale too."""
    for scale in (0.7, -0.7):
        codes = np.zeros(n, np.int64)
        at = 10, n - count - 1
        codes[list(at)] = 127 if scale > 0 else -127
        out, lse, v, x = run(n, count, hq, hkv, 64, False, 1.7 * 2.0 ** 40, codes, scale=scale)
        s = abs(float(np.float32(scale)) * x * 127)
        G = hq // hkv
        pair = np.stack([v[list(at), h // G] for h in range(hq)], 1)  # [2][hq][d]
        bar = 600 * U * np.abs(pair).mean(0) + n * 2.0 ** -39 * np.abs(v).max()
        assert (np.abs(out - pair.mean(0)) <= bar).all()
        assert (np.abs(lse - s) <= 10 * U * s + 600 * U).all()


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("n,count,hq,hkv", FORMS)
def test_scores_past_fp32(gpu, bf16, n, count, hq, hkv):
    """Queries of 1e38 over keys of some hundred: NaN and NaN, in every form; against keys of the other sign -inf, which weighs nothing."""
    codes = np.zeros(n, np.int64)
    codes[n - count - 7] = 100
    out, lse, _, _ = run(n, count, hq, hkv, 64, bf16, 1e38, codes, ks=4.0, scale=1.0)
    assert np.isnan(out).all() and np.isnan(lse).all()
    codes[:] = -100
    codes[[5, 77]] = 0
    out, lse, v, _ = run(n, count, hq, hkv, 64, bf16, 1e38, codes, ks=4.0, scale=1.0)
    G = hq // hkv
    want = np.stack([v[[5, 77], h // G].mean(0) for h in range(hq)])
    bar = 600 * U * np.stack([np.abs(v[[5, 77], h // G]).mean(0) for h in range(hq)]) + n * 2.0 ** -39 * np.abs(v).max()
    assert (np.abs(out - want) <= bar + (2.0 ** -8 * np.abs(want) if bf16 else 0)).all()
    assert (np.abs(lse - np.log(2)) <= 600 * U).all()
    codes[:] = -100
    out, lse, _, _ = run(n, count, hq, hkv, 64, bf16, 1e38, codes, ks=4.0, scale=1.0)
    assert not out.any() and np.isneginf(lse).all()
