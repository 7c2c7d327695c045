"""Log probabilities of given tokens (ouro_token_logprobs) against float64.

U = 2^-24.  x - m is rounded once, so e^(x - m) is off by at most |x - m| U of
itself and exp's own error, 4 U; the sum over a row runs in chains and trees of
at most C = ceil(n / 256) + 24 roundings.  With D the mean of |x - m| under the
softmax, l is within (C + 4 + D) U of itself, so lse and a logprob are within
(C + 8 + D) U + 2 U (|m| + |x_t - m| + |lse|); the entropy subtracts a mean of
|x - m| with the same relative error, plus the spread of |x - m| under e^-|x-m|:
(C + 8 + D) U (1 + 2 D) + 4 U (entropy + D) + U mean (x - m)^2.
Ids and ranks are compared as they are: ties are broken by the index."""
import numpy as np
import pytest

from ouroboros_amd import ops
from ouroboros_amd._lib import OuroError
from ouroboros_amd.device import DeviceBuffer, Stream
from ouroboros_amd.quant import bf16_bits_to_f32, f32_to_bf16_bits

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def check(x, targets, k, *, bf16=False, stride=0, stream=None, offset=0):
    """x [rows, n] as float32; runs on device buffers, rows `stride` apart."""
    rows, n = x.shape
    raw = f32_to_bf16_bits(x) if bf16 else x.astype(np.float32)
    x = bf16_bits_to_f32(raw) if bf16 else raw
    wide = np.full((rows, max(stride, n)), 0x7f80 if bf16 else np.inf, raw.dtype)  # the gap: +inf
    wide[:, :n] = raw
    flat = np.concatenate([np.zeros(offset, raw.dtype), wide.reshape(-1)])
    xb = DeviceBuffer.from_host(flat)
    tb = DeviceBuffer.from_host(np.asarray(targets, np.int32))
    out = {"entropy": DeviceBuffer((rows,), np.float32), "lse": DeviceBuffer((rows,), np.float32),
           "logprob": DeviceBuffer((rows,), np.float32), "rank": DeviceBuffer((rows,), np.int32)}
    if k:
        out.update(top_id=DeviceBuffer((rows, k), np.int32), top_logprob=DeviceBuffer((rows, k), np.float32))
    ops.token_logprobs(xb.ptr + offset * raw.itemsize, rows, n, dtype="bf16" if bf16 else "f32", row_stride=stride, targets=tb, k=k,
                       stream=stream.handle if stream else None, **out)
    if stream:
        stream.synchronize()
    got = {a: b.download() for a, b in out.items()}
    X = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    C = -(-n // 256) + 24
    for r in range(rows):
        m = X[r].max()
        with np.errstate(invalid="ignore", divide="ignore"):
            diff = np.where(X[r] == m, 0.0, X[r] - m)
        order = np.lexsort((np.arange(n), -X[r]))
        rank = np.empty(n, np.int64)
        rank[order] = np.arange(n)
        t = int(targets[r])
        given = 0 <= t < n
        assert got["rank"][r] == (rank[t] if given else -1), r
        if k:
            ids = [int(i) if X[r, i] > -np.inf else -1 for i in order[:k]]
            assert got["top_id"][r].tolist() == ids + [-1] * (k - len(ids)), r
        if m == -np.inf:
            assert got["lse"][r] == -np.inf and got["entropy"][r] == 0
            assert got["logprob"][r] == (-np.inf if given else 0)
            assert k == 0 or (got["top_logprob"][r] == -np.inf).all()
            continue
        e = np.exp(diff)
        p = e / e.sum()
        seen = e > 0
        ln, D = np.log(e.sum()), (p[seen] * -diff[seen]).sum()
        sq = (p[seen] * diff[seen] ** 2).sum()
        base = (C + 8 + D) * U
        if np.isfinite(m):
            assert abs(got["lse"][r] - (m + ln)) <= base + 2 * U * (abs(m) + abs(m + ln)), r
        else:
            assert got["lse"][r] == np.inf
        H = ln + D
        assert abs(got["entropy"][r] - H) <= base * (1 + 2 * D) + 4 * U * (H + D) + U * sq, r

        def near(g, i):
            w = diff[i] - ln
            return g == -np.inf if w == -np.inf else abs(g - w) <= base + 2 * U * (abs(diff[i]) + abs(w))
        assert near(got["logprob"][r], t) if given else got["logprob"][r] == 0, r
        for i in range(k):
            j = got["top_id"][r, i]
            assert got["top_logprob"][r, i] == -np.inf if j < 0 else near(got["top_logprob"][r, i], j), (r, i)
    return got


def logits(seed, rows, n, scale=3.0):
    return (scale * np.random.default_rng(seed).standard_normal((rows, n))).astype(np.float32)


@pytest.mark.parametrize("n", [1, 2, 3, 63, 64, 65, 255, 257, 1000, 1023, 4097, 32003, 70001])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("k", [0, 1, 5, 64])
def test_sizes(gpu, n, bf16, k):
    x = logits(n, 3, n)
    check(x, [0, n - 1, n // 2], k, bf16=bf16)


@pytest.mark.parametrize("rows", [1, 2, 7, 130])
def test_vocabulary(gpu, rows):
    """The head of the decoder stack, from one row to more than half the CUs."""
    x = logits(rows, rows, 248320 if rows < 100 else 20693)
    check(x, np.random.default_rng(rows).integers(0, x.shape[1], rows), 20)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("stride,offset", [(0, 1), (1027, 0), (1027, 3), (1032, 8)])
def test_strides_and_alignment(gpu, bf16, stride, offset):
    check(logits(5, 9, 1025), [0, 1, 2, 3, 1024, 1023, 500, -1, 1025], 7, bf16=bf16, stride=stride, offset=offset)


@pytest.mark.parametrize("k", [1, 20, 64])
def test_ties(gpu, k):
    """Few distinct values: the lowest indices come first, across every split of the row."""
    rng = np.random.default_rng(k)
    x = rng.integers(-2, 3, (6, 30000)).astype(np.float32)
    x[1] = 0.0
    x[2, ::2] = -0.0
    x[2, 1::2] = 0.0
    x[3] = 1.0
    x[3, 29990:] = 2.0
    x[4] = -5.0
    x[4, ::997] = 7.0
    check(x, [29999, 15000, 3, 29995, 997, 0], k)


@pytest.mark.parametrize("n", [10, 3000, 70000])
def test_masked_infinite_and_nan(gpu, n):
    rng = np.random.default_rng(n)
    x = logits(n, 9, n)
    x[0, rng.random(n) < 0.9] = -np.inf          # most tokens ruled out
    x[1] = -np.inf                                # all of them
    x[2] = -np.inf
    x[2, n // 2] = -3.0                           # all but one
    x[3, rng.random(n) < 0.5] = np.nan
    x[4] = np.nan
    x[5, n - 1] = np.inf                          # one takes all
    x[6, [0, n // 3, n - 1]] = np.inf             # three share
    x[7] = np.finfo(np.float32).min               # a mask of the type's lowest value, everywhere
    x[8, : n - 2] = np.finfo(np.float32).min      # and on all but two
    t = [n // 4, 5, n // 2, int(np.flatnonzero(np.isnan(x[3]))[0]), 1, n - 1, 2, n - 1, n - 2]
    check(x, t, 12)
    check(x, t, 12, bf16=True)
    check(x[[5, 6]], [3, n - 1], 2)


def test_far_logits(gpu):
    """e^x alone would pass fp32's range, and almost all of the mass underflows."""
    x = logits(1, 4, 5000, 200.0)
    x[1] += 3e4
    x[2] = -np.arange(5000, dtype=np.float32) * 20
    x[3] = 0.0
    check(x, [0, 1, 2, 3], 10)


def test_numpy_and_partial_outputs(gpu):
    x = logits(2, 5, 777)
    got = ops.token_logprobs(x, 5, 777, targets=[1, 2, 3, 4, 5], k=3)
    want = check(x, [1, 2, 3, 4, 5], 3)
    for name in want:
        assert np.array_equal(got[name], want[name]), name
    assert set(ops.token_logprobs(x, 5, 777)) == {"entropy", "lse"}
    half = ops.token_logprobs(f32_to_bf16_bits(x), 5, 777, k=2)
    assert half["top_id"].shape == (5, 2)
    xb, lse = DeviceBuffer.from_host(x), DeviceBuffer((5,), np.float32)
    ops.token_logprobs(xb, 5, 777, lse=lse)
    assert np.array_equal(lse.download(), want["lse"])
    ops.token_logprobs(xb, 5, 777)  # nothing asked for


def test_row_alone_and_in_any_batch(gpu):
    """A row's bits do not depend on the rows beside it."""
    x = logits(8, 40, 50000)
    t = np.arange(40) * 7
    whole = check(x, t, 8)
    for r in (0, 17, 39):
        one = check(x[r:r + 1], t[r:r + 1], 8)
        assert all(np.array_equal(one[name][0], whole[name][r]) for name in whole), r


def test_streams(gpu):
    s = [Stream(), Stream()]
    for _ in range(2):
        for i in range(2):
            check(logits(20 + i, 3, 60000), [1, 2, 3], 5, stream=s[i])


@pytest.mark.parametrize("code,more", [
    (2, dict(n=0)), (2, dict(n=1 << 24)), (2, dict(row_stride=99)), (2, dict(k=65)), (1, dict(k=1)), (1, dict(logits=None)),
    (1, dict(logprob=True)), (1, dict(rank=True)), (3, dict(logits="odd")),
])
def test_refusals(gpu, code, more):
    x, o = DeviceBuffer((2, 100), np.float32), DeviceBuffer((2, 64), np.float32)
    a = dict(logits=x, rows=2, n=100)
    a.update({key: o if v is True else x.ptr + 2 if v == "odd" else v for key, v in more.items()})
    with pytest.raises(OuroError) as e:
        ops.token_logprobs(**a)
    assert e.value.code == code and "ouro_token_logprobs" in str(e.value)
    with pytest.raises(ValueError):
        ops.token_logprobs(x, 2, 100, dtype="f16")


def test_no_rows(gpu):
    ops.token_logprobs(DeviceBuffer((1,), np.float32), 0, 100)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("n", [8178, 8186, 8191, 8193, 16390, 24577, 32754, 32762, 32767, 32769])
def test_rows_of_few_parts(gpu, n, bf16):
    """Without alternatives, around the lengths at which a row takes one, two .. five parts."""
    rng = np.random.default_rng(n)
    x = logits(n, 6, n)
    x[0, rng.random(n) < 0.9] = -np.inf
    x[1] = -np.inf
    x[2, n - 1] = np.inf
    x[3, rng.random(n) < 0.5] = np.nan
    x[4] = np.finfo(np.float32).min
    t = [n // 3, 0, n - 1, n - 2, 5, n // 2]
    check(x, t, 0, bf16=bf16)
    check(x, t, 0, bf16=bf16, offset=3, stride=n + 2)
    check(x[5:], [n - 1], 0, bf16=bf16)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("n", [9000, 32000])
def test_few_rows_and_many(gpu, n, bf16):
    """A row's bits are those of a call of few rows, of many and with alternatives."""
    x = logits(n, 8, n)
    raw = f32_to_bf16_bits(x) if bf16 else x
    t = np.arange(8) * 11
    got = [ops.token_logprobs(np.tile(raw, (m, 1)), 8 * m, n, targets=np.tile(t, m).astype(np.int32), k=k) for m, k in ((1, 0), (64, 0), (65, 0), (1, 3))]
    for other in got[1:]:
        for name in ("logprob", "rank", "entropy", "lse"):
            assert np.array_equal(other[name][-8:], got[0][name]), name
