"""Attention over a paged cache (ouro_kv_attend) with NaN and infinities where
they count: in queries and in visible rows.  The formula in IEEE arithmetic
holds: a NaN score, or one of +inf, makes its head NaN; a score of -inf weighs
nothing; a value that is not finite makes its own dimension what the sum of
p v is, and no other.  Rows of a bf16 cache and of an fp32 cache alike, whatever
the queries' type, and no slot that is not visible is touched by any of it.

What is finite is held to the bars of test_gpu_kv_cache.py."""
import numpy as np
import pytest

from ouroboros_amd.device import DeviceBuffer
from ouroboros_amd.kvcache import History

from test_gpu_kv_cache import U, Setup, dec, enc, name

pytestmark = pytest.mark.gpu
TYPES = [(True, False), (True, True), (False, False), (False, True)]  # (bf16 cache, bf16 rows)
HKV, G, D, PAGE = 2, 3, 72, 16
LENS = [(40,), (700, 33)]  # one split, and several


class Call:
    """Rows that a test changes before check(); slot 5 is masked, slots 16 .. 31 of sequence 0 are a hole."""

    def __init__(self, lens, cache, io, seed=0):
        self.io, self.cache, self.lens = io, cache, lens
        self.t = Setup(seed + len(lens), lens, HKV, D, PAGE, cache, holes=[(0, 1, -1)] if lens[0] > PAGE else ())
        self.q = self.t.rng.standard_normal((len(lens), HKV * G, D)).astype(np.float32)
        self.mask = np.ones((len(lens), self.t.max_len), np.uint8)
        self.mask[:, 5:6] = 0

    def row(self, pool, b, slot):
        return self.t.view(pool)[self.t.table[b, slot // PAGE], slot % PAGE]

    def put(self, pool, b, slot, head, dim, x):
        self.row(pool, b, slot)[head, dim] = enc(np.full(1, x, np.float32), self.cache)[0]

    def check(self, scale=None):
        t, B, H, L = self.t, len(self.lens), HKV * G, self.t.max_len
        c = t.open()
        q = enc(self.q, self.io)
        w0 = t.rng.uniform(0, 4, (B, HKV, L)).astype(np.float32)
        wb, pb = DeviceBuffer.from_host(w0), DeviceBuffer((B, HKV, L), np.int32, zero=True)
        out = DeviceBuffer.from_host(enc(np.full((B, H, D), 77.0), self.io))
        lse, lens = DeviceBuffer.from_host(np.full((B, H), 77.0, np.float32)), DeviceBuffer.from_host(t.lens)
        c.attend(DeviceBuffer.from_host(q), out, lens, B, L, H, dtype=name(self.io), lse=lse, scale=scale,
                 mask=DeviceBuffer.from_host(self.mask), history=History(wb, pb, HKV, L))
        got, lse, w = dec(out.download()).astype(np.float64), lse.download(), wb.download()
        for b in range(B):
            j, k, v = t.rows(b)
            live = self.mask[b, j] != 0
            j, k, v = j[live], k[live], v[live]
            hidden = np.setdiff1d(np.arange(L), j)
            assert np.array_equal(w[b][:, hidden], w0[b][:, hidden])
            want_w, bar_w = w0[b][:, j].astype(np.float64), U * w0[b][:, j]
            for h in range(H):
                with np.errstate(all="ignore"):
                    qv, sc = dec(q[b, h]).astype(np.float64), D ** -0.5 if scale is None else scale
                    s = sc * (k[:, h // G] * qv).sum(1)
                    S = np.abs(sc * (np.abs(k[:, h // G]) * np.abs(qv))).sum(1)
                    S = S[np.isfinite(S)].max(initial=0.0)
                    if (s == -np.inf).all():
                        assert (got[b, h] == 0).all() and lse[b, h] == -np.inf, (b, h)
                        continue
                    e = np.exp(s - s.max())
                    p = e / e.sum()
                    o = (p[:, None] * v[:, h // G]).sum(0)
                    size = (p[:, None] * np.abs(v[:, h // G])).sum(0)
                bar = 2 * 68 * U * S + 600 * U
                if np.isnan(p).any():
                    assert np.isnan(got[b, h]).all() and np.isnan(lse[b, h]), (b, h, got[b, h, 0], lse[b, h])
                    # every slot whose score is not -inf takes the NaN
                    want_w[h // G, s != -np.inf] = np.nan
                    continue
                w_lse = s.max() + np.log(e.sum())
                assert abs(lse[b, h] - w_lse) <= 68 * U * S + 600 * U + 2 * U * abs(w_lse), (b, h)
                fine = np.isfinite(o)
                assert np.array_equal(got[b, h][~fine], o[~fine], equal_nan=True), (b, h)
                room = bar * size[fine] + (2.0 ** -8 * np.abs(o[fine]) if self.io else 0)
                assert (np.abs(got[b, h][fine] - o[fine]) <= room).all(), (b, h)
                want_w[h // G] += p
                bar_w[h // G] += (bar + 4 * U) * p + U * want_w[h // G]
            nan = np.isnan(want_w)
            assert np.array_equal(np.isnan(w[b][:, j]), nan)
            assert (np.abs(w[b][:, j] - want_w)[~nan] <= bar_w[~nan]).all()
        return got


def each(f):
    f = pytest.mark.parametrize("lens", LENS, ids=str)(f)
    return pytest.mark.parametrize("cache,io", TYPES)(f)


@each
def test_nan_query(gpu, lens, cache, io):
    """A head whose query holds a NaN is NaN, its neighbours are not."""
    c = Call(lens, cache, io)
    c.q[0, 1, 7] = np.nan
    c.q[-1, 5] = np.nan
    c.check()


@each
def test_nan_key(gpu, lens, cache, io):
    """A visible key that holds a NaN makes its kv head NaN."""
    c = Call(lens, cache, io)
    c.put(c.t.k, 0, 9, 1, 70, np.nan)
    c.check()
    c = Call(lens, cache, io)
    c.put(c.t.k, 0, lens[0] - 1, 0, 0, np.nan)  # the last split's last slot
    c.check()


@pytest.mark.parametrize("cache,io", TYPES)
def test_lone_nan_key(gpu, cache, io):
    """The only visible slot, and the only one of its split."""
    c = Call((1,), cache, io)
    c.put(c.t.k, 0, 0, 0, 3, np.nan)
    c.check()
    c = Call((600,), cache, io)
    c.mask[0, 256:512] = 0
    c.mask[0, 300] = 1
    c.put(c.t.k, 0, 300, 1, 3, np.nan)
    c.check()


@each
def test_keys_of_minus_infinity(gpu, lens, cache, io):
    """A visible key that scores -inf weighs nothing, for queries that bf16 holds and others."""
    for whole in (False, True):
        c = Call(lens, cache, io)
        c.q[..., 11] = np.abs(c.q[..., 11]) + np.float32(0.1)
        if whole:
            c.q = dec(enc(c.q, True))
        c.put(c.t.k, 0, 3, 0, 11, -np.inf)
        c.put(c.t.k, 0, 35, 1, 11, -np.inf)
        c.check()


@each
def test_keys_of_infinity(gpu, lens, cache, io):
    """Queries of either sign: a head's score is -inf or +inf, whose softmax is NaN; 0 times infinity is NaN."""
    c = Call(lens, cache, io)
    c.put(c.t.k, 0, 3, 0, 11, np.inf)
    c.q[0, 0, 11] = 0
    c.q[0, 1, 11] = -0.7
    c.q[0, 2, 11] = 0.7
    c.check()


@pytest.mark.parametrize("cache,io", TYPES)
def test_all_scores_minus_infinity(gpu, cache, io):
    """No score above -inf: as where no slot is visible."""
    c = Call((40,), cache, io)
    c.q[..., 11] = np.abs(c.q[..., 11]) + np.float32(0.1)
    for j in range(40):
        if j // PAGE != 1:
            c.put(c.t.k, 0, j, 0, 11, -np.inf)
    c.check()


@each
def test_infinite_and_nan_values(gpu, lens, cache, io):
    """A value that is not finite decides its own dimension: inf, -inf, NaN, and inf beside -inf."""
    c = Call(lens, cache, io)
    for slot, dim, x in ((3, 0, np.inf), (35, 1, -np.inf), (36, 2, np.nan), (3, 71, np.inf), (37, 71, -np.inf), (38, 40, np.inf), (39, 40, np.inf)):
        c.put(c.t.v, 0, slot, 1, dim, x)
    got = c.check()
    assert got[0, G, 0] == np.inf and got[0, G, 1] == -np.inf and np.isnan(got[0, G, [2, 71]]).all() and got[0, G, 40] == np.inf


@pytest.mark.parametrize("cache,io", TYPES)
def test_infinite_value_alone(gpu, cache, io):
    """Weight 1 exactly: nothing is left for a weight's lower parts."""
    c = Call((1,), cache, io)
    c.put(c.t.v, 0, 0, 0, 3, -np.inf)
    c.put(c.t.v, 0, 0, 1, 4, np.nan)
    c.check()


@pytest.mark.parametrize("cache", [True, False])
def test_infinite_and_largest_queries(gpu, cache):
    """An infinite query has scores of +inf and -inf; the type's largest one is a number like others."""
    c = Call((300,), cache, False)
    c.q[0, 0, 5] = np.inf
    c.q[0, 4, 6] = -np.inf
    c.check()
    c = Call((300,), cache, False)
    c.q[0, 1, 5] = np.finfo(np.float32).max
    c.q[0, 3, 6] = -np.finfo(np.float32).max
    for j in range(300):
        if j // PAGE != 1:
            for dim in (5, 6):
                for head in range(HKV):
                    c.put(c.t.k, 0, j, head, dim, c.t.rng.integers(-3, 4) * 2.0 ** -125)
    c.check()
