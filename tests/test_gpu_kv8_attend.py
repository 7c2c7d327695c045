"""Attention over a cache of 8-bit codes (ouro_kv8_attend) against a plain float64
restatement.

Bars, U = 2^-24.  A query is held to 2 U of its row's largest magnitude, the sum
over the dims is exact, and putting it together and scaling it takes six roundings
of its size; so a score's error is at most ds = 8 U S, S = |scale| max |q| sum |k|
(the largest over the slots).  e^(s - m) and its sum move by that each; running
maxima, sums over the slots and exp itself add less than 600 U.  A weight against V
is held to 2^-22 of its size, which the 600 U cover, or to 2^-40 of the largest
weight times the largest scale, at most n 2^-39 max |v| over n slots.  So the output is within
(2 ds + 600 U) sum p |v| + n 2^-39 max |v|, lse within ds + 600 U + 2 U |lse|.  A
bf16 output adds its rounding, 2^-8 of its size, the gate 8 U.

Where a sequence has more than 256 rows of a kv head (and heads of up to 128 dims)
the queries are two fp16 operands, 2^-22 = 4 U of each value, and the sums over the
dims are made in fp32: 2 * 128 products at most, and six roundings more, so that
ds = (4 + 256 + 6) U |scale| sum |q k| there, the largest over the slots.

A slot left out, or counted twice, moves the output by its weight, at 1 / n on
average many times the bar at the lengths here."""
import numpy as np
import pytest

from ouroboros_amd._lib import OuroError
from ouroboros_amd.device import DeviceBuffer, Stream, synchronize
from ouroboros_amd.kvcache import KVCache8, attend8_workspace_bytes

from test_gpu_kv8_cache import Cache8, dec, enc, name

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def plain(q, k, v, seen, scale, many=False):
    """(out, lse, ds / 8 U, sum p |v|) of one row's heads: q [hq][d], k and v [slots][hkv][d], seen [slots]."""
    hq, d = q.shape
    hkv = k.shape[1]
    out, lse, size, spread = np.zeros((hq, d)), np.full(hq, -np.inf), np.zeros(hq), np.zeros((hq, d))
    k, v = k[seen], v[seen]
    if not len(k):
        return out, lse, size, spread
    for h in range(hq):
        g = h // (hq // hkv)
        s = scale * (k[:, g] @ q[h])
        m = s.max()
        p = np.exp(s - m)
        lse[h] = m + np.log(p.sum())
        p /= p.sum()
        out[h], spread[h] = p @ v[:, g], p @ np.abs(v[:, g])
        size[h] = abs(scale) * (266 / 8 * (np.abs(k[:, g]) @ np.abs(q[h])).max() if many else np.abs(q[h]).max() * np.abs(k[:, g]).sum(1).max())
    return out, lse, size, spread


def check(seed, lens, counts, hq, hkv, d, page, block, *, bf16=False, layout="token", window=0, sinks=0, mask=None, gate=False, holes=(),
          gap=0, extra=0, uniform=False, max_len=None, q_scale=1.0, v_size=1.0, scale=None, workspace=0, behind=0, stream=None):
    B, L = len(lens), max(max(lens), 1) if max_len is None else max_len
    t = Cache8(seed, B, L, hkv, d, page, block, layout, holes, gap)
    t.fill([min(n, L) for n in lens], v_size)
    rng, unit = t.rng, 8 if bf16 else 4
    cu = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    used, most = int(cu[-1]), max(counts)
    rows = used + behind
    qs, os_ = hq * d + extra * unit, hq * d + 2 * extra * unit
    q = enc(q_scale * rng.standard_normal((rows + 1, qs)), bf16)
    gt = enc(rng.standard_normal((rows + 1, qs)), bf16)
    c = t.open()
    out = DeviceBuffer.from_host(np.full((rows + 2, os_), 9, q.dtype))
    lse = DeviceBuffer.from_host(np.full((rows + 2, hq), 9, np.float32))
    up = DeviceBuffer.from_host
    mb = None if mask is None else up(np.ascontiguousarray(np.pad(mask, ((0, 0), (0, 5)), constant_values=1), np.uint8))
    held = up(q), up(gt), up(np.array(lens, np.int32)), up(cu)
    need = workspace if workspace > 1 else attend8_workspace_bytes(B, rows, most, hq, hkv, d, L)
    ws = DeviceBuffer.from_host(np.full(max(need, 1) + 256, 0xa5, np.uint8)) if workspace else None
    c.attend(held[0], out, held[2], B, rows, most, L, hq, cu=None if uniform else held[3], dtype=name(bf16), window=window,
             sinks=sinks, mask=mb, mask_stride=L + 5 if mask is not None else 0, gate=held[1] if gate else None, lse=lse, scale=scale,
             q_stride=qs if extra else 0, out_stride=os_ if extra else 0, workspace=ws, stream=stream)
    if stream is not None:
        synchronize(stream)
    raw_o, raw_l = out.download(), lse.download()
    if ws is not None:
        assert (ws.download()[max(need, 1):] == 0xa5).all(), "past its workspace"
    assert (raw_o[used:] == 9).all() and (raw_l[used:] == 9).all() and (raw_o[:, hq * d:] == 9).all()
    sc = d ** -0.5 if scale is None else scale
    worst = 0.0
    for b in range(B):
        n = min(max(lens[b], 0), L)
        k, v, there = t.values(b, 0, n)
        big = np.abs(v[there]).max() if there.any() else 0.0
        for i in range(counts[b]):
            at, r = n - counts[b] + i, cu[b] + i
            j = np.arange(n)
            seen = there & (j <= at)
            if window:
                seen &= (at - j < window) | (j < sinks)
            if mask is not None:
                seen &= mask[b, :n] != 0
            with np.errstate(invalid="ignore"):
                o, l, size, spread = plain(dec(q[r, :hq * d]).reshape(hq, d), k, v, seen, sc, most * (hq // hkv) > 256 and d <= 128)
            ds = 8 * U * size
            got_o, got_l = dec(raw_o[r, :hq * d]).reshape(hq, d), raw_l[r].astype(np.float64)
            assert np.array_equal(np.isneginf(got_l), np.isneginf(l)), (b, i)
            fine = np.isfinite(l)
            assert (np.abs(got_l[fine] - l[fine]) <= ds[fine] + 600 * U + 2 * U * np.abs(l[fine])).all(), (b, i)
            bar = (2 * ds[:, None] + 600 * U) * spread + n * 2.0 ** -39 * big
            if gate:
                g = 1 / (1 + np.exp(-dec(gt[r, :hq * d]).reshape(hq, d)))
                o, bar = o * g, bar * g + 8 * U * np.abs(o)
            bar = bar + (2.0 ** -8 * np.abs(o) if bf16 else 0)
            err = np.abs(got_o - o)
            assert (err <= bar).all(), (b, i, float((err / np.maximum(bar, 1e-300)).max()))
            if not seen.any():
                assert not got_o.any()
            worst = max(worst, float((err / np.maximum(bar, 1e-300)).max()))
    return raw_o, raw_l, worst


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("hq,hkv,d,page,block,layout", [
    (16, 4, 128, 64, 64, "token"), (4, 4, 64, 16, 16, "head"), (8, 1, 80, 64, 32, "token"), (12, 3, 96, 32, 16, "head"),
    (32, 2, 64, 128, 128, "token"), (20, 1, 128, 256, 256, "head"), (2, 2, 256, 32, 32, "token"), (24, 8, 192, 16, 16, "token"),
    (1, 1, 16, 16, 16, "token"), (40, 2, 48, 64, 16, "head")])
def test_one_token(gpu, bf16, hq, hkv, d, page, block, layout):
    """Lengths of one, around tiles, blocks, pages and splits, and none at all."""
    check(hq + d, (1, 2, 15, 16, 17, 63, 64, 65, 255, 256, 257, 300, 513, 0, 1100), [1] * 15, hq, hkv, d, page, block, bf16=bf16,
          layout=layout, uniform=True)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("hq,hkv,d,page,block", [(16, 4, 128, 64, 64), (32, 2, 64, 32, 32), (8, 8, 80, 16, 16), (3, 1, 256, 64, 16),
                                                 (20, 1, 128, 64, 32), (12, 3, 192, 32, 16)])
def test_drafted_tokens(gpu, bf16, hq, hkv, d, page, block):
    """Ragged counts, sequences with none, with all of their slots new, and with one."""
    check(d + hq, (6, 300, 17, 64, 700, 0, 33, 1), (6, 5, 1, 7, 4, 0, 0, 1), hq, hkv, d, page, block, bf16=bf16)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("hq,hkv,d", [(4, 1, 128), (2, 2, 64), (8, 1, 80), (2, 1, 256)])
def test_prompts(gpu, bf16, hq, hkv, d):
    """Whole prompts and pieces of them, over many tiles of rows."""
    check(d, (150, 333, 70, 1), (150, 60, 33, 1), hq, hkv, d, 64, 64, bf16=bf16)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("hq,hkv,d,page,block,layout", [(4, 1, 64, 64, 64, "token"), (6, 2, 128, 16, 16, "head"), (8, 1, 80, 128, 32, "token"),
                                                        (5, 1, 96, 32, 32, "head"), (3, 1, 16, 64, 16, "token"), (9, 3, 112, 256, 256, "token")])
def test_many_rows(gpu, bf16, hq, hkv, d, page, block, layout):
    """More than 256 rows of a kv head: whole prompts, pieces behind a context, a last tile of one row, sequences with few and none."""
    G = hq // hkv
    n = 257 // G + 1
    check(d, (n, 700, 64 * 3, 1, 90, 0), (n, n - 1, 65, 1, 90, 0), hq, hkv, d, page, block, bf16=bf16, layout=layout, gate=True, gap=1, extra=1)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("window,sinks", [(1, 0), (33, 4), (200, 70), (1500, 0)])
def test_many_rows_behind_windows(gpu, bf16, window, sinks):
    """Stages that no row sees are not walked; masks and holes in those that some do."""
    rng = np.random.default_rng(window)
    mask = (rng.random((2, 2300)) < 0.8).astype(np.uint8)
    mask[1, :400] = 0
    check(window, (2300, 500), (70, 130), 8, 2, 64, 32, 16, window=window, sinks=sinks, bf16=bf16, mask=mask, holes=((0, 60, -1), (1, 13, -5)))
    check(window + 1, (2300, 500), (70, 130), 4, 1, 128, 64, 64, window=window, sinks=sinks, bf16=bf16)


def test_many_splits(gpu):
    """Splits beyond those that one group of lanes joins at a time, of one row, of some and of many."""
    check(40, (9000, 100), (1, 1), 2, 1, 64, 256, 256)
    check(41, (9000, 5200), (9, 2), 2, 1, 64, 256, 64)
    check(42, (17000,), (140,), 2, 1, 64, 256, 256, bf16=True)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 0), (17, 4), (100, 16), (64, 70), (300, 5), (5000, 3), (1 << 40, 0)])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (4, 1, 64)])
def test_windows(gpu, window, sinks, hq, hkv, d):
    check(window % 1000 + sinks, (1, 40, 700, 333, 18), (1, 3, 1, 200, 18), hq, hkv, d, 32, 16, window=window, sinks=sinks)


@pytest.mark.parametrize("bf16", [False, True])
def test_window_of_long_contexts(gpu, bf16):
    """Most of the cache out of sight."""
    check(4, (9000, 4097), (3, 1), 8, 2, 64, 64, 64, window=700, sinks=4, bf16=bf16)


def test_masks_and_holes(gpu):
    """Left padding, all padding, single slots, the row's own slot masked; pages missing at the start, the middle and the end."""
    rng = np.random.default_rng(5)
    lens, counts = (300, 300, 300, 300, 90), (1, 4, 2, 70, 5)
    mask = np.ones((5, 300), np.uint8)
    mask[0, :123] = 0
    mask[1] = 0
    mask[2] = 0
    mask[2, 77] = 255
    mask[3] = rng.random(300) < 0.3
    mask[4, 86:] = 0
    for more in (dict(), dict(window=50, sinks=2), dict(bf16=True, gate=True)):
        check(6, lens, counts, 8, 2, 64, 32, 16, mask=mask, **more)
        check(7, lens, counts, 8, 2, 64, 16, 16, mask=mask, holes=((0, 18, -1), (2, 4, 1 << 30), (3, 2, -2), (3, 3, -1), (4, 0, -1)), **more)
    check(8, (64, 64), (3, 64), 4, 1, 128, 32, 32, holes=((0, 0, -1), (0, 1, -1), (1, 1, -9)))


@pytest.mark.parametrize("bf16", [False, True])
def test_gate_strides_and_workspace(gpu, bf16):
    s = Stream()
    for counts in ((1, 1, 1), (3, 2, 4), (100, 20, 90)):
        check(9, (400, 20, 900), counts, 8, 2, 64, 64, 32, bf16=bf16, gate=True, gap=1, extra=1, workspace=True)
        check(10, (400, 20, 900), counts, 4, 4, 128, 64, 64, bf16=bf16, workspace=True, max_len=1000, stream=s.handle)


@pytest.mark.parametrize("bf16", [False, True])
def test_one_workspace_for_shorter_calls(gpu, bf16):
    """A workspace of the most rows and slots serves fewer, also where the packed arrays stay as long as for the most."""
    for hq, hkv, d, most in ((8, 2, 64, 5), (4, 2, 128, 140), (4, 1, 192, 70)):
        need = attend8_workspace_bytes(3, 3 * most, most, hq, hkv, d, 2300)
        for counts in ((1, 1, 1), (4, 2, 4), (5, 5, 1), (70, 1, 30), (most, 1, most)):
            if max(counts) > most:
                continue
            for L in (2300, 1100):
                for behind in (0, 3 * most - sum(counts)):
                    check(21, (L, 5, L - 40), counts, hq, hkv, d, 64, 32, bf16=bf16, workspace=need, max_len=L, behind=behind)


@pytest.mark.parametrize("q_scale,size,scale", [(30.0, 1.0, None), (1e20, 1e-20, None), (1e-18, 1e18, None), (1.0, 1.0, -0.3), (2.0, 1.0, 0.0)])
def test_sizes_of_values(gpu, q_scale, size, scale):
    """Sharp and flat softmaxes, tiny and huge numbers, a negative and a zero scale."""
    check(11, (700, 33), (2, 1), 8, 2, 128, 64, 16, q_scale=q_scale, v_size=size, scale=scale)


def test_blocks_of_unlike_scale(gpu):
    """V's scales over 2^40 and zeros among them, keys flat: what the large blocks leave of the small ones' share is within the bar."""
    B, n = 1, 640
    for order in (1, -1):
        t = Cache8(12, B, n, 1, 64, 32, 16)
        t.fill([n])
        for j0 in range(0, n, 16):
            p, tok = t.at(0, j0)
            t.scales[0][p, tok // 16] = 2.0 ** -10
            t.scales[1][p, tok // 16] = 0.0 if j0 == 320 else 2.0 ** (order * (j0 // 16 - 20))
        rng = t.rng
        q = rng.standard_normal((2, 4 * 64)).astype(np.float32)
        c = t.open()
        out = DeviceBuffer((2, 256), np.float32)
        c.attend(DeviceBuffer.from_host(q), out, DeviceBuffer.from_host(np.array([n], np.int32)), 1, 2, 2, n, 4)
        k, v, _ = t.values(0, 0, n)
        for i in range(2):
            o, _, size, spread = plain(q[i].astype(np.float64).reshape(4, 64), k, v, np.arange(n) <= n - 2 + i, 0.125)
            bar = (16 * U * size[:, None] + 600 * U) * spread + n * 2.0 ** -39 * np.abs(v).max()
            assert (np.abs(out.download()[i].reshape(4, 64) - o) <= bar).all()


@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf])
def test_queries_that_are_not_numbers(gpu, what):
    """The head that holds one is NaN, and no other."""
    for bf16 in (False, True):
        for counts in ((1, 1), (4, 3), (40, 50)):
            t = Cache8(13, 2, 400, 2, 64, 64, 64)
            t.fill([400, 70])
            rows, hq = sum(counts), 8
            q = enc(t.rng.standard_normal((rows, hq, 64)), bf16)
            got = []
            spoilt = [(0, 3, 5), (rows - 1, 7, 63)]
            for spoil in (False, True):
                for r, h, e in spoilt if spoil else ():
                    q[r, h, e] = enc(np.float32([what]), bf16)[0]
                c = t.open()
                out, lse = DeviceBuffer((rows, hq, 64), q.dtype), DeviceBuffer((rows, hq), np.float32)
                c.attend(DeviceBuffer.from_host(q), out, DeviceBuffer.from_host(np.array([400, 70], np.int32)), 2, rows, max(counts), 400, hq,
                         cu=DeviceBuffer.from_host(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)), dtype=name(bf16), lse=lse)
                got.append((dec(out.download()), lse.download().astype(np.float64)))
            for a, b in zip(*got):
                bad = np.zeros(a.shape[:2], bool)
                for r, h, _ in spoilt:
                    bad[r, h] = True
                assert np.isnan(b[bad]).all()
                assert np.array_equal(a[~bad], b[~bad])


def test_scales_that_are_not_numbers(gpu):
    """A visible NaN scale makes what sees it NaN; the same scale out of sight (past the row, behind the window, masked, in a hole) changes nothing."""
    t = Cache8(14, 1, 256, 1, 64, 64, 16)
    t.fill([256])
    q = t.rng.standard_normal((2, 4, 64)).astype(np.float32)
    lens, qb = DeviceBuffer.from_host(np.array([256], np.int32)), DeviceBuffer.from_host(q)

    def run(**more):
        c = t.open()
        out, lse = DeviceBuffer((2, 4, 64), np.float32), DeviceBuffer((2, 4), np.float32)
        c.attend(qb, out, lens, 1, 2, 2, 256, 4, lse=lse, **more)
        return np.concatenate([out.download().reshape(-1), lse.download().reshape(-1)])

    mask = np.ones((1, 256), np.uint8)
    mask[0, 64:96] = 0
    forms = (dict(window=100), dict(window=100, sinks=16), dict(mask=DeviceBuffer.from_host(mask)))
    want = [run(**f) for f in forms]
    p, tok = t.at(0, 80)
    for which in (0, 1):
        kept = t.scales[which][p, tok // 16].copy()
        for bad in (np.nan, np.inf):
            t.scales[which][p, tok // 16] = bad
            for f, w in zip(forms, want):
                assert np.array_equal(run(**f), w)
            assert np.isnan(run()).any()
        t.scales[which][p, tok // 16] = kept


def test_numbers_out_of_range(gpu):
    """Lengths past max_len and below 0, offsets past the rows, counts above max_new and above the length."""
    t = Cache8(15, 3, 64, 1, 64, 16, 16)
    t.fill([64, 0, 2])
    c = t.open()
    q = t.rng.standard_normal((9, 64)).astype(np.float32)
    out, lse = DeviceBuffer.from_host(np.full((9, 64), 7, np.float32)), DeviceBuffer.from_host(np.full((9, 1), 7, np.float32))
    lens, cu = np.array([1 << 30, -5, 2], np.int32), np.array([-9, 3, 3, 1 << 30], np.int32)
    c.attend(DeviceBuffer.from_host(q), out, DeviceBuffer.from_host(lens), 3, 9, 3, 64, 1, cu=DeviceBuffer.from_host(cu), lse=lse)
    o, l = out.download(), lse.download()
    for b, n, first, count in ((0, 64, 0, 3), (2, 2, 3, 3)):
        k, v, _ = t.values(b, 0, n)
        for i in range(count):
            w, wl, size, spread = plain(q[first + i].astype(np.float64).reshape(1, 64), k, v, np.arange(n) <= n - count + i, 0.125)
            assert (np.abs(o[first + i] - w) <= (16 * U * size[:, None] + 600 * U) * spread + 1e-7).all()
            assert np.isneginf(l[first + i, 0]) == np.isneginf(wl[0])
    assert not o[3].any()  # a row before slot 0
    assert (o[6:] == 7).all() and (l[6:] == 7).all()


def test_a_sequence_does_not_depend_on_its_batch(gpu):
    """Alone, with others, again: the same bits."""
    for d, counts in ((128, (1, 1, 1, 1)), (64, (5, 2, 6, 1)), (64, (130, 40, 7, 64))):
        t = Cache8(16, 4, 2000, 2, d, 64, 32)
        lens = np.array([2000, 40, 700, 64], np.int32)
        t.fill(lens)
        t.open()
        hq, rows = 8, sum(counts)
        cu = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        q = t.rng.standard_normal((rows, hq, d)).astype(np.float32)

        def run(bs):
            pick = np.concatenate([np.arange(cu[b], cu[b + 1]) for b in bs])
            c = KVCache8(*t.dev[:4], DeviceBuffer.from_host(t.table[list(bs)]), n_pages=t.n_pages, max_pages=t.maxp, page_tokens=64,
                         block_tokens=32, n_head_kv=2, head_dim=d, strides=t.strides)
            out = DeviceBuffer((len(pick), hq, d), np.float32)
            c.attend(DeviceBuffer.from_host(q[pick]), out, DeviceBuffer.from_host(lens[list(bs)]), len(bs), len(pick), max(counts), 2000, hq,
                     cu=DeviceBuffer.from_host(np.concatenate([[0], np.cumsum([counts[b] for b in bs])]).astype(np.int32)))
            return out.download()

        whole = run((0, 1, 2, 3))
        assert np.array_equal(run((0, 1, 2, 3)), whole)
        for b in range(4):
            assert np.array_equal(run((b,)), whole[cu[b]:cu[b + 1]])


def test_bf16_rows_are_rounded_once(gpu):
    """With queries that bf16 holds, a bf16 output is the fp32 call's rounded to nearest even."""
    for counts in ((1, 1), (6, 3), (90, 70)):
        t = Cache8(17, 2, 500, 2, 128, 64, 64)
        t.fill([500, 80])
        c, rows = t.open(), sum(counts)
        q = enc(t.rng.standard_normal((rows, 8, 128)), True)
        cu = DeviceBuffer.from_host(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32))
        got = []
        for bf16 in (False, True):
            out = DeviceBuffer((rows, 8, 128), np.uint16 if bf16 else np.float32)
            c.attend(DeviceBuffer.from_host(q if bf16 else dec(q).astype(np.float32)), out, DeviceBuffer.from_host(np.array([500, 80], np.int32)),
                     2, rows, max(counts), 500, 8, cu=cu, dtype=name(bf16))
            got.append(out.download())
        assert np.array_equal(enc(got[0], True), got[1])


def test_large_offsets(gpu):
    """Pages past 2^32 bytes into the pool, read and written there."""
    page, d = 256, 256
    n_pages = (1 << 32) // (page * d) + 8000
    k, v = (DeviceBuffer((n_pages, page * d), np.int8) for _ in range(2))
    ks, vs = (DeviceBuffer((n_pages, 1, 1), np.float32, zero=True) for _ in range(2))
    table = DeviceBuffer.from_host(np.array([[n_pages - 1, n_pages - 2]], np.int32))
    c = KVCache8(k, v, ks, vs, table, n_pages=n_pages, max_pages=2, page_tokens=page, block_tokens=page, n_head_kv=1, head_dim=d)
    rng = np.random.default_rng(3)
    x, y = (rng.integers(-127, 128, (300, d)).astype(np.float32) for _ in range(2))
    x[::256], y[::256] = 127, 127
    lens = DeviceBuffer.from_host(np.array([300], np.int32))
    c.write(DeviceBuffer.from_host(x), DeviceBuffer.from_host(y), lens, 1, 300, 300)
    q = (0.01 * rng.standard_normal((2, 2, d))).astype(np.float32)
    out = DeviceBuffer((2, 2, d), np.float32)
    c.attend(DeviceBuffer.from_host(q), out, lens, 1, 2, 2, 300, 2)
    for i in range(2):
        o, _, size, spread = plain(q[i].astype(np.float64), x[:, None].astype(np.float64), y[:, None].astype(np.float64),
                                   np.arange(300) <= 298 + i, d ** -0.5)
        assert (np.abs(out.download()[i] - o) <= (16 * U * size[:, None] + 600 * U) * spread + 300 * 2.0 ** -39 * 127).all()


def test_refusals(gpu):
    b = DeviceBuffer((1 << 16,), np.uint8, zero=True)

    def call(q=b, o=b, lens=b, rows=2, new=1, seqs=2, max_len=32, hq=4, d=32, hkv=2, **more):
        c = KVCache8(b, b, b, b, b, n_pages=2, max_pages=2, page_tokens=16, block_tokens=16, n_head_kv=hkv, head_dim=d)
        c.attend(q, o, lens, seqs, rows, new, max_len, hq, **more)

    for code, more in ((1, dict(q=None)), (1, dict(o=None)), (1, dict(lens=None)), (1, dict(scale=float("inf"))), (1, dict(scale=float("nan"))),
                       (2, dict(max_len=33)), (2, dict(hq=3)), (2, dict(hq=0)), (2, dict(d=40)), (2, dict(rows=3)), (2, dict(q_stride=120)),
                       (2, dict(out_stride=120)), (2, dict(mask=b, mask_stride=31)), (2, dict(seqs=70000, rows=70000)), (2, dict(hq=70000)),
                       (3, dict(q=b.ptr + 4)), (3, dict(o=b.ptr + 8)), (3, dict(gate=b.ptr + 4)), (3, dict(q_stride=130))):
        with pytest.raises(OuroError) as e:
            call(**more)
        assert e.value.code == code, more
    with pytest.raises(ValueError):
        call(dtype="f16")
    call(seqs=0, rows=0, new=0)
    call(max_len=0)


def test_two_streams_in_flight(gpu):
    """Calls of both streams queued in turn, small ones ahead of larger ones so that the scratch grows between them."""
    made = []
    for i in range(2):
        for B, count in ((1, 1), (24, 5)):
            t = Cache8(30 + i + B, B, 3000, 2, 64, 64, 64)
            t.fill([3000] * B)
            c = t.open()
            q = DeviceBuffer.from_host(t.rng.standard_normal((B * count, 8, 64)).astype(np.float32))
            made.append((i, t, c, q, DeviceBuffer.from_host(np.full(B, 3000, np.int32)), B, count))

    def run(m, stream):
        _, _, c, q, lens, B, count = m
        out = DeviceBuffer((B * count, 8, 64), np.float32, zero=True)
        synchronize()
        return lambda: (c.attend(q, out, lens, B, B * count, count, 3000, 8, stream=stream), out)[1]

    streams = [Stream(), Stream()]
    queue = [(m, run(m, streams[m[0]].handle)) for _ in range(4) for m in sorted(made, key=lambda m: m[5])]
    got = [(m, go()) for m, go in queue]
    for s in streams:
        s.synchronize()
    want = {id(m): run(m, None)().download() for m in made}
    for m, o in got:
        assert np.array_equal(o.download(), want[id(m)])
