"""Attention of one new token over a paged cache (ouro_kv_attend) and eviction
from it (ouro_kv_evict) against plain float64 restatements.

Attention's bars, U = 2^-24.  A score is a sum of head_dim products in chains
and trees of at most 64 roundings (products of bf16 operands, and of fp32 ones
split in three, are as exact as fp32), scaled once or twice, so its error is at
most ds = 68 U S, S = |scale| sum |q k| (the largest over the slots).  e^(s - m)
and its sum move by that each; the running maximum's corrections, the sums over
the slots (chains of at most 512 roundings: a split's slots, then the splits)
and exp itself add less than 600 U.  So the output is within
(2 ds + 600 U) sum p |v|, a slot's weight within (2 ds + 600 U) of its own size
and a rounding of the history's, lse within ds + 600 U + 2 U |lse|.  A bf16
output adds its rounding, 2^-8 of its size.  The gate adds 8 U.

A slot left out, or counted twice, moves the output by its weight, at 1 / n on
average 50 times the bar of the longest sequences here.

Eviction moves bytes and whole numbers: everything is compared bit for bit."""
import numpy as np
import pytest

from ouroboros_amd import _lib
from ouroboros_amd._lib import DT_BF16, DT_F32, KvCacheDesc, OuroError, call
from ouroboros_amd.device import DeviceBuffer, Stream
from ouroboros_amd.kvcache import History, KVCache, attend_workspace_bytes, evict_workspace_bytes
from ouroboros_amd.quant import bf16_bits_to_f32, f32_to_bf16_bits

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def enc(x, bf16):
    return f32_to_bf16_bits(np.ascontiguousarray(x, np.float32)) if bf16 else np.ascontiguousarray(x, np.float32)


def dec(x):
    return bf16_bits_to_f32(x) if x.dtype == np.uint16 else x


def name(bf16):
    return "bf16" if bf16 else "f32"


GARBAGE = np.array([np.nan, np.inf, -np.inf, 3e38, -3e38], np.float32)


class Setup:
    """A cache whose unused slots hold NaN, infinities and huge values."""

    def __init__(self, seed, lens, hkv, d, page, bf16, layout="token", max_len=None, holes=(), extra_stride=0):
        rng = np.random.default_rng(seed)
        self.rng, self.lens, self.hkv, self.d, self.page, self.bf16, self.layout = rng, np.array(lens, np.int32), hkv, d, page, bf16, layout
        self.max_len = max(int(max(lens)), 1) if max_len is None else max_len
        B, self.maxp = len(lens), -(-max(self.max_len, 1) // page)
        self.n_pages = B * self.maxp + 2
        self.table = rng.permutation(self.n_pages)[:B * self.maxp].astype(np.int32).reshape(B, self.maxp)
        for b, p, what in holes:
            self.table[b, p] = what
        row = d + extra_stride
        shape = (self.n_pages, hkv, page, row) if layout == "head" else (self.n_pages, page, hkv, row)
        self.strides = (hkv * page * row, row, page * row) if layout == "head" else (hkv * page * row, hkv * row, row)
        self.k, self.v = (enc(rng.choice(GARBAGE, shape), bf16) for _ in range(2))
        for b, n in enumerate(lens):
            for j in range(min(n, self.max_len)):
                p = self.table[b, j // page]
                if 0 <= p < self.n_pages:
                    for pool in (self.k, self.v):
                        self.view(pool)[p, j % page] = enc(rng.standard_normal((hkv, d)), bf16)

    def view(self, pool):
        x = pool.transpose(0, 2, 1, 3) if self.layout == "head" else pool
        return x[..., :self.d]

    def open(self):
        self.kb, self.vb = DeviceBuffer.from_host(self.k), DeviceBuffer.from_host(self.v)
        self.pb = DeviceBuffer.from_host(self.table)
        return KVCache(self.kb, self.vb, self.pb, n_pages=self.n_pages, max_pages=self.maxp, page_tokens=self.page,
                       n_head_kv=self.hkv, head_dim=self.d, dtype=name(self.bf16), strides=self.strides)

    def rows(self, b):
        """Live slots of sequence b (page there) and their rows in float64."""
        j = np.arange(max(0, min(self.lens[b], self.max_len)))
        p = self.table[b, j // self.page]
        j = j[(p >= 0) & (p < self.n_pages)]
        p = self.table[b, j // self.page]
        k, v = (dec(self.view(pool)[p, j % self.page]).astype(np.float64) for pool in (self.k, self.v))
        return j, k, v


def check_attend(seed, lens, hq, hkv, d, page, *, cache=True, io=False, layout="token", mask=None, gate=False,
                 history=None, append=True, max_len=None, holes=(), extra=0, q_scale=1.0, scale=None, workspace=False,
                 stream=None):
    """Runs one call and checks every output; returns the raw ones."""
    t = Setup(seed, lens, hkv, d, page, cache, layout, max_len, holes, extra * (8 if cache else 4))
    rng, B, G, L = t.rng, len(lens), hq // hkv, t.max_len
    unit = 8 if io else 4
    qs, ns, os_ = (hq * d + extra * unit, hkv * d + 2 * extra * unit, hq * d + 3 * extra * unit)
    q = enc(np.float32(q_scale) * rng.standard_normal((B, qs)).astype(np.float32), io)
    kn, vn = (enc(rng.standard_normal((B, ns)), io) for _ in range(2))
    gt = enc(rng.standard_normal((B, qs)), io) if gate else None
    n = np.clip(t.lens, 0, L)
    pos_new = (7000 + np.arange(B)).astype(np.int32)
    hs = {None: 0, "heads": hkv, "shared": 1}[history]
    slots = L + 3
    w0 = rng.uniform(0, 4, (B, hs, slots)).astype(np.float32)
    p0 = rng.integers(0, 5000, (B, hs, slots)).astype(np.int32)
    c = t.open()
    if append:  # the new row as the cache stores it
        for b in range(B):
            if n[b]:
                p = t.table[b, (n[b] - 1) // page]
                if 0 <= p < t.n_pages:
                    for pool, new in ((t.k, kn), (t.v, vn)):
                        t.view(pool)[p, (n[b] - 1) % page] = enc(dec(new[b, :hkv * d]).reshape(hkv, d), cache)
    dev = {x: DeviceBuffer.from_host(y) for x, y in dict(q=q, kn=kn, vn=vn, lens=t.lens, pos=pos_new).items()}
    mb = None if mask is None else DeviceBuffer.from_host(np.ascontiguousarray(np.pad(mask, ((0, 0), (0, 5)), constant_values=1), np.uint8))
    gb = DeviceBuffer.from_host(gt) if gate else None
    hist = wb = pb = None
    if history:
        wb, pb = DeviceBuffer.from_host(w0), DeviceBuffer.from_host(p0)
        hist = History(wb, pb, hs, slots)
    sent = enc(np.full((B, os_), 77.0), io)
    ob, lb = DeviceBuffer.from_host(sent), DeviceBuffer((B, hq), np.float32)
    ws = None
    if workspace:
        ws = DeviceBuffer((max(1, attend_workspace_bytes(B, hq, d, L, history is not None)),), np.uint8)
    h = stream.handle if stream else None
    c.attend(dev["q"], ob, dev["lens"], B, L, hq, dtype=name(io), k_new=dev["kn"] if append else None,
             v_new=dev["vn"] if append else None, pos_new=dev["pos"] if append else None, history=hist, mask=mb,
             mask_stride=L + 5 if mask is not None else 0, gate=gb, lse=lb, scale=scale, q_stride=qs, new_stride=ns, out_stride=os_, workspace=ws, stream=h)
    if stream:
        stream.synchronize()
    out, lse = ob.download(), lb.download()
    assert np.array_equal(out[:, hq * d:], sent[:, hq * d:])  # the gap between rows
    got = dec(out[:, :hq * d]).reshape(B, hq, d).astype(np.float64)
    sc = d ** -0.5 if scale is None else scale
    want_w = w0.astype(np.float64)
    bar_w = U * np.abs(want_w)
    if append and history:
        for b in range(B):
            if n[b]:
                want_w[b, :, n[b] - 1] = 0
    # every slot of the pools: the new rows alone changed
    assert np.array_equal(t.kb.download().view(np.uint8), t.k.view(np.uint8)) and np.array_equal(t.vb.download().view(np.uint8), t.v.view(np.uint8))
    for b in range(B):
        j, k, v = t.rows(b)
        if mask is not None:
            live = mask[b, j] != 0
            j, k, v = j[live], k[live], v[live]
        for hh in range(hq):
            if not len(j):
                assert (got[b, hh] == 0).all() and lse[b, hh] == -np.inf
                continue
            qv = dec(q[b, hh * d:(hh + 1) * d]).astype(np.float64)
            s = sc * (k[:, hh // G] @ qv)
            S = abs(sc) * (np.abs(k[:, hh // G]) @ np.abs(qv)).max()
            e = np.exp(s - s.max())
            p = e / e.sum()
            bar = 2 * 68 * U * S + 600 * U
            w_lse = s.max() + np.log(e.sum())
            assert abs(lse[b, hh] - w_lse) <= 68 * U * S + 600 * U + 2 * U * abs(w_lse), (b, hh)
            o, room = p @ v[:, hh // G], bar * (p @ np.abs(v[:, hh // G]))
            if gate:
                g = 1 / (1 + np.exp(-dec(gt[b, hh * d:(hh + 1) * d]).astype(np.float64)))
                o, room = o * g, room * g + 8 * U * np.abs(o * g)
            if io:
                room = room + 2.0 ** -8 * np.abs(o)
            assert (np.abs(got[b, hh] - o) <= room).all(), (b, hh, np.abs(got[b, hh] - o).max())
            if history:
                hw = hh // G if history == "heads" else 0
                want_w[b, hw, j] += p
                bar_w[b, hw, j] += (bar + 4 * U) * p + U * want_w[b, hw, j]
    if history:
        w, p = wb.download(), pb.download()
        assert (np.abs(w - want_w) <= bar_w).all()
        if append:
            for b in range(B):
                if n[b]:
                    p0[b, :, n[b] - 1] = pos_new[b]
        assert np.array_equal(p, p0)
        return out, lse, w
    return out, lse


@pytest.mark.parametrize("lens", [(1,), (2, 3, 63), (64, 65, 31, 33), (255, 256, 257, 0), (300, 1, 511, 513), (2305,)], ids=str)
@pytest.mark.parametrize("cache,io", [(True, False), (True, True), (False, False), (False, True)])
def test_lengths_and_types(gpu, lens, cache, io):
    check_attend(len(lens) + sum(lens), lens, 8, 2, 128, 64, cache=cache, io=io)


@pytest.mark.parametrize("d", [8, 24, 64, 72, 80, 96, 128, 136, 192, 256])
@pytest.mark.parametrize("cache", [True, False])
def test_head_widths(gpu, d, cache):
    check_attend(d, (70, 300, 5), 6, 2, d, 32, cache=cache, history="heads")


@pytest.mark.parametrize("hq,hkv", [(1, 1), (4, 4), (3, 1), (16, 1), (17, 1), (40, 2), (14, 7)])
@pytest.mark.parametrize("history", ["heads", "shared"])
def test_heads_over_kv_heads(gpu, hq, hkv, history):
    check_attend(hq, (41, 290), hq, hkv, 64, 16, history=history)


@pytest.mark.parametrize("page", [1, 2, 8, 16, 128, 1024])
@pytest.mark.parametrize("layout", ["token", "head"])
def test_pages_and_layouts(gpu, page, layout):
    """Pages that end inside a tile of slots, and that hold more than a split."""
    check_attend(page, (37, 300, 129), 4, 2, 64, page, layout=layout, history="heads")
    check_attend(page, (37, 300, 129), 4, 2, 64, page, cache=False, layout=layout, append=False)


@pytest.mark.parametrize("cache,io", [(True, False), (False, False), (True, True)])
def test_strides(gpu, cache, io):
    check_attend(3, (100, 17), 4, 2, 80, 16, cache=cache, io=io, extra=3, gate=True)


@pytest.mark.parametrize("cache", [True, False])
def test_masks_and_holes(gpu, cache):
    """Masked slots, rows that a mask or holes leave empty, a masked new slot, ids out of range."""
    lens = (300, 70, 33, 64, 5, 600)
    rng = np.random.default_rng(1)
    mask = (rng.random((6, 600)) < 0.5).astype(np.uint8) * 255
    mask[1] = 0
    mask[2, :32] = 0       # the new slot alone
    mask[3, 63] = 0        # the new slot not
    mask[5, :512] = 0      # whole splits of nothing
    holes = [(0, 1, -1), (0, 2, 1 << 30), (4, 0, -5)]
    for history in ("heads", "shared"):
        check_attend(9, lens, 8, 2, 64, 32, cache=cache, mask=mask, holes=holes, history=history, gate=True)
    check_attend(9, lens, 8, 2, 64, 32, cache=cache, mask=mask, holes=holes, append=False, io=True)


def test_lens_past_the_bound_and_below_zero(gpu):
    check_attend(4, (500, -3, 40), 4, 2, 64, 16, max_len=100, history="heads")


def test_no_slots_at_all(gpu):
    check_attend(4, (0, 0), 4, 2, 64, 16, append=False, max_len=0)


@pytest.mark.parametrize("q_scale", [0.0, 1e-3, 30.0])
@pytest.mark.parametrize("cache", [True, False])
def test_score_sizes(gpu, q_scale, cache):
    """30: e^score alone would pass fp32's range; 0: all slots alike."""
    check_attend(5, (700, 33), 8, 2, 128, 64, cache=cache, q_scale=q_scale, history="heads")


def test_given_scale_and_workspace(gpu):
    check_attend(6, (520, 9), 8, 4, 64, 16, scale=-0.3, history="shared", workspace=True)


def test_infinite_scores(gpu):
    """A visible key of -inf scores -inf (weight 0) where others are finite."""
    t = Setup(1, (40,), 1, 64, 16, False)
    t.view(t.k)[t.table[0, 0], 3] = -np.inf
    c = t.open()
    q = DeviceBuffer.from_host(np.ones((1, 2, 64), np.float32))
    out, lb, lens = DeviceBuffer((1, 2, 64), np.float32), DeviceBuffer((1, 2), np.float32), DeviceBuffer.from_host(t.lens)
    c.attend(q, out, lens, 1, 40, 2, lse=lb)
    j, k, v = t.rows(0)
    s = k[:, 0].sum(1) / 8.0
    p = np.exp(s - s.max())
    p /= p.sum()
    assert p[3] == 0
    assert np.abs(out.download()[0] - p @ v[:, 0]).max() <= 1e-4 * np.abs(v).max()


def test_alone_and_in_any_batch_and_twice(gpu):
    """A sequence's rows do not depend on the batch it is in; the same call gives the same bits."""
    lens = (2305, 1, 256, 257, 512, 900)
    t = Setup(7, lens, 2, 128, 32, True)
    t_q = t.rng.standard_normal((len(lens), 8, 128)).astype(np.float32)

    def run(rows):
        table = np.ascontiguousarray(t.table[rows])
        kb, vb, pb = (DeviceBuffer.from_host(x) for x in (t.k, t.v, table))
        c = KVCache(kb, vb, pb, n_pages=t.n_pages, max_pages=t.maxp, page_tokens=32, n_head_kv=2, head_dim=128)
        w = DeviceBuffer.from_host(np.zeros((len(rows), 2, 2305), np.float32))
        p = DeviceBuffer.from_host(np.zeros((len(rows), 2, 2305), np.int32))
        o = DeviceBuffer((len(rows), 8, 128), np.float32)
        ln = DeviceBuffer.from_host(t.lens[rows])
        c.attend(DeviceBuffer.from_host(t_q[rows]), o, ln, len(rows), int(t.lens[rows].max()), 8, history=History(w, p, 2, 2305))
        return o.download(), w.download()

    o, w = run(list(range(len(lens))))
    o2, w2 = run(list(range(len(lens))))
    assert np.array_equal(o, o2) and np.array_equal(w, w2)
    for b in range(len(lens)):
        for rows in ([b], [b, 0]):
            oo, ww = run(rows)
            assert np.array_equal(oo[0], o[b]) and np.array_equal(ww[0], w[b]), (b, rows)


def test_streams(gpu):
    """Two streams at once, each with the library's own scratch."""
    s1, s2 = Stream(), Stream()
    want = [check_attend(50 + i, (1500, 7), 8, 2, 128, 64, history="heads") for i in range(2)]
    for _ in range(2):
        for i, s in enumerate((s1, s2)):
            got = check_attend(50 + i, (1500, 7), 8, 2, 128, 64, history="heads", stream=s)
            assert all(np.array_equal(a, b) for a, b in zip(got, want[i]))


def test_offsets_past_32_bits(gpu):
    """Pages past 2^32 elements of the pools: attended to, appended to and moved."""
    page, hkv, d = 64, 2, 128
    per = page * hkv * d
    n_pages = (1 << 32) // per + 4
    rng = np.random.default_rng(3)
    kb, vb = DeviceBuffer((n_pages, per), np.uint16), DeviceBuffer((n_pages, per), np.uint16)
    ids = np.array([[n_pages - 1, 1, n_pages - 2]], np.int32)
    rows = [enc(rng.standard_normal((3, page, hkv, d)), True) for _ in range(2)]
    for buf, r in zip((kb, vb), rows):
        for i, p in enumerate(ids[0]):
            part = np.ascontiguousarray(r[i])
            call("ouro_memcpy_htod", buf.ptr + int(p) * per * 2, part.ctypes.data, part.nbytes)
    c = KVCache(kb, vb, DeviceBuffer.from_host(ids), n_pages=n_pages, max_pages=3, page_tokens=page, n_head_kv=hkv, head_dim=d)
    q = rng.standard_normal((1, 2, d)).astype(np.float32)
    new = enc(rng.standard_normal((1, hkv, d)), False)
    n = 190
    out = DeviceBuffer((1, 2, d), np.float32)
    lens = DeviceBuffer.from_host(np.array([n], np.int32))
    nb = DeviceBuffer.from_host(new)
    c.attend(DeviceBuffer.from_host(q), out, lens, 1, n, 2, k_new=nb, v_new=nb)
    k, v = (bf16_bits_to_f32(r).reshape(-1, hkv, d)[:n].astype(np.float64) for r in rows)
    k[n - 1] = v[n - 1] = bf16_bits_to_f32(enc(new, True))[0]
    for h in range(2):
        s = k[:, h] @ q[0, h] / np.sqrt(d)
        p = np.exp(s - s.max())
        p /= p.sum()
        S = (np.abs(k[:, h]) @ np.abs(q[0, h])).max() / np.sqrt(d)
        assert (np.abs(out.download()[0, h] - p @ v[:, h]) <= (136 * U * S + 600 * U) * (p @ np.abs(v[:, h]))).all()
    w = np.zeros((1, 1, n), np.float32)
    w[0, 0, 130:150] = 1.0  # of the last page, into the second
    w[0, 0, :44] = 2.0
    h = History(DeviceBuffer.from_host(w), DeviceBuffer.from_host(np.arange(n, dtype=np.int32).reshape(1, 1, n)), 1, n)
    left, src = DeviceBuffer((1,), np.int32), DeviceBuffer((1, 1, 64), np.int32)
    c.evict(h, lens, 1, n, 64, 0, left, slot_from=src)
    assert src.download()[0, 0].tolist() == list(range(44)) + list(range(130, 150))
    got = np.empty((page, hkv, d), np.uint16)
    call("ouro_memcpy_dtoh", got.ctypes.data, kb.ptr + int(ids[0, 0]) * per * 2, got.nbytes)
    assert np.array_equal(got[44:], rows[0][2, 2:22])


# ---- eviction ----

def expected(t, w, pos, keep, recent):
    """slot_from, and the history and pools left, by sorting."""
    B, H, _ = w.shape
    src = np.full((B, H, keep), -1, np.int32)
    k, v = t.k.copy(), t.v.copy()
    w1, p1 = w.copy(), pos.copy()
    for b in range(B):
        n = int(np.clip(t.lens[b], 0, t.max_len))
        for h in range(H):
            at = np.arange(min(n, keep))
            if n > keep:
                x = w[b, h, :n].astype(np.float64)
                new = pos[b, h, :n].astype(np.int64) > int(pos[b, h, :n].max()) - recent
                order = sorted(range(n), key=lambda j: (not new[j], np.isnan(x[j]), -x[j] if x[j] == x[j] else 0.0, j))
                stays = set(order[:keep])
                at[[j for j in range(keep) if j not in stays]] = sorted(j for j in stays if j >= keep)
            src[b, h, :len(at)] = at
            w1[b, h, :len(at)], p1[b, h, :len(at)] = w[b, h, at], pos[b, h, at]
            for j, s in enumerate(at):
                a, c = t.table[b, j // t.page], t.table[b, s // t.page]
                if j != s and 0 <= a < t.n_pages and 0 <= c < t.n_pages:
                    heads = slice(h, h + 1) if H > 1 else slice(None)
                    for old, pool in ((t.k, k), (t.v, v)):
                        t.view(pool)[a, j % t.page, heads] = t.view(old)[c, s % t.page, heads]
    return src, w1, p1, k, v


def check_evict(seed, lens, hkv, d, page, keep, recent, *, heads=None, cache=True, layout="token", weights="spread",
                shuffled=False, apart=False, max_len=None, holes=(), extra=0, stream=None, workspace=False, positions=None):
    t = Setup(seed, lens, hkv, d, page, cache, layout, max_len, holes, extra * 8)
    rng, B, H = t.rng, len(lens), hkv if heads is None else heads
    slots = t.max_len + 2
    w = np.exp(3 * rng.standard_normal((B, H, slots))).astype(np.float32)
    if weights == "ties":
        w = rng.integers(0, 3, w.shape).astype(np.float32)
    elif weights == "equal":
        w = np.full_like(w, 0.25)
    elif weights == "odd":  # every kind of value
        w = rng.choice(np.array([np.nan, np.inf, -np.inf, 0.0, -0.0, -1.0, 1.0, 1e-42, -1e-42, 3e38], np.float32), w.shape)
    pos = np.broadcast_to(np.arange(slots, dtype=np.int32), w.shape).copy()
    if shuffled:
        pos = rng.permuted(pos * 3 - 50, axis=2)
    if positions is not None:
        pos = rng.choice(positions, pos.shape)
    src, w1, p1, k, v = expected(t, w, pos, keep, recent)
    c = t.open()
    hist = History(DeviceBuffer.from_host(w), DeviceBuffer.from_host(pos), H, slots)
    lens_b, left_b, src_b = DeviceBuffer.from_host(t.lens), DeviceBuffer((B,), np.int32), DeviceBuffer((B, H, keep), np.int32)
    out = None
    if apart:
        m = min(keep, t.max_len)
        out = History(DeviceBuffer.from_host(np.full((B, H, m), -9, np.float32)), DeviceBuffer.from_host(np.full((B, H, m), -9, np.int32)), H, m)
    ws = DeviceBuffer((evict_workspace_bytes(B, H, t.max_len, keep),), np.uint8) if workspace else None
    c.evict(hist, lens_b, B, t.max_len, keep, recent, left_b, out=out, slot_from=src_b, workspace=ws,
            stream=stream.handle if stream else None)
    if stream:
        stream.synchronize()
    n = np.clip(t.lens, 0, t.max_len)
    assert np.array_equal(left_b.download(), np.minimum(n, keep))
    assert np.array_equal(src_b.download(), src)
    got_w, got_p = (out or hist).weight.download(), (out or hist).pos.download()
    if apart:
        for b in range(B):
            m = min(n[b], keep)
            assert (got_w[b, :, m:] == -9).all() and (got_p[b, :, m:] == -9).all()
            assert np.array_equal(got_w[b, :, :m].view(np.uint32), w1[b, :, :m].view(np.uint32)) and np.array_equal(got_p[b, :, :m], p1[b, :, :m])
        assert np.array_equal(hist.weight.download().view(np.uint32), w.view(np.uint32))
    else:
        assert np.array_equal(got_w.view(np.uint32), w1.view(np.uint32)) and np.array_equal(got_p, p1)
    assert np.array_equal(t.kb.download().view(np.uint8), k.view(np.uint8))
    assert np.array_equal(t.vb.download().view(np.uint8), v.view(np.uint8))
    return src


@pytest.mark.parametrize("n,keep,recent", [(1, 1, 0), (2, 1, 0), (2, 1, 1), (65, 64, 8), (65, 64, 64), (300, 64, 0), (300, 299, 1),
                                           (257, 255, 300), (1025, 1024, 128), (900, 100, 100), (3000, 1200, 77)])
@pytest.mark.parametrize("weights", ["spread", "ties", "equal", "odd"])
def test_evict_sizes_and_weights(gpu, n, keep, recent, weights):
    check_evict(n + keep, (n, max(1, n // 2), n), 2, 16, 16, keep, recent, weights=weights, shuffled=n % 2 == 0)


@pytest.mark.parametrize("heads", [None, 1])
@pytest.mark.parametrize("layout", ["token", "head"])
@pytest.mark.parametrize("cache", [True, False])
def test_evict_layouts(gpu, heads, layout, cache):
    check_evict(3, (130, 0, 400, 64, -2), 3, 80, 32, 64, 10, heads=heads, layout=layout, cache=cache, shuffled=True)
    check_evict(4, (130, 31, 400), 3, 80, 32, 100, 10, heads=heads, layout=layout, cache=cache, apart=True, workspace=True, extra=2)


def test_evict_keep_past_the_bound(gpu):
    check_evict(5, (30, 100), 2, 64, 16, 150, 10)
    check_evict(5, (30, 100), 2, 64, 16, 150, 10, apart=True)
    check_evict(5, (300, 100), 2, 64, 16, 50, 10, max_len=200)


def test_evict_holes(gpu):
    """History and counts go on as usual; rows of holes are not touched."""
    check_evict(6, (200, 150), 2, 64, 16, 70, 5, holes=[(0, 1, -1), (0, 11, 1 << 20), (1, 8, -7)])


@pytest.mark.parametrize("n", [16384, 16385, 40000])
def test_evict_long(gpu, n):
    check_evict(7, (n, n - 1), 1, 8, 64, n // 5, n // 50, shuffled=True)
    check_evict(8, (n,), 1, 8, 64, n - 1, 100, weights="ties")


@pytest.mark.parametrize("heads", [None, 1])
@pytest.mark.parametrize("n,keep,d,cache", [(2000, 900, 80, True), (700, 340, 256, True), (700, 340, 256, False), (1100, 500, 96, False)])
def test_evict_many_moves(gpu, heads, n, keep, d, cache):
    check_evict(n, (n, n // 2, n - 1), 2, d, 32, keep, 30, heads=heads, cache=cache, shuffled=True, apart=d == 256, holes=[(0, 1, -1), (2, n // 32, 1 << 30)])


@pytest.mark.parametrize("recent", [0, 1, 3, 20, 1 << 30])
def test_evict_positions(gpu, recent):
    """Positions from one end of their type to the other."""
    check_evict(9, (40, 7, 1000), 2, 16, 16, 24, recent, positions=np.array([-2 ** 31, -2 ** 31 + 1, -1, 0, 1, 2 ** 31 - 2, 2 ** 31 - 1], np.int32))
    check_evict(9, (40, 100), 2, 16, 16, 24, recent, positions=np.array([-2 ** 31, -2 ** 31 + 1], np.int32), apart=True)


def test_evict_streams(gpu):
    s = [Stream(), Stream()]
    for _ in range(2):
        for i in range(2):
            check_evict(60 + i, (1000, 300), 2, 64, 16, 200, 20, stream=s[i])


def test_attend_evict_attend(gpu):
    """A cache held at a budget: evicting everything but what a second call sees is a no-op for it."""
    lens, hkv, d, page, keep = (90, 40), 2, 64, 16, 48
    t = Setup(11, lens, hkv, d, page, False)
    c = t.open()
    B, n = 2, 90
    w, p = DeviceBuffer.from_host(np.zeros((B, hkv, n), np.float32)), DeviceBuffer.from_host(np.broadcast_to(np.arange(n, dtype=np.int32), (B, hkv, n)).copy())
    h = History(w, p, hkv, n)
    q = t.rng.standard_normal((B, 4, d)).astype(np.float32)
    qb, lens_b, left_b = DeviceBuffer.from_host(q), DeviceBuffer.from_host(t.lens), DeviceBuffer((B,), np.int32)
    out = DeviceBuffer((B, 4, d), np.float32)
    c.attend(qb, out, lens_b, B, n, 4, history=h)
    weight = w.download()
    c.evict(h, lens_b, B, n, keep, 4, left_b)
    c.attend(qb, out, left_b, B, keep, 4)
    got = out.download()
    for b in range(B):
        j, k, v = t.rows(b)
        for hh in range(4):
            kv = hh // 2
            order = sorted(j, key=lambda i: (i <= j[-1] - 4, -weight[b, kv, i], i))[:keep]
            s = k[order, kv] @ q[b, hh] / 8.0
            e = np.exp(s - s.max())
            e /= e.sum()
            S = (np.abs(k[order, kv]) @ np.abs(q[b, hh])).max() / 8.0
            assert (np.abs(got[b, hh] - e @ v[order, kv]) <= (136 * U * S + 600 * U) * (e @ np.abs(v[order, kv]))).all()


# ---- refusals ----

def small():
    t = Setup(0, (20, 9), 2, 64, 16, True)
    c = t.open()
    b = dict(q=DeviceBuffer((2, 4, 64), np.float32), out=DeviceBuffer((2, 4, 64), np.float32), lens=DeviceBuffer.from_host(t.lens),
             w=DeviceBuffer((2, 2, 32), np.float32), p=DeviceBuffer((2, 2, 32), np.int32), n=DeviceBuffer((2, 2, 64), np.float32))
    return t, c, b


ARG, SHAPE, ALIGN = 1, 2, 3


@pytest.mark.parametrize("code,more", [
    (SHAPE, dict(n_head=3)), (SHAPE, dict(n_head=0)), (SHAPE, dict(max_len=33)), (SHAPE, dict(seqs=70000)), (SHAPE, dict(q_stride=252)),
    (SHAPE, dict(out_stride=4)), (ALIGN, dict(q_stride=257)), (ALIGN, dict(out_stride=258)), (ARG, dict(scale=float("nan"))),
    (ARG, dict(scale=float("inf"))), (ARG, dict(k_new="n")), (ARG, dict(v_new="n")), (SHAPE, dict(k_new="n", v_new="n", new_stride=64)),
    (ALIGN, dict(k_new="n", v_new="n", new_stride=130)), (ARG, dict(k_new="n", v_new="n", history=(2, 32))), (SHAPE, dict(history=(3, 32))),
    (SHAPE, dict(history=(2, 19))), (ARG, dict(q=None)), (ARG, dict(out=None)), (ARG, dict(lens=None)), (SHAPE, dict(mask="n", mask_stride=10)),
    (ALIGN, dict(q="odd")),
])
def test_attend_refusals(gpu, code, more):
    t, c, b = small()
    a = dict(q=b["q"], out=b["out"], lens=b["lens"], seqs=2, max_len=20, n_head=4)
    a.update(more)
    for key, x in a.items():
        if x == "n":
            a[key] = b["n"]
        elif x == "odd":
            a[key] = b["q"].ptr + 4
        elif key == "history":
            a[key] = History(b["w"], b["p"], *x)
    before = b["out"].download().view(np.uint8)
    with pytest.raises(OuroError) as e:
        c.attend(**a)
    assert e.value.code == code and "ouro_kv_attend" in str(e.value)
    assert np.array_equal(b["out"].download().view(np.uint8), before)


@pytest.mark.parametrize("code,field,x", [
    (ARG, "k", None), (ARG, "v", None), (ARG, "pages", None), (ARG, "dtype", 2), (SHAPE, "n_pages", 0), (SHAPE, "max_pages", 0),
    (SHAPE, "n_head_kv", 0), (SHAPE, "head_dim", 0), (SHAPE, "head_dim", 12), (SHAPE, "head_dim", 264), (SHAPE, "page_tokens", 0),
    (SHAPE, "page_tokens", 48), (SHAPE, "page_stride", -8), (ALIGN, "token_stride", 130), (SHAPE, "token_stride", (1 << 24) + 8),
    (ALIGN, "head_stride", 4), (ALIGN, "k", "odd"),
])
def test_cache_refusals(gpu, code, field, x):
    t, c, b = small()
    setattr(c._c, field, t.kb.ptr + 2 if x == "odd" else x)
    with pytest.raises(OuroError) as e:
        c.attend(b["q"], b["out"], b["lens"], 2, 20, 4)
    assert e.value.code == code
    with pytest.raises(OuroError) as e:
        c.evict(History(b["w"], b["p"], 2, 32), b["lens"], 2, 20, 4, 1, DeviceBuffer((2,), np.int32))
    assert e.value.code == code


@pytest.mark.parametrize("code,more", [
    (SHAPE, dict(keep=0)), (SHAPE, dict(max_len=33)), (SHAPE, dict(seqs=70000)), (ARG, dict(lens=None)), (ARG, dict(lens_out=None)),
    (ARG, dict(lens_out="lens")), (SHAPE, dict(history=(2, 19))), (SHAPE, dict(history=(3, 32))), (SHAPE, dict(out=(2, 3))),
    (SHAPE, dict(out=(1, 32))), (SHAPE, dict(recent=1 << 31)),
])
def test_evict_refusals(gpu, code, more):
    t, c, b = small()
    other = DeviceBuffer((2, 2, 32), np.float32), DeviceBuffer((2, 2, 32), np.int32)
    a = dict(history=(2, 32), lens=b["lens"], seqs=2, max_len=20, keep=8, recent=2, lens_out=DeviceBuffer((2,), np.int32))
    a.update(more)
    a["history"] = History(b["w"], b["p"], *a["history"])
    if "out" in a:
        a["out"] = History(*other, *a["out"])
    if a["lens_out"] == "lens":
        a["lens_out"] = b["lens"]
    with pytest.raises(OuroError) as e:
        c.evict(**a)
    assert e.value.code == code and "ouro_kv_evict" in str(e.value)


def test_history_left_half_apart(gpu):
    t, c, b = small()
    h, mixed = History(b["w"], b["p"], 2, 32), History(b["w"], DeviceBuffer((2, 2, 32), np.int32), 2, 32)
    for out in (mixed, History(b["w"], b["p"], 2, 30)):
        with pytest.raises(OuroError) as e:
            c.evict(h, b["lens"], 2, 20, 8, 2, DeviceBuffer((2,), np.int32), out=out)
        assert e.value.code == ARG


def test_nothing_to_do(gpu):
    t, c, b = small()
    c.attend(b["q"], b["out"], b["lens"], 0, 20, 4)
    c.evict(History(b["w"], b["p"], 2, 32), b["lens"], 0, 20, 8, 2, DeviceBuffer((2,), np.int32))
