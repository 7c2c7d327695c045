"""A paged cache of 8-bit codes: ouro_kv8_write and ouro_kv8_read against plain
restatements, bit for bit.

The scale is a power of two, so x / scale is exact and its nearest integer has no
room for rounding: codes and scales are compared as they are.  Read back, code *
scale is exact in both types."""
import numpy as np
import pytest

from ouroboros_amd._lib import OuroError
from ouroboros_amd.device import DeviceBuffer
from ouroboros_amd.kvcache import KVCache8
from ouroboros_amd.quant import bf16_bits_to_f32, f32_to_bf16_bits

pytestmark = pytest.mark.gpu


def enc(x, bf16):
    return f32_to_bf16_bits(np.ascontiguousarray(x, np.float32)) if bf16 else np.ascontiguousarray(x, np.float32)


def dec(x):
    return (bf16_bits_to_f32(x) if x.dtype == np.uint16 else x).astype(np.float64)


def name(bf16):
    return "bf16" if bf16 else "f32"


def scale_for(m):
    """The smallest power of two s with m <= 127 s, at least 2^-126; 0 for 0."""
    if m == 0:
        return 0.0
    s = 2.0 ** -126
    e = np.floor(np.log2(m)) - 8
    s = max(s, 2.0 ** e)
    while m > 127 * s:
        s *= 2
    return s


class Cache8:
    """Pools whose unused codes are anything and whose unused scales are NaN, with
    a host copy that `write` keeps as the definition says."""

    def __init__(self, seed, seqs, slots, hkv, d, page, block, layout="token", holes=(), gap=0, spare=2):
        rng = self.rng = np.random.default_rng(seed)
        self.hkv, self.d, self.page, self.block, self.layout, self.slots = hkv, d, page, block, layout, slots
        self.maxp = -(-max(slots, 1) // page)
        self.n_pages = seqs * self.maxp + spare
        self.table = rng.permutation(self.n_pages)[:seqs * self.maxp].astype(np.int32).reshape(seqs, self.maxp)
        for b, p, what in holes:
            self.table[b, p] = what
        row = d + 16 * gap
        shape = (self.n_pages, hkv, page, row) if layout == "head" else (self.n_pages, page, hkv, row)
        self.strides = (hkv * page * row, row, page * row) if layout == "head" else (hkv * page * row, hkv * row, row)
        self.codes = [rng.integers(-128, 128, shape).astype(np.int8) for _ in range(2)]
        self.scales = [np.full((self.n_pages, page // block, hkv), np.nan, np.float32) for _ in range(2)]

    def view(self, pool):
        x = pool.transpose(0, 2, 1, 3) if self.layout == "head" else pool
        return x[..., :self.d]

    def open(self):
        self.dev = [DeviceBuffer.from_host(x) for x in (*self.codes, *self.scales, self.table)]
        self.c = KVCache8(*self.dev, n_pages=self.n_pages, max_pages=self.maxp, page_tokens=self.page, block_tokens=self.block,
                          n_head_kv=self.hkv, head_dim=self.d, strides=self.strides)
        return self.c

    def at(self, b, j):
        """(page, token) of a slot, None of a hole."""
        p = int(self.table[b, j // self.page])
        return (p, j % self.page) if 0 <= p < self.n_pages else None

    def write(self, new, lens, counts, firsts):
        """new: [k, v] rows [rows][hkv][d] float64."""
        for b, (n, t, first) in enumerate(zip(lens, counts, firsts)):
            n = min(max(n, 0), self.maxp * self.page)
            start = n - t
            for j0 in range(max(start, 0) // self.block * self.block, n, self.block):
                lo, hi = max(start, 0, j0), min(n, j0 + self.block)
                where = self.at(b, j0)
                if where is None or lo >= hi:
                    continue
                p, t0 = where
                for pool, scales, rows in zip(self.codes, self.scales, new):
                    x = rows[first + lo - start:first + hi - start]
                    codes = self.view(pool)[p, t0:t0 + self.block]
                    for h in range(self.hkv):
                        v = x[:, h]
                        s = scale_for(np.abs(np.where(np.isfinite(v), v, 0)).max())
                        if lo > j0:
                            before = float(scales[p, t0 // self.block, h])
                            s = max(s, before)
                            if s != before:
                                codes[:lo - j0, h] = np.rint(codes[:lo - j0, h].astype(np.float64) * (before / s))
                        with np.errstate(invalid="ignore"):
                            q = np.clip(np.rint(v / s), -127, 127) if s else np.zeros_like(v)
                        codes[lo - j0:hi - j0, h] = np.where(np.isnan(v), 0, q)
                        scales[p, t0 // self.block, h] = s

    def same(self):
        for x, y in zip((*self.codes, *self.scales), self.dev[:4]):
            got = y.download()
            assert np.array_equal(got.view(np.uint8), x.view(np.uint8)), int((got != x).sum())

    def values(self, b, lo, hi):
        """[k, v] of slots lo .. hi - 1 in float64 [slots][hkv][d], and which have a page."""
        k, v = (np.zeros((hi - lo, self.hkv, self.d)) for _ in range(2))
        there = np.zeros(hi - lo, bool)
        for j in range(max(lo, 0), hi):
            where = self.at(b, j)
            if where is not None:
                p, t = where
                there[j - lo] = True
                for out, pool, scales in zip((k, v), self.codes, self.scales):
                    out[j - lo] = self.view(pool)[p, t].astype(np.float64) * scales[p, t // self.block][:, None].astype(np.float64)
        return k, v, there

    def fill(self, lens, size=1.0):
        """Slots 0 .. lens[b] - 1 hold codes over their whole range and scales of unlike size."""
        rng = self.rng
        for b, n in enumerate(lens):
            for j0 in range(0, n, self.block):
                where = self.at(b, j0)
                if where is not None:
                    for pool, scales in zip(self.codes, self.scales):
                        self.view(pool)[where[0], where[1]:where[1] + self.block] = np.clip(
                            np.rint(40 * rng.standard_normal((self.block, self.hkv, self.d))), -127, 127)
                        scales[where[0], where[1] // self.block] = size * 2.0 ** rng.integers(-8, -3, self.hkv)


def packed(rng, counts, hkv, d, bf16, extra=0, size=1.0):
    """Rows of unlike size with `extra` values between them, their offsets, and [rows][hkv][d] float64."""
    rows = int(sum(counts))
    unit = 8 if bf16 else 4
    stride = hkv * d + extra * unit
    raw = [enc(rng.standard_normal((rows + 1, stride)) * np.exp(size * rng.standard_normal((rows + 1, 1))), bf16) for _ in range(2)]
    cu = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    return raw, stride, cu, [dec(x[:rows, :hkv * d]).reshape(rows, hkv, d) for x in raw]


def check_write(seed, steps, hkv, d, page, block, *, bf16=False, layout="token", holes=(), gap=0, extra=0, uniform=False, spoil=()):
    """steps: a list of (lens, counts), written one after another."""
    seqs, slots = len(steps[0][0]), max(max(lens) for lens, _ in steps)
    t = Cache8(seed, seqs, slots, hkv, d, page, block, layout, holes, gap)
    c = t.open()
    for lens, counts in steps:
        raw, stride, cu, new = packed(t.rng, counts, hkv, d, bf16, extra, 1.0)
        for row, value in spoil:
            if row < cu[-1]:
                for x, y in zip(raw, new):
                    x[row, 1:1 + len(value)] = enc(np.float32(value), bf16)
                    y[row].reshape(-1)[1:1 + len(value)] = dec(enc(np.float32(value), bf16))
        lens_b, cu_b = DeviceBuffer.from_host(np.array(lens, np.int32)), DeviceBuffer.from_host(cu)
        kb, vb = (DeviceBuffer.from_host(x) for x in raw)
        most = max(counts)
        c.write(kb, vb, lens_b, seqs, int(cu[-1]), most, cu=None if uniform and min(counts) == most else cu_b, dtype=name(bf16),
                new_stride=stride if extra else 0)
        t.write(new, lens, counts, cu[:-1])
        t.same()
    return t


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("hkv,d,page,block,layout", [(1, 16, 16, 16, "token"), (4, 128, 64, 64, "token"), (2, 80, 32, 16, "head"),
                                                     (3, 96, 128, 128, "head"), (1, 256, 256, 256, "token"), (2, 192, 64, 32, "token")])
def test_prompts_then_steps(gpu, bf16, hkv, d, page, block, layout):
    """Ragged prompts that end inside, at and past blocks, then single tokens and a few at once, one sequence at rest."""
    lens = np.array([1, block - 1, block, block + 1, 3 * block + 5])
    steps = [(lens, lens)]
    for counts in ([1, 1, 1, 1, 1], [1, 1, 1, 1, 0], [4, 2, 1, 3, 6]):
        lens = lens + counts
        steps.append((lens, counts))
    check_write(d + block, steps, hkv, d, page, block, bf16=bf16, layout=layout)


def test_uniform_rows_and_gaps(gpu):
    check_write(1, [((17, 34), (17, 34)), ((20, 37), (3, 3)), ((21, 38), (1, 1))], 2, 64, 32, 16, uniform=True)
    check_write(2, [((20, 30), (20, 30)), ((20, 37), (0, 7)), ((21, 38), (1, 1))], 2, 48, 32, 16, gap=1, extra=2, bf16=True)


def test_holes_are_dropped(gpu):
    check_write(3, [((70, 20), (70, 20)), ((70, 70), (0, 50)), ((71, 71), (1, 1))], 2, 64, 16, 16, holes=((0, 1, -1), (1, 3, 1 << 20), (0, 4, -7)))


@pytest.mark.parametrize("bf16", [False, True])
def test_not_numbers(gpu, bf16):
    """NaN as 0, infinities as the ends, and no part in the scale; rows of them alone, of zeros, of the smallest and largest numbers."""
    spoil = [(0, [np.nan, np.inf, -np.inf]), (3, [0.0] * 63), (5, [np.inf] * 63), (6, [3e38, -3e38]), (20, [1e-45, 1e-38])]
    check_write(4, [((8, 40), (8, 40)), ((9, 41), (1, 1)), ((10, 56), (1, 15))], 1, 64, 16, 16, bf16=bf16, spoil=spoil)
    t = Cache8(5, 1, 16, 1, 16, 16, 16)
    c = t.open()
    for n, row in ((1, [0.0] * 16), (2, [np.inf] + [0.0] * 15), (3, [1e-44] * 16), (4, [2.0 ** -119] * 16), (5, [1.0] * 16)):
        x = enc(np.float32([row]), bf16)
        b = DeviceBuffer.from_host(x)
        c.write(b, b, DeviceBuffer.from_host(np.array([n], np.int32)), 1, 1, 1, dtype=name(bf16))
        t.write([dec(x).reshape(1, 1, 16)] * 2, [n], [1], [0])
        t.same()


def test_scale_at_its_borders(gpu):
    """127 s is held with s, the next number above it with 2 s."""
    for e in (-20, 0, 13):
        for m in (127.0, np.nextafter(np.float32(127), np.float32(200)), 128.0, 63.5, np.nextafter(np.float32(63.5), np.float32(0))):
            t = Cache8(6, 1, 16, 1, 16, 16, 16)
            c = t.open()
            x = np.zeros((1, 16), np.float32)
            x[0, :3] = np.float32(m) * np.float32(2.0 ** e) * np.float32([1, -0.5, 0.25])
            b = DeviceBuffer.from_host(x)
            c.write(b, b, DeviceBuffer.from_host(np.array([1], np.int32)), 1, 1, 1)
            t.write([x.astype(np.float64).reshape(1, 1, 16)] * 2, [1], [1], [0])
            t.same()
            assert t.scales[0][t.table[0, 0], 0, 0] == (2.0 ** e if 63.5 < m <= 127 else 2.0 ** (e + 1) if m > 127 else 2.0 ** (e - 1))


def test_rows_that_come_one_at_a_time(gpu):
    """Tokens of growing size written singly: the scale is that of all at once, and
    every held value is within one step of the written one: the roundings at steps
    that at least double add up to less than the last step."""
    rng = np.random.default_rng(9)
    n, d = 64, 64
    x = (rng.standard_normal((n, 1, d)) * 1.15 ** np.arange(n)[:, None, None]).astype(np.float32)
    once, singly = (Cache8(10, 1, n, 1, d, 64, 64) for _ in range(2))
    a, b = once.open(), singly.open()
    xb = DeviceBuffer.from_host(x)
    lens = [DeviceBuffer.from_host(np.array([i + 1], np.int32)) for i in range(n)]
    a.write(xb, xb, lens[-1], 1, n, n)
    for i in range(n):
        b.write(xb.ptr + 4 * d * i, xb.ptr + 4 * d * i, lens[i], 1, 1, 1)
    outs = []
    for c in (a, b):
        o = DeviceBuffer((n, 1, d), np.float32)
        c.read(o, None, lens[-1], 1, n, n)
        outs.append(o.download().astype(np.float64))
    scale = [t.dev[2].download()[t.table[0, 0]] for t in (once, singly)]
    assert np.array_equal(*scale)
    step = float(scale[0][0, 0])
    assert (np.abs(outs[0] - x) <= step / 2).all()
    assert (np.abs(outs[1] - x) < step).all()
    assert not np.array_equal(*outs)  # the older rows did suffer more than one rounding


def test_rows_taken_back(gpu):
    """Drafted rows that are refused: the next rows go over them, in the blocks that are still held the scale stays grown."""
    t = Cache8(11, 2, 80, 2, 64, 32, 32)
    c = t.open()
    for lens, counts, size in (((30, 32), (30, 32), 0.1), ((35, 36), (5, 4), 3.0), ((32, 33), (1, 1), 0.1), ((36, 40), (4, 7), 0.1)):
        raw, _, cu, new = packed(t.rng, counts, 2, 64, False, size=size)
        c.write(*(DeviceBuffer.from_host(x) for x in raw), DeviceBuffer.from_host(np.array(lens, np.int32)), 2, int(cu[-1]),
                max(counts), cu=DeviceBuffer.from_host(cu))
        t.write(new, lens, counts, cu[:-1])
        t.same()


def test_numbers_out_of_range(gpu):
    """Lengths, offsets and counts past what the call may touch are held to it."""
    t = Cache8(12, 3, 64, 1, 32, 16, 16)
    t.fill([64, 0, 0])
    c = t.open()
    raw, _, _, new = packed(t.rng, [3, 3, 3], 1, 32, False)
    kb, vb = (DeviceBuffer.from_host(x) for x in raw)
    # lens: past the table, below 0, fewer slots than rows; cu: below 0 and past the rows; counts above max_new
    lens, cu = np.array([1 << 30, -5, 2], np.int32), np.array([-9, 3, 3, 1 << 30], np.int32)
    c.write(kb, vb, DeviceBuffer.from_host(lens), 3, 9, 3, cu=DeviceBuffer.from_host(cu))
    t.write(new, [64, 0, 2], [3, 0, 3], [0, 3, 3])
    t.same()
    out = [DeviceBuffer.from_host(np.full((9, 32), 5, np.float32)) for _ in range(2)]
    c.read(*out, DeviceBuffer.from_host(lens), 3, 9, 3, cu=DeviceBuffer.from_host(cu))
    want = [np.full((9, 32), 5.0) for _ in range(2)]
    for b, (n, first, count) in enumerate(((64, 0, 3), (0, 3, 0), (2, 3, 3))):
        for w, v in zip(want, t.values(b, n - count, n)[:2]):
            w[first:first + count] = v[:, 0]
    for o, w in zip(out, want):
        assert np.array_equal(o.download(), w.astype(np.float32))


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("hkv,d,page,block,layout,gap", [(4, 128, 64, 64, "token", 0), (1, 16, 16, 16, "head", 0), (3, 80, 64, 16, "head", 1),
                                                         (17, 256, 32, 32, "token", 0), (2, 96, 256, 128, "token", 2)])
def test_read(gpu, bf16, hkv, d, page, block, layout, gap):
    lens, counts = [5, 100, 0, 70, 33], [5, 100, 0, 9, 1]
    t = Cache8(d, 5, 100, hkv, d, page, block, layout, gap=gap, holes=((1, 0, -1),))
    t.fill(lens)
    c = t.open()
    cu = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    rows, unit = int(cu[-1]), 8 if bf16 else 4
    for stride in (0, hkv * d + unit):
        out = [DeviceBuffer.from_host(np.full((rows + 2, stride or hkv * d), 9, np.uint16 if bf16 else np.float32)) for _ in range(2)]
        c.read(*out, DeviceBuffer.from_host(np.array(lens, np.int32)), 5, rows, 100, cu=DeviceBuffer.from_host(cu), dtype=name(bf16),
               out_stride=stride)
        for i, o in enumerate(out):
            got = o.download()
            want = np.full(got.shape, 9, got.dtype)
            for b, (n, m) in enumerate(zip(lens, counts)):
                want[cu[b]:cu[b + 1], :hkv * d] = enc(t.values(b, n - m, n)[i].reshape(m, hkv * d), bf16)
            assert np.array_equal(got, want)
    one = DeviceBuffer((rows, hkv * d), np.uint16 if bf16 else np.float32)
    c.read(None, one, DeviceBuffer.from_host(np.array(lens, np.int32)), 5, rows, 100, cu=DeviceBuffer.from_host(cu), dtype=name(bf16))
    assert np.array_equal(one.download(), out[1].download()[:rows, :hkv * d])


def test_large_offsets(gpu):
    """Pages past 2^32 bytes into the pool: pools of 4.8 GB, one page at the far end."""
    page, d = 256, 256
    n_pages = (1 << 32) // (page * d) + 8000
    k, v = (DeviceBuffer((n_pages, page * d), np.int8) for _ in range(2))
    ks, vs = (DeviceBuffer((n_pages, 1, 1), np.float32, zero=True) for _ in range(2))
    table = DeviceBuffer.from_host(np.array([[n_pages - 1]], np.int32))
    c = KVCache8(k, v, ks, vs, table, n_pages=n_pages, max_pages=1, page_tokens=page, block_tokens=page, n_head_kv=1, head_dim=d)
    x = np.random.default_rng(3).integers(-127, 128, (page, d)).astype(np.float32)
    x[:, 0] = 127
    xb, lens = DeviceBuffer.from_host(x), DeviceBuffer.from_host(np.array([page], np.int32))
    c.write(xb, xb, lens, 1, page, page)
    out = [DeviceBuffer((page, d), np.float32) for _ in range(2)]
    c.read(*out, lens, 1, page, page)
    assert all(np.array_equal(o.download(), x) for o in out)
    assert ks.download()[n_pages - 1] == 1.0 and not ks.download()[:n_pages - 1].any()


def test_refusals(gpu):
    b = DeviceBuffer((1 << 16,), np.uint8, zero=True)
    good = dict(n_pages=2, max_pages=2, page_tokens=16, block_tokens=16, n_head_kv=2, head_dim=32)

    def call(what="write", k=b, v=b, ks=b, pages=b, rows=2, new=1, seqs=2, lens=b, x=b, cu=None, dtype="f32", stride=0, **more):
        c = KVCache8(k, v, ks, b, pages, **{**good, **more})
        if what == "write":
            c.write(x, b, lens, seqs, rows, new, cu=cu, dtype=dtype, new_stride=stride)
        else:
            c.read(x, b, lens, seqs, rows, new, cu=cu, dtype=dtype, out_stride=stride)

    bad = [(1, dict(k=None)), (1, dict(v=None)), (1, dict(ks=None)), (1, dict(pages=None)), (1, dict(lens=None)),
           (2, dict(n_pages=0)), (2, dict(max_pages=0)), (2, dict(n_head_kv=0)), (2, dict(n_head_kv=40000)), (2, dict(head_dim=8)),
           (2, dict(head_dim=24)), (2, dict(head_dim=272)), (2, dict(page_tokens=8)), (2, dict(page_tokens=48)),
           (2, dict(page_tokens=1 << 21)), (2, dict(block_tokens=8)), (2, dict(block_tokens=32)),
           (2, dict(page_tokens=512, block_tokens=512)), (2, dict(page_tokens=64, block_tokens=48)), (2, dict(seqs=70000, rows=70000)),
           (2, dict(rows=3)), (2, dict(rows=(1 << 23) + 1, cu=b)), (2, dict(stride=60)),
           (2, dict(strides=(-16, 64, 32))), (2, dict(strides=(1024, 1 << 25, 32))), (3, dict(strides=(1024, 72, 32))),
           (3, dict(k=b.ptr + 8)), (3, dict(ks=b.ptr + 2)), (3, dict(x=b.ptr + 4)), (3, dict(stride=66))]
    for code, more in bad:
        for what in ("write", "read"):
            with pytest.raises(OuroError) as e:
                call(what, **more)
            assert e.value.code == code, (what, more)
    with pytest.raises(OuroError) as e:
        call("write", x=None)
    assert e.value.code == 1
    with pytest.raises(ValueError):
        call(dtype="f16")
    with pytest.raises(ValueError):
        call(layout="page")
    call(seqs=0, rows=0, new=0)
    call("read", seqs=0, rows=0, new=0)
