"""ouro_verify_drafts against a float64 restatement.

Everything that comes back is a whole number, so it is equal or wrong; what keeps a
rounding from deciding is checked, not hoped for: the restatement gives how near a
comparison came to its border, and a case whose margin is below 1e-10 (sums in 64
bits over at most 248320 terms are within 1e-11 of each other) fails as badly
chosen.  Inputs are fixed by their seeds."""
import numpy as np
import pytest
import torch

from ouroboros_amd import ops
from ouroboros_amd._lib import OuroError
from ouroboros_amd.device import DeviceBuffer, Stream, synchronize
from ouroboros_amd.quant import bf16_bits_to_f32, f32_to_bf16_bits

pytestmark = pytest.mark.gpu


def enc(x, bf16):
    return f32_to_bf16_bits(np.ascontiguousarray(x, np.float32)) if bf16 else np.ascontiguousarray(x, np.float32)


def dec(x):
    return (bf16_bits_to_f32(x) if x.dtype == np.uint16 else x).astype(np.float64)


def softmax(x, heat=1.0):
    """Of a row; None where it has no mass."""
    x = np.where(np.isnan(x), -np.inf, x)
    m = x.max()
    if m == -np.inf:
        return None
    with np.errstate(invalid="ignore"):
        p = np.where(x == m, 1.0, np.exp((x - m) / heat))
    p[p < 2.0 ** -1000] = 0
    return p / p.sum()


def plain(logits, draft, tokens, heat, u_accept, u_next):
    """(accepted, next, margin) of one sequence's rows."""
    T, n = logits.shape
    margin, greedy = np.inf, not heat > 0
    for i in range(T):
        p = softmax(logits[i], 1.0 if greedy else heat)
        left = p
        if i + 1 < T:
            t = int(tokens[i + 1])
            known = 0 <= t < n
            if greedy:
                if known and p is not None and t == int(np.argmax(np.where(np.isnan(logits[i]), -np.inf, logits[i]))):
                    continue
            else:
                q = np.zeros(n)
                if draft is None:
                    if known:
                        q[t] = 1
                else:
                    got = softmax(draft[i])
                    q = q if got is None else got
                pt, qt = (p[t] if known and p is not None else 0.0), (q[t] if known else 0.0)
                if pt > 0 and u_accept[i] * qt > 0:  # else nothing is rounded
                    margin = min(margin, abs(u_accept[i] * qt - pt) / pt)
                if known and u_accept[i] * qt < pt:
                    continue
                if p is not None:
                    left = np.maximum(p - q, 0)
                    left = left if left.sum() > 0 else p
        if p is None:
            return i, -1, margin
        if greedy:
            return i, int(np.argmax(np.where(np.isnan(logits[i]), -np.inf, logits[i]))), margin
        sums = np.cumsum(left)
        want = u_next * sums[-1]
        at = int(np.searchsorted(sums, want, side="right"))
        if want > 0:
            margin = min(margin, np.abs(sums - want).min() / sums[-1])
        return i, at, margin
    raise AssertionError


class Case:
    """Ragged rows of logits; the drafter's are the target's with an error, its tokens drawn from them."""

    def __init__(self, seed, counts, n, *, bf16=False, draft=True, dbf16=None, error=0.4, heat=None, gap=0):
        rng = self.rng = np.random.default_rng(seed)
        self.counts, self.n, self.rows, self.B = counts, n, int(sum(counts)), len(counts)
        self.bf16, self.dbf16 = bf16, bf16 if dbf16 is None else dbf16
        self.cu = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        self.stride, self.dstride = n + gap, n + 3 * gap
        x = 2.0 * rng.standard_normal((self.rows, n))
        np.put_along_axis(x, rng.integers(0, n, (self.rows, 3)), 10.0 + rng.random((self.rows, 3)), 1)  # a few likely tokens
        y = x + error * rng.standard_normal(x.shape)
        fill = lambda z, s, half: enc(np.concatenate([z, np.full((self.rows, s - n), 1e30)], 1), half)
        self.logits, self.draft = fill(x, self.stride, self.bf16), fill(y, self.dstride, self.dbf16) if draft else None
        self.tokens = np.full(self.rows, -77, np.int32)
        drawn = y + rng.gumbel(size=y.shape)
        for b in range(self.B):
            for i in range(1, counts[b]):
                self.tokens[self.cu[b] + i] = np.argmax((x if i % 2 else drawn)[self.cu[b] + i - 1])
        self.heat = None if heat is None else np.array(heat, np.float32)
        self.u_accept, self.u_next = rng.random(self.rows, np.float32), rng.random(self.B, np.float32)
        self.lens = rng.integers(50, 90, self.B).astype(np.int32)

    def want(self):
        out = np.zeros((3, self.B), np.int32)
        for b in range(self.B):
            r = slice(self.cu[b], self.cu[b + 1])
            if not self.counts[b]:
                out[:, b] = 0, -1, self.lens[b]
                continue
            a, t, margin = plain(dec(self.logits[r, :self.n]), None if self.draft is None else dec(self.draft[r, :self.n]),
                                 self.tokens[r], 1.0 if self.heat is None else float(self.heat[b]), self.u_accept[r].astype(np.float64),
                                 float(self.u_next[b]))
            assert margin > 1e-10, (b, margin)
            out[:, b] = a, t, self.lens[b] - (self.counts[b] - 1 - a)
        return out

    def upload(self):
        up = lambda x: None if x is None else DeviceBuffer.from_host(x)
        self.dev = {k: up(getattr(self, k)) for k in ("logits", "draft", "tokens", "cu", "heat", "u_accept", "u_next", "lens")}
        return self

    def run(self, stream=None, uniform=False, workspace=None, lens=True):
        d = self.dev
        o = [DeviceBuffer.from_host(np.full(self.B, -99, np.int32)) for _ in range(3)]
        ops.verify_drafts(d["logits"], d["tokens"], d["u_accept"], d["u_next"], o[0], o[1], seqs=self.B, rows=self.rows,
                          max_new=max(self.counts, default=0), n=self.n, dtype="bf16" if self.bf16 else "f32", row_stride=self.stride,
                          cu=None if uniform else d["cu"], draft=d["draft"], draft_dtype="bf16" if self.dbf16 else "f32",
                          draft_stride=self.dstride, temperature=d["heat"], lens=d["lens"] if lens else None,
                          lens_out=o[2] if lens else None, workspace=workspace, stream=stream)
        return o

    def check(self, **more):
        got = np.stack([x.download() for x in self.upload().run(**more)])
        assert np.array_equal(got, self.want()), (got, self.want())
        return got


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("n", [1, 2, 7, 63, 1000, 8185, 8192, 8193, 32003, 65537])
def test_sizes(gpu, bf16, draft, n):
    heat = np.array([1.0, 0.7, 0.0, 1.3, 0.5, -1.0, 1.0])
    Case(n, [1, 5, 4, 3, 9, 2, 0], n, bf16=bf16, draft=draft, heat=heat).check()


@pytest.mark.parametrize("draft", [False, True])
def test_large_vocabulary(gpu, draft):
    Case(5, [5, 1, 3, 5], 248320, draft=draft, heat=[0.8, 1.0, 0.6, 0.0], error=0.5).check()


@pytest.mark.parametrize("gap", [1, 4, 5])
@pytest.mark.parametrize("bf16,dbf16", [(False, False), (True, True), (False, True), (True, False)])
def test_strides_and_types(gpu, gap, bf16, dbf16):
    """Rows that start anywhere, the drafter's otherwise than the target's and of another type."""
    Case(gap, [4, 3, 1, 6], 20001, bf16=bf16, dbf16=dbf16, gap=gap).check()


def test_all_kept_and_none(gpu):
    """A drafter that is the target keeps all whatever u; one that is nowhere near keeps none."""
    c = Case(6, [6, 6, 6], 5000, error=0.0)
    c.u_accept[:] = 0.9999
    got = c.check(uniform=True)
    assert (got[0] == 5).all()
    c = Case(7, [6, 6, 6], 5000, error=0.0)
    for r in range(c.rows):
        if r + 1 < c.rows and c.tokens[r + 1] >= 0:
            c.logits[r, c.tokens[r + 1]] = -np.inf
    got = c.check(uniform=True)
    assert (got[0] == 0).all()


def test_banned_infinite_and_nan_logits(gpu):
    """-inf and NaN hold no mass, +inf all of it; whole rows without any."""
    for draft in (False, True):
        c = Case(8, [3, 3, 3, 3, 3, 3], 4000, draft=draft, heat=[1.0, 1.0, 1.0, 0.0, 1.0, 0.0])
        rng = np.random.default_rng(1)
        c.logits[:, rng.random(4000) < 0.5] = -np.inf
        c.logits[:, rng.random(4000) < 0.1] = np.nan
        c.logits[3:6, [7, 100, 3999]] = np.inf
        c.logits[6:9] = -np.inf
        c.logits[9:12] = np.nan
        if draft:
            c.draft[12] = -np.inf
            c.draft[13] = np.nan
            c.draft[0, rng.random(c.dstride) < 0.5] = -np.inf
        got = c.check()
        assert got[1, 2] == -1 and got[1, 3] == -1 and got[1, 1] in (7, 100, 3999)


def test_tokens_outside_the_vocabulary(gpu):
    c = Case(9, [3, 3, 3, 3], 300, draft=True, heat=[1.0, 0.0, 1.0, 1.0])
    c.tokens[[1, 4, 7, 10]] = [-1, 300, 1 << 30, -(1 << 31)]
    got = c.check()
    assert (got[0] == 0).all()
    Case.check(c)
    c.draft = None
    c.check()


def test_ends_of_u(gpu):
    """u' = 0 takes the first token that has any weight, the largest below 1 the last with its share; u = 0 keeps whatever p can be."""
    for draft in (False, True):
        c = Case(10, [2, 2, 1, 1], 9000, draft=draft)
        c.logits[:, :11] = -np.inf
        c.logits[:, 8990:] = -np.inf
        c.u_next[:] = [0, np.nextafter(np.float32(1), np.float32(0)), 0, np.nextafter(np.float32(1), np.float32(0))]
        c.u_accept[:] = 0
        for b in (0, 1):
            c.tokens[c.cu[b] + 1] = 20 + b
        got = c.check()
        assert (got[0, :2] == 1).all() and (got[1, [0, 2]] == 11).all() and (got[1] >= 11).all() and (got[1] < 8990).all()


def test_nothing_left(gpu):
    """u = 1, which a caller should not give, refuses a token of equal p and q; with nothing left of p - q the next is drawn from p."""
    c = Case(11, [2, 2], 700, error=0.0)
    c.u_accept[:] = 1.0
    got = np.stack([x.download() for x in c.upload().run()])
    for b in range(2):
        p = softmax(dec(c.logits[c.cu[b]]))
        assert got[0, b] == 0 and got[1, b] == np.searchsorted(np.cumsum(p), float(c.u_next[b]), side="right")


def test_the_answer_is_the_targets(gpu):
    """Over many draws the first token of an answer falls on each token as often as
    the target's p says, drafted or drawn.  8 tokens, 40000 sequences: the largest
    share is off by at most 5 sigma = 5 sqrt(p (1 - p) / 40000) <= 0.0125 but for
    one seed in a million; the seed is fixed."""
    rng = np.random.default_rng(12)
    B, n = 40000, 8
    p_logits, q_logits = rng.standard_normal(n), rng.standard_normal(n)
    c = Case(12, [2] * B, n, error=0.0)
    c.logits[:], c.draft[:] = p_logits, q_logits
    c.tokens[1::2] = rng.choice(n, B, p=softmax(c.draft[0].astype(np.float64)))
    accepted, token, _ = (x.download() for x in c.upload().run(uniform=True))
    first = np.where(accepted == 1, c.tokens[1::2], token)
    share = np.bincount(first, minlength=n) / B
    assert np.abs(share - softmax(c.logits[0].astype(np.float64))).max() < 0.0125


def test_cu_out_of_range(gpu):
    """Offsets past the rows and counts above max_new are held to them."""
    c = Case(13, [3, 3, 3], 500)
    c.upload()
    c.cu = np.array([-4, 3, 3, 1 << 30], np.int32)
    c.dev["cu"] = DeviceBuffer.from_host(c.cu)
    got = [x.download() for x in c.run()]
    c.counts, c.cu = [3, 0, 3], np.array([0, 3, 3, 6], np.int32)
    want = np.zeros((3, 3), np.int32)
    for b, first in ((0, 0), (2, 3)):
        r = slice(first, first + 3)
        a, t, margin = plain(dec(c.logits[r]), dec(c.draft[r]), c.tokens[r], 1.0, c.u_accept[r], float(c.u_next[b]))
        assert margin > 1e-10
        want[:, b] = a, t, c.lens[b] - (2 - a)
    want[:, 1] = 0, -1, c.lens[1]
    assert np.array_equal(np.stack(got), want)


def test_optional_arguments(gpu):
    """Without lens, with a workspace of its own, lens_out over lens, no sequences, no rows."""
    c = Case(14, [3, 1, 4], 3000)
    want = c.want()
    ws = DeviceBuffer((ops.verify_workspace_bytes(3, 8, 3000),), np.uint8)
    got = [x.download() for x in c.upload().run(workspace=ws, lens=False)]
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1]) and (got[2] == -99).all()
    d = c.dev
    ops.verify_drafts(d["logits"], d["tokens"], d["u_accept"], d["u_next"], *(DeviceBuffer((3,), np.int32) for _ in range(2)), seqs=3,
                      rows=8, max_new=4, n=3000, cu=d["cu"], draft=d["draft"], lens=d["lens"], lens_out=d["lens"])
    assert np.array_equal(d["lens"].download(), want[2])
    Case(15, [0, 0], 100).check()


def test_refusals(gpu):
    b = DeviceBuffer((4096,), np.uint8, zero=True)
    good = dict(seqs=1, rows=2, max_new=2, n=64)
    call = lambda x=b, t=b, ua=b, un=b, acc=b, nxt=b, **more: ops.verify_drafts(x, t, ua, un, acc, nxt, **{**good, **more})
    for code, more in ((1, dict(x=None)), (1, dict(t=None)), (1, dict(ua=None)), (1, dict(un=None)), (1, dict(acc=None)),
                       (1, dict(nxt=None)), (1, dict(lens_out=b)), (2, dict(n=0)), (2, dict(n=1 << 24)), (2, dict(rows=3)),
                       (2, dict(seqs=70000, rows=140000)), (2, dict(rows=40000, max_new=40000)),
                       (2, dict(row_stride=63)), (2, dict(draft=b, draft_stride=63)), (3, dict(x=b.ptr + 2)),
                       (3, dict(draft=b.ptr + 2)), (3, dict(dtype="bf16", x=b.ptr + 1))):
        with pytest.raises(OuroError) as e:
            call(**more)
        assert e.value.code == code, more
    with pytest.raises(ValueError):
        call(dtype="f16")
    call(seqs=0, rows=0, max_new=0)


def test_two_streams_in_flight(gpu):
    """Calls of both streams queued in turn, small ones ahead of larger ones so that the scratch grows between them."""
    calls = [[Case(20 + 2 * i + j, counts, 30000, heat=None).upload() for j, counts in enumerate(([2], [6] * 20))] for i in range(2)]
    streams = [Stream(), Stream()]
    synchronize()
    got = [[], []]
    for j in range(2):
        for _ in range(5):
            for i in range(2):
                got[i].append((j, calls[i][j].run(streams[i].handle)))
    for s in streams:
        s.synchronize()
    for i in range(2):
        want = [c.want() for c in calls[i]]
        for j, o in got[i]:
            assert np.array_equal(np.stack([x.download() for x in o]), want[j]), (i, j)


def test_captured(gpu):
    """Replays with new inputs in between: the eager call's tokens."""
    g = torch.Generator(device="cuda").manual_seed(2)
    rows, n, B = 12, 20000, 4
    x, y = (2.5 * torch.randn(rows, n, generator=g, device="cuda") for _ in range(2))
    tokens = torch.randint(0, n, (rows,), generator=g, device="cuda").int()
    u, v = torch.rand(rows, generator=g, device="cuda"), torch.rand(B, generator=g, device="cuda")
    lens = torch.full((B,), 40).int().cuda()
    outs = [[torch.zeros(B).int().cuda() for _ in range(3)] for _ in range(2)]
    scratch = [torch.zeros(ops.verify_workspace_bytes(B, rows, n), dtype=torch.uint8).cuda() for _ in range(2)]

    def run(i, stream):
        p = lambda t: t.data_ptr()
        ops.verify_drafts(p(x), p(tokens), p(u), p(v), p(outs[i][0]), p(outs[i][1]), seqs=B, rows=rows, max_new=3, n=n, draft=p(y),
                          lens=p(lens), lens_out=p(outs[i][2]), workspace=p(scratch[i]), stream=stream)

    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    run(0, s.cuda_stream)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        run(1, torch.cuda.current_stream().cuda_stream)
    seen = set()
    for i in range(5):
        graph.replay()
        run(0, None)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(*outs)), i
        seen.add(tuple(outs[0][1].tolist()))
        tokens.copy_(torch.argmax(x + (3 - i) * torch.randn(rows, n, generator=g, device="cuda"), 1).int().roll(1))
        for t in (u, v):
            t.copy_(torch.rand(t.shape, generator=g, device="cuda"))
        torch.cuda.synchronize()
    assert len(seen) > 1
