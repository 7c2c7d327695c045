"""ouro_qk_norm_rope against a float64 restatement.

Bar, U = 2^-24.  The sum of at most 256 squares takes 16 roundings in a lane and 6
across lanes, so 1 / sqrt(mean + eps) is within (22 / 2 + 4) U and a normed value
within 17 U of its size.  A cosine or sine: the rest of the turn is rounded once
(U), its series of five terms in Horner form adds 4 U and leaves out 2^-31.  The
rotated value a c - b s is therefore within (17 + 6 + 2) U (|a| + |b|); the bar is
32 U (|a| + |b|), and 32 U |x| of dims that are not rotated.  The angle's product
in 64 bits is the same on both sides.  bf16 adds its rounding, 2^-8 of the size."""
import numpy as np
import pytest
import torch

from ouroboros_amd import ops
from ouroboros_amd._lib import OuroError
from ouroboros_amd.device import DeviceBuffer
from ouroboros_amd.quant import bf16_bits_to_f32, f32_to_bf16_bits

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def enc(x, bf16):
    return f32_to_bf16_bits(np.ascontiguousarray(x, np.float32)) if bf16 else np.ascontiguousarray(x, np.float32)


def dec(x):
    return (bf16_bits_to_f32(x) if x.dtype == np.uint16 else x).astype(np.float64)


def plain(x, gain, pos, axis, freq, adjacent, eps):
    """(result, |a| + |b| of each value) of heads x [rows][heads][d]."""
    half, d = len(freq), x.shape[-1]
    if gain is not None:
        with np.errstate(invalid="ignore", divide="ignore"):
            x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * gain
    i = np.arange(half)
    one, two = (2 * i, 2 * i + 1) if adjacent else (i, i + half)
    t = (pos[axis].T.astype(np.float64) * freq.astype(np.float64))[:, None, :]
    a, b = x[..., one], x[..., two]
    out, size = x.copy(), np.abs(x)
    out[..., one], out[..., two] = a * np.cos(t) - b * np.sin(t), b * np.cos(t) + a * np.sin(t)
    size[..., one] = size[..., two] = np.abs(a) + np.abs(b)
    return out, size


def check(seed, rows, hq, hkv, d, n_rot, *, bf16=False, adjacent=False, axes=1, norm=True, gap=0, place=False, far=False,
          eps=1e-6, spoil=None):
    rng = np.random.default_rng(seed)
    half, unit = n_rot // 2, 8 if bf16 else 4
    hs = d + gap * unit  # a head's stride in the input: the gap is not read, or written in place
    strides = [h * hs + 2 * gap * unit for h in (hq, hkv)]
    raw = [enc(3.0 * rng.standard_normal((rows, s)), bf16) for s in strides]
    if spoil is not None:
        raw[0][rows // 2, 0] = enc(np.float32([spoil]), bf16)[0]
    gains = [(1 + 0.3 * rng.standard_normal(d)).astype(np.float32) if norm else None for _ in range(2)]
    pos = rng.integers(-2 ** 31, 2 ** 31 - 1, (axes, rows), dtype=np.int64) if far else rng.integers(0, 5000, (axes, rows))
    pos = pos.astype(np.int32)
    freq = (1e4 ** -(np.arange(half) / max(half, 1))).astype(np.float32)
    axis = rng.integers(0, axes, half).astype(np.int32)
    dev = [DeviceBuffer.from_host(x) for x in raw]
    outs = dev if place else [DeviceBuffer.from_host(np.full((rows, h * d + 3 * unit), 77, x.dtype)) for h, x in zip((hq, hkv), raw)]
    up = lambda x: None if x is None or not x.size else DeviceBuffer.from_host(x)
    held = [up(x) for x in (*gains, pos, freq, axis)]
    ops.qk_norm_rope(dev[0], dev[1] if hkv else None, outs[0], outs[1] if hkv else None, held[2], held[3], rows=rows, n_head=hq,
                     n_head_kv=hkv, head_dim=d, n_rot=n_rot, dtype="bf16" if bf16 else "f32", q_gain=held[0], k_gain=held[1],
                     eps=eps, axes=axes, axis=held[4] if axes > 1 else None, adjacent=adjacent, q_stride=strides[0],
                     q_head_stride=hs, k_stride=strides[1], k_head_stride=hs, q_out_stride=0 if place else hq * d + 3 * unit,
                     k_out_stride=0 if place else hkv * d + 3 * unit)
    for x, o, g, h, s in zip(raw, outs, gains, (hq, hkv), strides):
        if not h:
            continue
        heads = lambda m: np.lib.stride_tricks.as_strided(m, (rows, h, d), (m.strides[0], hs * m.itemsize, m.itemsize))
        want, size = plain(dec(heads(x)), g, pos, axis if axes > 1 else axis * 0, freq, adjacent, eps)
        y = o.download()
        if place:
            got = dec(heads(y))
            kept = y.copy()
            heads(kept)[...] = heads(x)
            assert np.array_equal(kept, x), "what lies between the heads was written"
        else:
            got = dec(y[:, :h * d].reshape(rows, h, d))
            assert (y[:, h * d:] == 77).all()
        fine = np.isfinite(want)
        assert np.array_equal(got[~fine], want[~fine], equal_nan=True)
        err = np.abs(got[fine] - want[fine])
        bar = 32 * U * size[fine] + (2.0 ** -8 * np.abs(want[fine]) if bf16 else 0)
        assert (err <= bar + 1e-37).all(), float((err / (bar + 1e-37)).max())


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("rows,hq,hkv,d,n_rot", [
    (1, 1, 0, 8, 8), (1, 16, 4, 128, 32), (3, 3, 1, 128, 128), (65, 5, 2, 80, 40), (7, 4, 4, 96, 24), (5, 2, 1, 24, 12),
    (9, 20, 1, 256, 256), (4, 3, 3, 192, 4), (6, 7, 1, 64, 0), (2049, 3, 1, 64, 64), (2050, 2, 1, 248, 100), (11, 1, 1, 16, 8)])
def test_shapes(gpu, bf16, rows, hq, hkv, d, n_rot):
    check(rows + d, rows, hq, hkv, d, n_rot, bf16=bf16)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("adjacent", [False, True])
@pytest.mark.parametrize("axes,norm,gap,place", [(3, True, 0, False), (1, False, 1, False), (2, True, 2, True), (1, True, 0, True)])
def test_forms(gpu, bf16, adjacent, axes, norm, gap, place):
    for rows, d, n_rot in ((5, 128, 64), (2051, 80, 20)):
        check(9 * axes + gap, rows, 6, 2, d, n_rot, bf16=bf16, adjacent=adjacent, axes=axes, norm=norm, gap=gap, place=place)


def test_far_positions(gpu):
    """Positions over the whole of 32 bits keep their angle."""
    check(3, 300, 2, 1, 128, 128, far=True)
    check(4, 2100, 2, 1, 64, 64, far=True, adjacent=True, axes=3)


@pytest.mark.parametrize("what", [np.nan, np.inf, 0.0])
def test_non_finite_heads(gpu, what):
    """As the formula takes them, and no other head is touched."""
    check(5, 9, 3, 1, 64, 32, spoil=what)
    check(6, 9, 3, 1, 64, 32, spoil=what, norm=False)


def test_axes_out_of_range(gpu):
    """An axis outside 0 .. axes - 1 is read as the nearest: no read outside pos."""
    rng = np.random.default_rng(8)
    x = DeviceBuffer.from_host(rng.standard_normal((4, 2, 16)).astype(np.float32))
    pos, freq = DeviceBuffer.from_host(np.arange(8, dtype=np.int32).reshape(2, 4)), DeviceBuffer.from_host(np.ones(8, np.float32))
    got = []
    for axis in ((-5, 0, 1, 9, -2 ** 31, 2 ** 31 - 1, 1, 0), (0, 0, 1, 1, 0, 1, 1, 0)):
        out = DeviceBuffer((4, 2, 16), np.float32)
        ops.qk_norm_rope(x, None, out, None, pos, freq, rows=4, n_head=2, n_head_kv=0, head_dim=16, n_rot=16, axes=2,
                         axis=DeviceBuffer.from_host(np.array(axis, np.int32)))
        got.append(out.download())
    assert np.array_equal(*got)


def test_refusals(gpu):
    x = DeviceBuffer((64,), np.float32, zero=True)
    good = dict(rows=1, n_head=1, n_head_kv=1, head_dim=16, n_rot=8)
    call = lambda q=x, k=x, qo=x, ko=x, pos=x, freq=x, **more: ops.qk_norm_rope(q, k, qo, ko, pos, freq, **{**good, **more})
    call()
    for code, more in ((1, dict(q=None)), (1, dict(k=None)), (1, dict(qo=None)), (1, dict(ko=None)), (1, dict(pos=None)),
                       (1, dict(freq=None)), (1, dict(eps=-1.0)), (1, dict(eps=float("nan"))), (1, dict(q_out_stride=20)),
                       (2, dict(head_dim=12)), (2, dict(head_dim=264)), (2, dict(head_dim=0)), (2, dict(n_rot=6)),
                       (2, dict(n_rot=20)), (2, dict(n_head=0)), (2, dict(axes=0)), (2, dict(q_stride=12)),
                       (2, dict(q_head_stride=12)), (2, dict(rows=(1 << 24) + 1)), (3, dict(q=x.ptr + 4)), (3, dict(k_stride=18))):
        with pytest.raises(OuroError) as e:
            call(**more)
        assert e.value.code == code, more
    call(q=x, k=None, ko=None, n_head_kv=0, pos=None, freq=None, n_rot=0)
    call(rows=0)
    with pytest.raises(ValueError):
        call(dtype="f16")


def test_streams_and_capture(gpu):
    """On a stream of its own and replayed from a graph with new inputs in between: the bits of the eager call."""
    g = torch.Generator().manual_seed(1)
    q, k = torch.randn(33, 8, 64, generator=g).cuda(), torch.randn(33, 2, 64, generator=g).cuda()
    pos, freq = torch.arange(33).int().cuda(), (100.0 ** -torch.linspace(0, 1, 32)).cuda()
    gain = torch.rand(64, generator=g).cuda()
    outs = [[torch.zeros_like(x) for x in (q, k)] for _ in range(2)]

    def run(o, stream):
        ops.qk_norm_rope(q.data_ptr(), k.data_ptr(), o[0].data_ptr(), o[1].data_ptr(), pos.data_ptr(), freq.data_ptr(), rows=33,
                         n_head=8, n_head_kv=2, head_dim=64, n_rot=64, q_gain=gain.data_ptr(), k_gain=gain.data_ptr(), stream=stream)

    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    run(outs[0], s.cuda_stream)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        run(outs[1], torch.cuda.current_stream().cuda_stream)
    for i in range(4):
        graph.replay()
        run(outs[0], None)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(*outs)), i
        q.mul_(-0.9).add_(0.1)
        pos.add_(100000)
        torch.cuda.synchronize()
