"""ouro_kv_attend's bf16 outputs are its fp32 outputs rounded once.

With queries that bf16 holds, a call with bf16 rows and one with fp32 rows have
the same scores, and both hold the softmax weights in fp32: nothing but the
last rounding may differ, so the bf16 output is the fp32 one rounded to nearest
even, bit for bit."""
import numpy as np
import pytest

from ouroboros_amd.device import DeviceBuffer
from ouroboros_amd.quant import f32_to_bf16_bits

from test_gpu_kv_cache import Setup, dec, enc, name

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cache", [True, False])
@pytest.mark.parametrize("lens,hq,hkv,d", [((1, 40, 255), 4, 2, 128), ((2000, 700, 0), 32, 2, 64), ((900, 300), 6, 2, 192)])
def test_rounded_once(gpu, cache, lens, hq, hkv, d):
    t = Setup(d, lens, hkv, d, 32, cache)
    c = t.open()
    B = len(lens)
    q, gate = (enc(t.rng.standard_normal((B, hq, d)), True) for _ in range(2))
    lens_b = DeviceBuffer.from_host(t.lens)
    got = {}
    for io in (False, True):
        rows = [DeviceBuffer.from_host(x if io else dec(x)) for x in (q, gate)]
        out, lse = DeviceBuffer((B, hq, d), np.uint16 if io else np.float32), DeviceBuffer((B, hq), np.float32)
        c.attend(rows[0], out, lens_b, B, t.max_len, hq, dtype=name(io), gate=rows[1], lse=lse)
        got[io] = out.download(), lse.download()
    assert np.array_equal(got[True][0], f32_to_bf16_bits(got[False][0]))
    assert np.array_equal(got[True][1], got[False][1])
