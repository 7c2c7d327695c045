"""ouro_kv8_attend refuses strides that no array has, as its neighbours do."""
import numpy as np
import pytest

from ouroboros_amd._lib import OuroError
from ouroboros_amd.device import DeviceBuffer
from ouroboros_amd.kvcache import KVCache8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("more", [dict(q_stride=(1 << 40) + 8), dict(out_stride=1 << 63), dict(q_stride=(1 << 64) - 8), dict(mask_stride=1 << 62)])
def test_strides_past_any_array(gpu, more):
    b = DeviceBuffer((1 << 16,), np.uint8, zero=True)
    c = KVCache8(b, b, b, b, b, n_pages=2, max_pages=2, page_tokens=16, block_tokens=16, n_head_kv=2, head_dim=32)
    with pytest.raises(OuroError) as e:
        c.attend(b, b, b, 2, 2, 1, 32, 4, mask=b, **more)
    assert e.value.code == 2
