"""ouro_verify_drafts leaves no answer unwritten, whatever the offsets say."""
import numpy as np
import pytest

from ouroboros_amd.device import DeviceBuffer

from test_gpu_verify import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("draft", [False, True])
def test_rows_of_two_sequences(gpu, draft):
    """Offsets that fall give greedy and drawing sequences the same rows: each still gets a token or -1, and a count of its own rows."""
    B, n = 60, 4100
    c = Case(41, [2] * B, n, draft=draft, heat=[0.0 if b % 4 == 0 else 0.9 for b in range(B)])
    c.upload()
    # every other sequence has rows 3 and 4, those between them none
    cu = np.array([3 if i % 2 == 0 else 5 for i in range(B + 1)], np.int32)
    c.dev["cu"] = DeviceBuffer.from_host(cu)
    accepted, token, lens = (x.download() for x in c.run())
    has = cu[1:] > cu[:-1]
    assert np.array_equal(has, np.arange(B) % 2 == 0)
    assert ((token[has] >= -1) & (token[has] < n)).all(), token
    assert ((accepted[has] >= 0) & (accepted[has] <= 1)).all() and np.array_equal(lens[has], c.lens[has] - 1 + accepted[has])
    assert (token[~has] == -1).all() and not accepted[~has].any() and np.array_equal(lens[~has], c.lens[~has])
