"""Attention over a paged cache, eviction and token log probabilities on two
streams with work of both in flight: inputs and outputs are made first, the
calls are queued in turn without a wait, each stream with the library's own
scratch, small calls ahead of larger ones so that the scratch grows between
them, and only then are the streams waited for.  Every result equals, bit for
bit, that of the same call alone on the null stream."""
import numpy as np
import pytest

from ouroboros_amd import _lib, ops
from ouroboros_amd.device import DeviceBuffer, Stream, synchronize
from ouroboros_amd.kvcache import History, KVCache, attend_workspace_bytes, evict_workspace_bytes

from test_gpu_kv_cache import Setup, enc

pytestmark = pytest.mark.gpu
ROUNDS = 6


class Attend:
    """`seqs` sequences of a cache of 48, with a history."""

    def __init__(self, seed, seqs):
        rng = np.random.default_rng(seed)
        lens = rng.integers(1, 4001, 48)
        lens[0] = 4000
        t = self.t = Setup(seed, (1,), 2, 64, 64, True, max_len=64 * 64)
        t.k, t.v = (enc(rng.standard_normal(t.k.shape), True) for _ in range(2))
        t.open()
        table = rng.integers(0, t.n_pages, (48, 64)).astype(np.int32)  # pages shared by sequences: nothing is written
        self.pb = DeviceBuffer.from_host(table)
        self.c = KVCache(t.kb, t.vb, self.pb, n_pages=t.n_pages, max_pages=64, page_tokens=64, n_head_kv=2, head_dim=64)
        self.seqs = seqs
        self.q = DeviceBuffer.from_host(rng.standard_normal((48, 8, 64)).astype(np.float32))
        self.lens = DeviceBuffer.from_host(lens.astype(np.int32))
        self.pos = DeviceBuffer((48, 2, 4000), np.int32, zero=True)

    def outputs(self):
        return {"out": DeviceBuffer((self.seqs, 8, 64), np.float32, zero=True), "lse": DeviceBuffer((self.seqs, 8), np.float32, zero=True),
                "weight": DeviceBuffer((self.seqs, 2, 4000), np.float32, zero=True)}

    def run(self, o, stream):
        self.c.attend(self.q, o["out"], self.lens, self.seqs, 4000, 8, history=History(o["weight"], self.pos, 2, 4000), lse=o["lse"], stream=stream)


class Evict:
    """More moves than the choosing workgroup makes itself; the history left is apart, so that a call can be made again."""

    def __init__(self, seed, seqs):
        rng = np.random.default_rng(seed)
        self.t = t = Setup(seed, (0,) * seqs, 2, 64, 64, True, max_len=1200)
        t.k, t.v = (enc(rng.standard_normal(t.k.shape), True) for _ in range(2))
        self.c, self.seqs = t.open(), seqs
        w = np.exp(rng.standard_normal((seqs, 2, 1200))).astype(np.float32)
        pos = np.broadcast_to(np.arange(1200, dtype=np.int32), w.shape)
        self.hist = History(DeviceBuffer.from_host(w), DeviceBuffer.from_host(pos), 2, 1200)
        self.lens = DeviceBuffer.from_host(np.full(seqs, 1200, np.int32))

    def outputs(self):
        return {"weight": DeviceBuffer((self.seqs, 2, 560), np.float32, zero=True), "pos": DeviceBuffer((self.seqs, 2, 560), np.int32, zero=True),
                "left": DeviceBuffer((self.seqs,), np.int32, zero=True), "k": self.t.kb, "v": self.t.vb}

    def run(self, o, stream):
        self.c.evict(self.hist, self.lens, self.seqs, 1200, 560, 40, o["left"], out=History(o["weight"], o["pos"], 2, 560), stream=stream)


class Logprobs:
    def __init__(self, seed, rows):
        rng = np.random.default_rng(seed)
        self.rows, self.n = rows, 500
        self.x = DeviceBuffer.from_host(rng.standard_normal((rows, self.n)).astype(np.float32))
        self.t = DeviceBuffer.from_host(rng.integers(0, self.n, rows).astype(np.int32))

    def outputs(self):
        f = {name: DeviceBuffer((self.rows,), np.float32, zero=True) for name in ("logprob", "entropy", "lse")}
        return {**f, "rank": DeviceBuffer((self.rows,), np.int32, zero=True), "top_id": DeviceBuffer((self.rows, 9), np.int32, zero=True),
                "top_logprob": DeviceBuffer((self.rows, 9), np.float32, zero=True)}

    def run(self, o, stream):
        ops.token_logprobs(self.x, self.rows, self.n, targets=self.t, k=9, stream=stream, **o)


@pytest.mark.parametrize("kind,sizes", [(Attend, (2, 48)), (Evict, (2, 200)), (Logprobs, (3, 9000))])
def test_two_streams_in_flight(gpu, kind, sizes):
    calls = [[kind(10 * i + j, n) for j, n in enumerate(sizes)] for i in range(2)]  # of each stream, the small one first
    made = [[[c.outputs() for _ in range(ROUNDS)] for c in row] for row in calls]
    alone = [[c.outputs() for c in row] for row in calls]
    streams = [Stream(), Stream()]
    synchronize()
    for j in range(len(sizes)):
        for r in range(ROUNDS):
            for i in range(2):
                calls[i][j].run(made[i][j][r], streams[i].handle)
    for s in streams:
        s.synchronize()
    for i in range(2):
        for j in range(len(sizes)):
            got = [{name: b.download() for name, b in o.items()} for o in made[i][j]]
            calls[i][j].run(alone[i][j], None)
            synchronize()
            for name, b in alone[i][j].items():
                want = b.download().view(np.uint8)
                assert want.any(), (i, j, name)
                for r in range(ROUNDS):
                    assert np.array_equal(got[r][name].view(np.uint8), want), (i, j, r, name)


def test_larger_calls_outgrow_the_scratch():
    """Of the sizes above the second takes more than the block that a stream's first call gets (1 MiB)."""
    for small, large in ((attend_workspace_bytes(2, 8, 64, 4000, True), attend_workspace_bytes(48, 8, 64, 4000, True)),
                         (evict_workspace_bytes(2, 2, 1200, 560), evict_workspace_bytes(200, 2, 1200, 560)),
                         [_lib.lib().ouro_token_logprobs_workspace_bytes(rows, 500, 9) for rows in (3, 9000)]):
        assert small < 1 << 20 < large
