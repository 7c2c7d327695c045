"""Entry points of the 8-bit cache, the head norms and the verification without a
GPU: their refusal before ouro_init, and the workspace sizes that they give."""
import subprocess
import sys
from pathlib import Path

import pytest

from ouroboros_amd import kvcache, ops

ROOT = Path(__file__).resolve().parents[1]


def test_calls_before_init_are_refused():
    code = (
        "from ouroboros_amd import _lib; L=_lib.lib()\n"
        "for name, (_, args) in _lib.SIGNATURES.items():\n"
        "    if name in ('ouro_qk_norm_rope','ouro_kv8_write','ouro_kv8_read','ouro_kv8_attend','ouro_verify_drafts'):\n"
        "        assert getattr(L, name)(*[None if a is _lib.vp else 0 for a in args]) == 7, name\n"
        "assert b'ouro_init' in L.ouro_last_error(); print('ok')"
    )
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)
    assert r.returncode == 0 and "ok" in r.stdout, r.stderr


@pytest.mark.parametrize("seqs,rows,n", [(1, 1, 1), (1, 5, 32003), (64, 320, 248320), (0, 0, 10), (3, 7, 2041), (3, 7, 2042)])
def test_verify_workspace(seqs, rows, n):
    segs = (n + 7 + 2047) // 2048  # the last of which may hold none where a row starts at a multiple of 16 bytes
    # a maximum, its place and a sum of each segment, of target and draft; what is left; what the sequence came to
    need = 2 * rows * segs * 16 + seqs * (segs * 8 + 48)
    got = ops.verify_workspace_bytes(seqs, rows, n)
    assert need <= got <= need + 4096


@pytest.mark.parametrize("seqs,rows,max_new,heads,kv,d,max_len", [
    (1, 1, 1, 16, 4, 128, 1), (64, 64, 1, 16, 4, 128, 2176), (48, 200, 6, 32, 2, 64, 8191), (2, 2048, 1024, 16, 4, 128, 16384), (1, 0, 0, 4, 1, 64, 100)])
def test_attend_workspace(seqs, rows, max_new, heads, kv, d, max_len):
    got = kvcache.attend8_workspace_bytes(seqs, rows, max_new, heads, kv, d, max_len)
    # outputs, maxima and sums of the splits, each of a whole number of 256 slots; none where one holds all
    most = -(-max_len // 256)
    assert got <= rows * heads * most * (d + 2) * 4 + 256
    assert got == 0 if max_len <= 256 or not rows else got >= rows * heads * 2 * (d + 2) * 4


@pytest.mark.parametrize("heads,kv,d", [(16, 4, 128), (32, 2, 64), (4, 4, 192), (8, 1, 128), (48, 1, 64)])
def test_attend_workspace_serves_shorter_calls(heads, kv, d):
    """Never less for more sequences, rows, new rows of a sequence or slots."""
    def need(seqs, rows, new, slots):
        return kvcache.attend8_workspace_bytes(seqs, rows, new, heads, kv, d, slots)

    for slots in (300, 5000, 40000):
        for grow in (lambda n: (3, 500, n, slots), lambda n: (3, 3 * n, n, slots)):
            sizes = [need(*grow(n)) for n in [*range(0, 400), *range(400, 3000, 37)]]
            assert sizes == sorted(sizes)
    for new in (1, 4, 5, 64, 300, 1024):
        sizes = [need(2, 2 * new, new, n) for n in [*range(0, 3000, 61), *range(3000, 300000, 1777)]]
        assert sizes == sorted(sizes)
        sizes = [need(n, 700, new, 9000) for n in range(0, 900)]
        assert sizes == sorted(sizes)
