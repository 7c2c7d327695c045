"""Entry points of the 8-bit cache, the head norms and the verification without a
GPU: their refusal before ouro_init, and the workspace sizes that they give."""
import subprocess
import sys
from pathlib import Path

import pytest

from ouroboros_amd import ops

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


@pytest.mark.parametrize("seqs,rows,n", [(1, 1, 1), (1, 5, 32003), (64, 320, 248320), (0, 0, 10), (3, 7, 8185), (3, 7, 8186)])
def test_verify_workspace(seqs, rows, n):
    parts = (n + 7 + 8191) // 8192  # the last of which may hold none where a row starts at a multiple of 16 bytes
    need = 2 * rows * parts * 16 + seqs * parts * 8  # a maximum, its place and a sum of each part, of target and draft; what is left
    got = ops.verify_workspace_bytes(seqs, rows, n)
    assert need <= got <= need + 4096
