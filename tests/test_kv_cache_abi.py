"""The paged cache's and log probabilities' entry points without a GPU: their
refusal before ouro_init, and the workspace sizes that they give."""
import subprocess
import sys
from pathlib import Path

import pytest

from ouroboros_amd import _lib, kvcache

ROOT = Path(__file__).resolve().parents[1]


def test_calls_before_init_are_refused():
    code = (
        "from ouroboros_amd import _lib; L=_lib.lib()\n"
        "assert L.ouro_kv_attend(*[None]*2,None,0,None,None,0,None,None,None,0,None,None,0,None,0,1,1,1,1.0,None,None)==7\n"
        "assert L.ouro_kv_evict(None,None,None,1,1,1,0,None,None,None,None,None)==7\n"
        "assert L.ouro_token_logprobs(None,0,1,1,0,None,0,*[None]*8)==7\n"
        "assert b'ouro_init' in L.ouro_last_error(); print('ok')"
    )
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)
    assert r.returncode == 0 and "ok" in r.stdout, r.stderr


@pytest.mark.parametrize("seqs,heads,d,max_len", [(1, 16, 128, 1), (1, 16, 128, 257), (64, 8, 80, 1025), (3, 20, 256, 16384)])
def test_attend_workspace(seqs, heads, d, max_len):
    splits = -(-max_len // 256)
    need = 0 if splits == 1 else seqs * heads * splits * (d + 2) * 4  # the splits' outputs, maxima and sums
    got = kvcache.attend_workspace_bytes(seqs, heads, d, max_len)
    assert need <= got <= need + 4096
    more = kvcache.attend_workspace_bytes(seqs, heads, d, max_len, True)
    assert more >= got + seqs * heads * max_len * 4  # the scores


@pytest.mark.parametrize("seqs,heads,max_len,keep", [(1, 1, 1, 1), (64, 4, 1025, 1024), (4, 4, 16384, 2048), (2, 8, 100, 200)])
def test_evict_workspace(seqs, heads, max_len, keep):
    moves = min(keep, max(max_len - keep, 0))
    need = seqs * heads * (8 * moves + 4 * (keep + 1))  # the moves, their number, and where each kept slot comes from
    got = kvcache.evict_workspace_bytes(seqs, heads, max_len, keep)
    assert need <= got <= need + 4096


@pytest.mark.parametrize("rows,n,k", [(1, 1, 0), (1, 8000, 0), (1, 8000, 1), (7, 32003, 0), (64, 248320, 20), (100000, 500, 5)])
def test_logprobs_workspace(rows, n, k):
    got = int(_lib.lib().ouro_token_logprobs_workspace_bytes(rows, n, k))
    if n <= 8192 - 8 and not k:
        assert got == 0
    else:
        parts = -(-n // 8192)
        launch = min(rows, 65535)
        assert got >= launch * parts * (16 + (128 if k else 0))
        assert got <= launch * (parts + 1) * (16 + (128 if k else 0)) + 4096
