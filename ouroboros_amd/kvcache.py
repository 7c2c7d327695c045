"""A caller's paged key-value cache on the GPU: attention of one new token a
sequence over it, and eviction from it by accumulated attention weight
(ouro_kv_attend, ouro_kv_evict); and one of 8-bit codes, written, read and
attended to by any number of new tokens (ouro_kv8_write, _read, _attend).

:class:`KVCache` and :class:`KVCache8` are descriptions of device memory that the
caller owns; they keep the addresses only (and the DeviceBuffers that they came from).
Arguments that are device memory are a DeviceBuffer or the address of another
runtime's allocation.
"""
from __future__ import annotations

import ctypes as C

from . import _lib
from ._lib import Kv8CacheDesc, KvCacheDesc, KvHistoryDesc, call, dtype_code
from .ops import _addr


class History:
    """Attention weight received [seqs][heads][slots] and token position of each
    slot: heads = the cache's kv heads, each by itself, or 1, all together."""

    def __init__(self, weight, pos, heads: int, slots: int):
        self.weight, self.pos, self.heads, self.slots = weight, pos, heads, slots
        self._c = KvHistoryDesc(_addr(weight), _addr(pos), heads, slots)
        self._ref = C.addressof(self._c)


def _strides(layout: str, strides, page_tokens: int, n_head_kv: int, head_dim: int) -> tuple:
    """(page, token, head) strides of a layout, or those that were given."""
    if strides is not None:
        return tuple(strides)
    if layout not in ("token", "head"):
        raise ValueError(f"layout {layout!r}: 'token' or 'head'")
    row = (n_head_kv * head_dim, head_dim) if layout == "token" else (head_dim, page_tokens * head_dim)
    return (page_tokens * n_head_kv * head_dim, *row)


class KVCache:
    """Pools k and v of n_pages pages of page_tokens tokens, and the page table
    pages [seqs][max_pages].

    layout "token": [page][token][head][head_dim], "head": [page][head][token]
    [head_dim]; or strides = (page, token, head) in elements."""

    def __init__(self, k, v, pages, *, n_pages: int, max_pages: int, page_tokens: int, n_head_kv: int, head_dim: int,
                 dtype="bf16", layout: str = "token", strides=None):
        _lib.init()
        strides = _strides(layout, strides, page_tokens, n_head_kv, head_dim)
        self.n_head_kv, self.head_dim, self.page_tokens = n_head_kv, head_dim, page_tokens
        self._held = (k, v, pages)
        self._c = KvCacheDesc(_addr(k), _addr(v), _addr(pages), *strides, n_pages, max_pages, page_tokens, n_head_kv,
                              head_dim, dtype_code(dtype))
        self._ref = C.addressof(self._c)
        self._scale = head_dim ** -0.5

    def attend(self, q, out, lens, seqs: int, max_len: int, n_head: int, *, dtype="f32", k_new=None, v_new=None,
               pos_new=None, history: History | None = None, mask=None, mask_stride: int = 0, gate=None, lse=None,
               scale: float | None = None, q_stride: int = 0, new_stride: int = 0, out_stride: int = 0, workspace=None,
               stream=None) -> None:
        """out = softmax(scale q.k) v of one token a sequence over its lens[b]
        slots, the new token's k_new, v_new written to the last of them first.
        scale: 1 / sqrt(head_dim) unless given."""
        call("ouro_kv_attend", self._ref, history._ref if history else None, _addr(q), q_stride, _addr(k_new),
             _addr(v_new), new_stride, _addr(pos_new), _addr(lens), _addr(mask), mask_stride, _addr(gate), _addr(out),
             out_stride, _addr(lse), dtype_code(dtype), seqs, n_head, max_len,
             self._scale if scale is None else scale, _addr(workspace), stream)

    def evict(self, history: History, lens, seqs: int, max_len: int, keep: int, recent: int, lens_out, *,
              out: History | None = None, slot_from=None, workspace=None, stream=None) -> None:
        """Cut every sequence to its `recent` newest positions and the heaviest
        other slots, `keep` in all; the history (or `out`) and lens_out describe
        what is left.  Every slot in use of a sequence that is cut has its page
        (the choice does not look at the page table), and masks are not moved."""
        call("ouro_kv_evict", self._ref, history._ref, _addr(lens), seqs, max_len, keep, recent,
             out._ref if out else None, _addr(lens_out), _addr(slot_from), _addr(workspace), stream)


class KVCache8:
    """Pools k and v of int8 codes, laid out as :class:`KVCache`'s, with float
    scales k_scale, v_scale [n_pages][page_tokens / block_tokens][n_head_kv]: an
    element stands for code * scale.

    The calls take each sequence's newest rows packed one after another: rows
    cu[b] .. cu[b + 1] - 1 (device int32; without cu, max_new of every sequence)
    are the last of its lens[b] slots; `rows` is their number over all sequences,
    max_new at least the most of one."""

    def __init__(self, k, v, k_scale, v_scale, pages, *, n_pages: int, max_pages: int, page_tokens: int,
                 block_tokens: int, n_head_kv: int, head_dim: int, layout: str = "token", strides=None):
        _lib.init()
        strides = _strides(layout, strides, page_tokens, n_head_kv, head_dim)
        self.n_head_kv, self.head_dim, self.page_tokens, self.block_tokens = n_head_kv, head_dim, page_tokens, block_tokens
        self._held = (k, v, k_scale, v_scale, pages)
        self._c = Kv8CacheDesc(_addr(k), _addr(v), _addr(k_scale), _addr(v_scale), _addr(pages), *strides, n_pages,
                               max_pages, page_tokens, block_tokens, n_head_kv, head_dim)
        self._ref = C.addressof(self._c)
        self._scale = head_dim ** -0.5

    def write(self, k_new, v_new, lens, seqs: int, rows: int, max_new: int, *, cu=None, dtype="f32", new_stride: int = 0,
              stream=None) -> None:
        """The newest rows' keys and values into the cache, each block's scale the
        power of two that its rows need (older rows are rounded to a scale that grew)."""
        call("ouro_kv8_write", self._ref, _addr(k_new), _addr(v_new), new_stride, dtype_code(dtype), _addr(lens), _addr(cu),
             seqs, rows, max_new, stream)

    def read(self, k_out, v_out, lens, seqs: int, rows: int, max_new: int, *, cu=None, dtype="f32", out_stride: int = 0,
             stream=None) -> None:
        """The newest rows as the numbers they stand for (all of a sequence's with
        as many rows as slots); k_out or v_out may be None."""
        call("ouro_kv8_read", self._ref, _addr(lens), _addr(cu), seqs, rows, max_new, _addr(k_out), _addr(v_out), out_stride,
             dtype_code(dtype), stream)

    def attend(self, q, out, lens, seqs: int, rows: int, max_new: int, max_len: int, n_head: int, *, cu=None, dtype="f32",
               window: int = 0, sinks: int = 0, mask=None, mask_stride: int = 0, gate=None, lse=None,
               scale: float | None = None, q_stride: int = 0, out_stride: int = 0, workspace=None, stream=None) -> None:
        """out = softmax(scale q.k) v of each newest row over the slots up to its
        own (the last `window` of them and the first `sinks`, if a window is given).
        scale: 1 / sqrt(head_dim) unless given."""
        call("ouro_kv8_attend", self._ref, _addr(q), q_stride, _addr(lens), _addr(cu), _addr(mask), mask_stride, _addr(gate),
             _addr(out), out_stride, _addr(lse), dtype_code(dtype), seqs, rows, max_new, n_head, max_len, window, sinks,
             self._scale if scale is None else scale, _addr(workspace), stream)


def attend8_workspace_bytes(seqs: int, rows: int, max_new: int, n_head: int, n_head_kv: int, head_dim: int,
                            max_len: int) -> int:
    """Bytes of scratch that KVCache8.attend takes (0 = none), enough also for calls of fewer sequences, rows, new rows
    of a sequence or slots."""
    return int(_lib.lib().ouro_kv8_attend_workspace_bytes(seqs, rows, max_new, n_head, n_head_kv, head_dim, max_len))


def attend_workspace_bytes(seqs: int, n_head: int, head_dim: int, max_len: int, with_history: bool = False) -> int:
    """Bytes of scratch that KVCache.attend takes (0 = none)."""
    return int(_lib.lib().ouro_kv_attend_workspace_bytes(seqs, n_head, head_dim, max_len, int(with_history)))


def evict_workspace_bytes(seqs: int, heads: int, max_len: int, keep: int) -> int:
    """Bytes of scratch that KVCache.evict takes."""
    return int(_lib.lib().ouro_kv_evict_workspace_bytes(seqs, heads, max_len, keep))
