"""The paged 8-bit key/value cache and the attention over it (jx_kv_* of include/jxmoe.h).

  KVCache    pages of int8 codes with one fp32 scale per 32 tokens and head; reserve / trim / fork / compact its
             pages, append keys and values, attend over it
  KVBatch    which sequences take part in a call, and which rows are theirs
  Attention  heads, type, masks and strides of an attention

Every call is enqueued on `stream` (a hipStream_t as an integer; None: the default stream) and returns without
synchronizing.  Device memory is given as a DeviceBuffer, as anything with a `ptr` or a `data_ptr()`, or as an address.
What only the device can see (a slot out of range, no free pages, ...) is told by `check_status`.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import formats as F
from ._lib import (JX_KV_BAD_ARG, JX_KV_BAD_PAGE, JX_KV_BLOCK, JX_KV_NO_PAGES, JX_KV_SHARED, JX_KV_STATUS_WORDS, AttentionDesc,
                   JxError, KVBatchDesc, KVCacheDesc, check, lib)
from .moe import DeviceBuffer, init

STATUS = {JX_KV_BAD_PAGE: "a table entry names no page of the cache",
          JX_KV_BAD_ARG: "a slot, length or row range out of its limits, or a slot twice in one list",
          JX_KV_NO_PAGES: "not enough free pages", JX_KV_SHARED: "an append into a page that another slot holds too"}


def _address(buffer) -> int | None:
    """The device address of a buffer (None: NULL)."""
    if buffer is None or isinstance(buffer, int):
        return buffer
    if hasattr(buffer, "data_ptr"):
        return buffer.data_ptr()
    ptr = buffer.ptr
    return ptr.value if isinstance(ptr, C.c_void_p) else ptr


class KVBatch:
    """Sequence i's rows are row_start[i] .. row_start[i + 1] - 1, the last tokens of slot seqs[i] (jx_kv_batch)."""

    def __init__(self, *, n_seqs: int, n_rows: int | None = None, max_rows: int = 1, max_len: int = 0, seqs=None,
                 row_start=None):
        self.keep = (seqs, row_start)
        self.desc = KVBatchDesc(n_seqs, n_seqs if n_rows is None else n_rows, max_rows, max_len, _address(seqs),
                                _address(row_start))
        self.ref = C.byref(self.desc)


class Attention:
    """What an attention computes (jx_attention); strides in elements, 0: contiguous rows."""

    def __init__(self, *, n_heads: int, scale: float, dtype: int = F.F32, softcap: float = 0.0, window: int = 0,
                 causal: bool = True, alibi=None, q_stride: int = 0, out_stride: int = 0):
        self.keep = alibi
        self.desc = AttentionDesc(n_heads, dtype, scale, softcap, window, 1 if causal else 0, q_stride, out_stride,
                                  _address(alibi))
        self.ref = C.byref(self.desc)


class KVCache:
    """A cache of n_layers x n_pages pages (jx_kv_cache).  `buffers`: device memory of the caller by field name ("codes",
    "scales", "table", "len", "ref", "status", "scratch"); what is not given is allocated, len, ref and status zeroed."""

    def __init__(self, *, n_layers: int, n_pages: int, page_tokens: int, n_kv_heads: int, head_dim: int, max_seqs: int,
                 max_pages: int, device: int = 0, buffers: dict | None = None):
        init(device)
        self.desc = KVCacheDesc(device, n_layers, n_pages, page_tokens, n_kv_heads, head_dim, max_seqs, max_pages)
        self.ref = C.byref(self.desc)
        words = lib().jx_kv_scratch_words(self.ref)
        if not words:
            raise JxError(f"KVCache: {lib().jx_moe_last_error().decode(errors='replace')}")
        blocks = n_layers * n_pages * 2 * n_kv_heads * (page_tokens // JX_KV_BLOCK)
        sizes = {"codes": blocks * JX_KV_BLOCK * head_dim, "scales": 4 * blocks, "table": 4 * max_seqs * max_pages,
                 "len": 4 * max_seqs, "ref": 4 * n_pages, "status": 4 * JX_KV_STATUS_WORDS, "scratch": 4 * words}
        unknown = set(buffers or {}) - set(sizes)
        if unknown:
            raise JxError(f"KVCache: no such buffer: {', '.join(sorted(unknown))}")
        self.buffers = dict(buffers or {})
        for name, size in sizes.items():
            if name not in self.buffers:
                self.buffers[name] = DeviceBuffer(size)
                if name in ("len", "ref", "status"):
                    self.buffers[name].upload(np.zeros(size, np.uint8))
            setattr(self.desc, name, _address(self.buffers[name]))

    def reserve(self, slots, n_new, n: int, stream: int | None = None) -> None:
        """Room for n_new[i] tokens (None: one each) behind slots[i], whose length grows by them."""
        check(lib().jx_kv_reserve(self.ref, _address(slots), _address(n_new), n, stream), "jx_kv_reserve")

    def trim(self, slots, new_len, n: int, stream: int | None = None) -> None:
        """slots[i] keeps new_len[i] tokens at most (None: none, the slot is freed)."""
        check(lib().jx_kv_trim(self.ref, _address(slots), _address(new_len), n, stream), "jx_kv_trim")

    def fork(self, src, dst, n: int, stream: int | None = None) -> None:
        """dst[i] becomes src[i] as it was before the call; full pages are shared."""
        check(lib().jx_kv_fork(self.ref, _address(src), _address(dst), n, stream), "jx_kv_fork")

    def compact(self, stream: int | None = None) -> None:
        """The pages in use become 0 .. count - 1 (count: word 1 of status)."""
        check(lib().jx_kv_compact(self.ref, stream), "jx_kv_compact")

    def append(self, batch: KVBatch, k, v, dtype: int = F.F32, layer: int = 0, row_stride: int = 0,
               stream: int | None = None) -> None:
        """Keys and values [n_rows][n_kv_heads][head_dim] of the batch's rows into `layer`."""
        check(lib().jx_kv_append(self.ref, batch.ref, layer, dtype, _address(k), _address(v), row_stride, stream),
              "jx_kv_append")

    def workspace(self, batch: KVBatch, attention: Attention) -> DeviceBuffer | None:
        """Workspace of an attention call of these sizes (None if it needs none)."""
        size = lib().jx_kv_attention_workspace(self.ref, batch.ref, attention.ref)
        return DeviceBuffer(size) if size else None

    def attend(self, batch: KVBatch, attention: Attention, q, out, ws=None, layer: int = 0, stream: int | None = None) -> None:
        """Attention of the rows q [n_rows][n_heads][head_dim] over their sequences in `layer`; ws: `workspace()`."""
        check(lib().jx_kv_attention(self.ref, batch.ref, attention.ref, layer, _address(q), _address(out), _address(ws),
                                    0 if ws is None else ws.nbytes, stream), "jx_kv_attention")

    def status(self) -> tuple[int, int]:
        """(error bits, pages in use after the last compaction); waits for the device."""
        words = np.zeros(JX_KV_STATUS_WORDS, np.int32)
        check(lib().jx_device_synchronize(), "jx_device_synchronize")
        check(lib().jx_memcpy_dtoh(C.c_void_p(words.ctypes.data), self.desc.status, words.nbytes), "jx_memcpy_dtoh")
        return int(words[0]), int(words[1])

    def check_status(self) -> None:
        """Raise JxError if a call found something wrong on the device, and let the cache go on."""
        bits = self.status()[0]
        if bits:
            zero = np.zeros(1, np.int32)
            check(lib().jx_memcpy_htod(self.desc.status, C.c_void_p(zero.ctypes.data), 4), "jx_memcpy_htod")
            raise JxError("KVCache: " + "; ".join(text for bit, text in STATUS.items() if bits & bit))
