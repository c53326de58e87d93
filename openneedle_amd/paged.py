"""Device int8 KV cache in pages, for many requests of different lengths.

Rows are quantized as in :class:`~openneedle_amd.kv.KVCache` (needle2/csrc/engine.cpp:1005-1021); the reference keeps one
sequence in one run of slots. Here requests share the cache's pages: :meth:`PagedCache.extend` deals pages to the requests
of a step on the device and says where every new token lies, :meth:`PagedCache.store` (or :meth:`PagedCache.store_rotated`)
puts the tokens' rows there, :meth:`PagedCache.attention` attends a ragged batch of new tokens, and
:meth:`PagedCache.trim` takes tokens back. All of them can be captured in a graph.
"""
from __future__ import annotations

import ctypes

from . import _ffi
from ._ffi import GpuError, addr, check
from .device import DeviceView, stream_ptr


class PagedCache:
    """``pages`` pages of ``page_size`` positions of ``kvheads`` rows per layer."""

    def __init__(self, layers: int, pages: int, page_size: int, kvheads: int, head_dim: int):
        self._lib = _ffi.lib()
        self.layers, self.pages, self.page_size, self.kvheads, self.head_dim = layers, pages, page_size, kvheads, head_dim
        self.ptr = self._lib.needle2_gpu_pages_create(layers, pages, page_size, kvheads, head_dim)
        if not self.ptr:
            raise GpuError(f"paged cache: {_ffi.last_error()}")

    def storage_bytes(self) -> int:
        return int(self._lib.needle2_gpu_pages_storage_bytes(self.ptr))

    def free_pages(self, stream=None) -> int:
        """Pages that are free once ``stream`` has run what it has (waits for it)."""
        n = ctypes.c_int()
        check(self._lib.needle2_gpu_pages_free(self.ptr, ctypes.byref(n), stream_ptr(stream)), "free pages")
        return n.value

    def reset(self, stream=None) -> None:
        """All pages are free again; tables made before are not to be used any more."""
        check(self._lib.needle2_gpu_pages_reset(self.ptr, stream_ptr(stream)), "paged cache reset")

    def extend(self, requests: int, d_counts, tokens: int, d_lengths, d_tables, width: int, d_starts, d_firsts, d_slots,
               d_positions, stream=None) -> None:
        """Pages for ``d_counts[r]`` new tokens of every request of ``d_lengths[r]`` positions, into ``d_tables``
        ``[requests][width]``; ``d_lengths`` advances. Results (all int32): ``d_starts [requests + 1]``, where each
        request's tokens begin in the batch; ``d_firsts [requests]``, the position of its first; ``d_slots`` and
        ``d_positions [tokens]``. A request whose tokens pass its table or the ``tokens`` of the batch, or for which the
        free pages no longer suffice, gets none: its length stays, its first position is -1, and so are its tokens'
        slots and positions, as are those behind the last request's."""
        check(self._lib.needle2_gpu_pages_extend(self.ptr, int(requests), addr(d_counts), int(tokens), addr(d_lengths),
                                                 addr(d_tables), int(width), addr(d_starts), addr(d_firsts),
                                                 addr(d_slots), addr(d_positions), stream_ptr(stream)), "page extension")

    def trim(self, requests: int, d_keep, d_lengths, d_tables, width: int, stream=None) -> None:
        """Cut every request to its first ``d_keep[r]`` positions (0: the request ends; negative: it stays as it is): pages
        that hold none of them are free again and -1 in ``d_tables``. With the ``d_firsts`` of an extension right before
        it, it undoes that. Only for tables whose pages :meth:`extend` dealt, each to one request."""
        check(self._lib.needle2_gpu_pages_trim(self.ptr, int(requests), addr(d_keep), addr(d_lengths), addr(d_tables),
                                               int(width), stream_ptr(stream)), "page trim")

    def store(self, layer: int, d_k, d_v, tokens: int, d_slots, k_stride: int = 0, v_stride: int = 0, stream=None) -> None:
        """Quantize device fp32 rows ``[tokens][kvheads][head_dim]`` into slots (``page * page_size + position in it``;
        outside the cache, as -1: not stored). Strides: floats from one token's row to the next (0: no gaps)."""
        row = self.kvheads * self.head_dim
        check(self._lib.needle2_gpu_pages_store(self.ptr, layer, addr(d_k), int(k_stride or row), addr(d_v),
                                                int(v_stride or row), int(tokens), addr(d_slots), stream_ptr(stream)),
              "paged store")

    def store_rotated(self, layer: int, d_q, d_k, d_v, heads: int, tokens: int, d_positions, d_slots, d_freq=None,
                      rotary: int = 0, d_q_gain=None, d_k_gain=None, eps: float = 1e-6, q_stride: int = 0,
                      k_stride: int = 0, v_stride: int = 0, d_q_out=None, q_out_stride: int = 0, d_k_out=None,
                      k_out_stride: int = 0, stream=None) -> None:
        """:func:`~openneedle_amd.heads.rotate_heads` of q and k and :meth:`store` of its k and of v, in one launch. q's
        result defaults to q's own place; k's is only stored unless ``d_k_out`` is given."""
        row = self.kvheads * self.head_dim
        qs = q_stride or heads * self.head_dim
        qo, qos = (d_q, qs) if d_q_out is None else (d_q_out, q_out_stride or heads * self.head_dim)
        check(self._lib.needle2_gpu_heads_store(self.ptr, layer, addr(d_q), int(qs), addr(qo), int(qos), int(heads),
                                                addr(d_k), int(k_stride or row), addr(d_k_out), int(k_out_stride or row),
                                                addr(d_v), int(v_stride or row), int(tokens), addr(d_positions),
                                                addr(d_slots), addr(d_q_gain), addr(d_k_gain), float(eps), addr(d_freq),
                                                int(rotary), stream_ptr(stream)), "heads into the paged cache")

    def attention(self, layer: int, d_q, d_out, heads: int, requests: int, tokens: int, count: int, d_starts, d_firsts,
                  d_tables, width: int, length: int = 0, window: int = 0, stream=None) -> None:
        """Attention of new tokens that are stored already: device q / out fp32 ``[tokens][heads][head_dim]``. Request
        ``r`` has rows ``d_starts[r] .. d_starts[r + 1] - 1``, at most ``count`` of them, the first at position
        ``d_firsts[r]`` (negative: zeros); a token attends its request's positions up to its own, the last ``window`` of
        them if that is not 0. ``length``: the most positions of a request (0: unknown), by which only the cut of the
        work goes: results for another one, or beside other requests, agree within the attention's exactness, not bit
        for bit. Rows of no request are left as they were."""
        check(self._lib.needle2_gpu_pages_attention(self.ptr, layer, addr(d_q), addr(d_out), int(heads), int(requests),
                                                    int(tokens), int(count), addr(d_starts), addr(d_firsts),
                                                    addr(d_tables), int(width), int(length), int(window),
                                                    stream_ptr(stream)), "paged attention")

    def device_pages(self, layer: int) -> DeviceView:
        """One layer's blocks as device memory of this cache, not copied: ``[pages][kvheads]`` blocks of K codes
        ``[page_size][head_dim]``, V codes, K scales ``[page_size]`` and V scales."""
        at = ctypes.c_void_p()
        check(self._lib.needle2_gpu_pages_layer(self.ptr, layer, ctypes.byref(at)), "paged cache layer")
        return DeviceView(self, at.value - self.ptr, self.storage_bytes() // self.layers)

    def close(self) -> None:
        ptr, self.ptr = getattr(self, "ptr", None), None
        if ptr:
            self._lib.needle2_gpu_pages_destroy(ptr)

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
