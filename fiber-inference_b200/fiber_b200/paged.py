"""Operators over the paged KV cache for ragged batches (include/fiber_paged.h).

``kv_append`` rotates and stores the new tokens' keys and values, ``attn_paged`` lets them
attend to their sequences' pages (chunks and single tokens alike). Buffers are plain device
addresses, as everywhere in this package; a view and a batch are made once and reused while
their buffers stay in place (the lengths themselves live in device memory).
"""
from __future__ import annotations

import ctypes as C

from .cuda import FiberError, _check, _stream_ptr, cuda_lib

__all__ = ["GGML_BF16", "PagedKV", "RaggedBatch", "Rope", "kv_view", "kv_append", "attn_paged", "attn_paged_workspace",
           "attn_paged_status", "attn_paged_drill"]

GGML_BF16 = 30


class PagedKV(C.Structure):
    """fiber_kv_view_t: one layer of a paged cache. Strides are in elements; by default pages
    are [n_kv_heads][page_size][head_dim], packed."""

    _fields_ = [("type", C.c_int), ("head_dim", C.c_int), ("n_kv_heads", C.c_int), ("page_size", C.c_int),
                ("n_pages", C.c_int), ("n_slots", C.c_int), ("max_pages", C.c_int), ("page_stride", C.c_int64),
                ("head_stride", C.c_int64), ("pos_stride", C.c_int64), ("k_pool", C.c_void_p), ("v_pool", C.c_void_p),
                ("page_table", C.c_void_p)]

    def __init__(self, k_pool: int, v_pool: int, page_table: int, *, n_slots: int, max_pages: int, n_pages: int,
                 page_size: int, n_kv_heads: int, head_dim: int, dtype: int = 1, page_stride: int | None = None,
                 head_stride: int | None = None, pos_stride: int | None = None):
        pos = head_dim if pos_stride is None else pos_stride
        head = page_size * head_dim if head_stride is None else head_stride
        page = n_kv_heads * page_size * head_dim if page_stride is None else page_stride
        super().__init__(dtype, head_dim, n_kv_heads, page_size, n_pages, n_slots, max_pages, page, head, pos, k_pool,
                         v_pool, page_table)


class RaggedBatch(C.Structure):
    """fiber_ragged_t: sequence s brings token rows q_start[s] .. q_start[s + 1] - 1 and has
    kv_len[s] positions cached with them (int32 device arrays)."""

    _fields_ = [("n_seqs", C.c_int), ("n_tokens", C.c_int), ("max_q", C.c_int), ("q_start", C.c_void_p),
                ("kv_len", C.c_void_p), ("slot", C.c_void_p)]

    def __init__(self, q_start: int, kv_len: int, *, n_seqs: int, n_tokens: int, max_q: int, slot: int | None = None):
        super().__init__(n_seqs, n_tokens, max_q, q_start, kv_len, slot)


class Rope(C.Structure):
    """fiber_rope_t: fp32 (cos, sin) table [max_pos][dim / 2][2] on the device."""

    _fields_ = [("table", C.c_void_p), ("max_pos", C.c_int), ("dim", C.c_int), ("adjacent", C.c_int)]

    def __init__(self, table: int, *, max_pos: int, dim: int, adjacent: bool = False):
        super().__init__(table, max_pos, dim, int(adjacent))


_lib = None


def _paged_lib() -> C.CDLL:
    global _lib
    if _lib is None:
        L = cuda_lib()
        V, B = C.POINTER(PagedKV), C.POINTER(RaggedBatch)
        L.fiber_kv_view.argtypes = [C.c_void_p, C.c_int, V]
        L.fiber_kv_append.argtypes = [V, B, C.c_int, C.c_void_p, C.c_int64, C.c_void_p, C.c_int64, C.c_void_p, C.c_int64,
                                      C.c_int, C.POINTER(Rope), C.c_void_p, C.c_int64, C.c_void_p]
        L.fiber_attn_paged_workspace.argtypes = [V, B, C.c_int]
        L.fiber_attn_paged_workspace.restype = C.c_size_t
        L.fiber_attn_paged.argtypes = [V, B, C.c_void_p, C.c_int64, C.c_void_p, C.c_int64, C.c_int, C.c_float, C.c_int,
                                       C.c_void_p, C.c_size_t, C.c_void_p]
        L.fiber_attn_paged_status.argtypes = [C.c_void_p, C.c_void_p]
        L.fiber_attn_paged_drill.argtypes = [C.c_int]
        _lib = L
    return _lib


def kv_view(cache, layer: int) -> PagedKV:
    """fiber_kv_view: one layer of a KVCache as the operators take it."""
    view = PagedKV(0, 0, 0, n_slots=0, max_pages=0, n_pages=0, page_size=0, n_kv_heads=0, head_dim=0)
    _check(_paged_lib().fiber_kv_view(cache.addr, layer, view), "fiber_kv_view")
    return view


def kv_append(kv: PagedKV, batch: RaggedBatch, in_type: int, q: int | None, k: int, v: int, *, ld: int = 0,
              ldq: int | None = None, ldk: int | None = None, ldv: int | None = None, n_heads: int = 0,
              q_out: int | None = None, ld_out: int = 0, rope: Rope | None = None, stream=None):
    """fiber_kv_append: q rotated into q_out, k rotated and v into the cache. `ld` is the row
    stride of q, k and v alike (one fused buffer); ldq / ldk / ldv set them apart."""
    rc = (_lib or _paged_lib()).fiber_kv_append(
        kv, batch, in_type, q, ld if ldq is None else ldq, k, ld if ldk is None else ldk, v, ld if ldv is None else ldv,
        n_heads, rope, q_out, ld_out, stream if type(stream) is int else _stream_ptr(stream))
    if rc:
        _check(rc, "fiber_kv_append")


def attn_paged_workspace(kv: PagedKV, batch: RaggedBatch, n_heads: int) -> int:
    """Bytes of zero-filled device memory that attn_paged needs for batches of this shape."""
    n = int(_paged_lib().fiber_attn_paged_workspace(kv, batch, n_heads))
    if n == 0:
        raise FiberError(f"fiber_attn_paged_workspace: {cuda_lib().fiber_last_error().decode()}")
    return n


def attn_paged(kv: PagedKV, batch: RaggedBatch, q: int, out: int, *, n_heads: int, ldq: int, ldo: int, scale: float,
               ws: int, ws_bytes: int, window: int = 0, stream=None):
    """fiber_attn_paged: causal attention of the batch's tokens over the cache."""
    rc = (_lib or _paged_lib()).fiber_attn_paged(kv, batch, q, ldq, out, ldo, n_heads, scale, window, ws, ws_bytes,
                                                 stream if type(stream) is int else _stream_ptr(stream))
    if rc:
        _check(rc, "fiber_attn_paged")


def attn_paged_status(ws: int, stream=None):
    """Waits for the stream; raises if a bounded wait inside an attn_paged call gave up, or q_start decreased."""
    _check(_paged_lib().fiber_attn_paged_status(ws, _stream_ptr(stream)), "fiber_attn_paged_status")


def attn_paged_drill(on: bool):
    """fiber_attn_paged_drill: while on, waits inside later attn_paged calls run out."""
    _check(_paged_lib().fiber_attn_paged_drill(int(on)), "fiber_attn_paged_drill")
