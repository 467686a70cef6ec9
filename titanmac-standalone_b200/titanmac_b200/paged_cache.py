"""Keys and values in pages that sequences share a pool of (``tmw_paged_append``, ``tmw_paged_attention``).

``RingCache`` keeps ``window + 1`` slots for every sequence of a fixed batch.  Here a sequence has as many pages of ``page_size``
tokens as it needs, anywhere in the pool: token ``t`` of sequence ``b`` is in slot ``t % page_size`` of page
``page_table[b, t // page_size]``.  Who hands out pages writes the table (on the device, in place if the calls are captured in a
graph); entries that no token needs may hold anything.  Sequences may share pages that nobody writes to, a batch may hold rows
without a sequence (``start`` / ``pos`` of -1), query heads may share key heads, and keys and queries can be rotated by their
positions on the way into the cache.

Serving only: no gradient flows through these calls (inputs that require one are taken as they are; forward-mode derivatives are
refused).

What the device finds wrong - a position or a page outside the table or the pool - makes NaN of what depends on it, touches nothing
else and is raised by ``_native.poll_status``.
"""

from __future__ import annotations

import struct
from typing import Optional

import torch

from . import _native

# tmw_pages; behind it the fields of tmw_paged_append_desc, of tmw_paged_attention_desc
_APPEND = struct.Struct("@8iq3Q 4i 4Q 12q 3Q")
_ATTENTION = struct.Struct("@8iq3Q 3if 4Q 4q Q")


def _refuse_devices(name: str, like: torch.Tensor, *tensors: Optional[torch.Tensor]) -> None:
    _native._require_cuda(like, *(t for t in tensors if t is not None))
    raise ValueError(f"{name}: every tensor must be on {like.device}")


def _page_numbers(name: str, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, batch: int):
    """``(dtype number, kv_heads, head_dim, page_size, pages, columns, row stride of the table)`` of a pool and its table."""
    shape, table, strides = k_pages.shape, page_table.shape, page_table.stride()
    if len(shape) != 4 or v_pages.shape != shape or not k_pages.is_contiguous() or not v_pages.is_contiguous():
        raise ValueError(f"{name}: k_pages and v_pages must be contiguous [pages, kv_heads, page_size, head_dim]")
    if len(table) != 2 or table[0] != batch or (strides[1] != 1 and table[1] > 1):
        raise ValueError(f"{name}: page_table must be [batch, columns] with contiguous rows")
    dtype = _native._DTYPES.get(k_pages.dtype)
    if dtype is None:
        raise TypeError(f"{name}: pages in float32, bfloat16 or float16 expected")
    return dtype, shape[1], shape[3], shape[2], shape[0], table[1], strides[0]


def _refuse_shape(name: str, t: torch.Tensor, shape) -> None:
    if t.shape != shape:
        raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
    raise ValueError("the head_dim axis must be contiguous")


def _check_numbers(name: str, t: torch.Tensor, batch: int) -> None:
    if t.shape != (batch,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous vector of one number per sequence")


def paged_append(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                 start: torch.Tensor, counts: Optional[torch.Tensor] = None, q: Optional[torch.Tensor] = None,
                 q_out: Optional[torch.Tensor] = None, inv_freq: Optional[torch.Tensor] = None,
                 interleaved: bool = False) -> Optional[torch.Tensor]:
    """New tokens into the pages: row ``r`` of ``k, v [B, kv_heads, rows, dh]`` (any strides, last axis contiguous) is token
    ``start[b] + r`` of sequence ``b``; rows from ``counts[b]`` on are left out (``start``, ``counts``: int32 ``[B]``).

    ``inv_freq`` (fp32, at most ``dh / 2`` numbers): the first ``2 * len(inv_freq)`` numbers of every key are rotated in pairs,
    pair ``i`` by ``t * inv_freq[i]`` at token ``t``; the pairs are ``(i, i + len(inv_freq))`` or, ``interleaved``,
    ``(2 i, 2 i + 1)``.  ``q [B, heads, rows, dh]`` is rotated likewise into ``q_out`` (may be ``q``; made if None), which is
    returned; its rows that are no new token's are left as they are.  Writes of the same slot twice in one call are the caller's
    to avoid.  Serving only: nothing that is returned or written carries a gradient."""
    index = k_pages.get_device()
    if not 0 <= index == k.get_device() == v.get_device() == v_pages.get_device() == page_table.get_device() == start.get_device():
        _refuse_devices("paged_append", k_pages, k, v, v_pages, page_table, start)
    dtype = k_pages.dtype
    if not (dtype is v_pages.dtype is k.dtype is v.dtype and torch.int32 is page_table.dtype is start.dtype):
        raise TypeError("paged_append: k, v and the pages must share one dtype; page_table and start must be int32")
    _native.refuse_tangents("paged_append", k, v, k_pages, v_pages, q)
    shape = k.shape
    if len(shape) != 4:
        raise ValueError("paged_append: k and v must be [batch, kv_heads, rows, head_dim]")
    B, rows = shape[0], shape[2]
    number, kv_heads, head_dim, page_size, pages, columns, table_stride = _page_numbers("paged_append", k_pages, v_pages, page_table,
                                                                                        B)
    ks, vs = k.stride(), v.stride()
    if shape[1] != kv_heads or shape[3] != head_dim or ks[3] != 1:
        _refuse_shape("k", k, (B, kv_heads, rows, head_dim))
    if v.shape != shape or vs[3] != 1:
        _refuse_shape("v", v, shape)
    _check_numbers("start", start, B)
    if counts is not None:
        if counts.get_device() != index:
            _refuse_devices("paged_append", k_pages, counts)
        if counts.dtype is not torch.int32:
            raise TypeError("counts must be int32")
        _check_numbers("counts", counts, B)
    rotated = 0
    if inv_freq is not None:
        if inv_freq.get_device() != index:
            _refuse_devices("paged_append", k_pages, inv_freq)
        if inv_freq.dtype is not torch.float32 or inv_freq.dim() != 1 or not inv_freq.is_contiguous():
            raise TypeError("inv_freq must be a contiguous fp32 vector")
        rotated = 2 * inv_freq.shape[0]
        if rotated > head_dim:
            raise ValueError("inv_freq has more than head_dim / 2 numbers")
    heads, qs, os_ = 0, (0, 0, 0, 1), (0, 0, 0, 1)
    if q is not None:
        if q.get_device() != index or (q_out is not None and q_out.get_device() != index):
            _refuse_devices("paged_append", k_pages, q, q_out)
        if q.dtype is not dtype or (q_out is not None and q_out.dtype is not dtype):
            raise TypeError("q and q_out must have the dtype of the pages")
        q_shape, qs = q.shape, q.stride()
        if len(q_shape) != 4:
            raise ValueError("q must be [batch, heads, rows, head_dim]")
        heads = q_shape[1]
        if q_shape[0] != B or q_shape[2] != rows or q_shape[3] != head_dim or qs[3] != 1:
            _refuse_shape("q", q, (B, heads, rows, head_dim))
        if q_out is None:
            q_out = torch.empty(B, rows, heads, head_dim, dtype=dtype, device=k_pages.device).permute(0, 2, 1, 3)
        os_ = q_out.stride()
        if q_out.shape != q_shape or os_[3] != 1:
            _refuse_shape("q_out", q_out, q_shape)
    elif q_out is not None:
        raise ValueError("q_out goes with q")
    if B == 0 or rows == 0:
        return q_out
    desc = _APPEND.pack(number, B, kv_heads, head_dim, page_size, pages, columns, 0, table_stride, k_pages.data_ptr(),
                        v_pages.data_ptr(), page_table.data_ptr(), rows, heads, rotated, interleaved, k.data_ptr(), v.data_ptr(),
                        q.data_ptr() if heads else 0, q_out.data_ptr() if heads else 0, ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], qs[0],
                        qs[1], qs[2], os_[0], os_[1], os_[2], start.data_ptr(),
                        counts.data_ptr() if counts is not None else 0, inv_freq.data_ptr() if rotated else 0)
    _native.launch(index, _native.lib().tmw_paged_append, desc)
    return q_out


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, pos: torch.Tensor,
                    window: Optional[int] = None, k_pers: Optional[torch.Tensor] = None, v_pers: Optional[torch.Tensor] = None,
                    scale: float = 0.0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of the newest token of every sequence, ``q [B, heads, dh]`` at ``pos[b]`` (int32 ``[B]``), whose keys and values
    have been appended: over tokens ``pos - window .. pos`` (None: all up to ``pos``) and the persistent keys
    ``k_pers, v_pers [kv_heads, Np, dh]``.  ``heads`` is a multiple of the pages' ``kv_heads``.  ``pos`` of -1: a sequence without
    tokens; it sees the persistent keys, and is zero without them.  ``out`` must not overlap ``q``.  Serving only: the output carries
    no gradient."""
    index = k_pages.get_device()
    if not 0 <= index == q.get_device() == v_pages.get_device() == page_table.get_device() == pos.get_device():
        _refuse_devices("paged_attention", k_pages, q, v_pages, page_table, pos)
    dtype = k_pages.dtype
    if not (dtype is v_pages.dtype is q.dtype and torch.int32 is page_table.dtype is pos.dtype):
        raise TypeError("paged_attention: q and the pages must share one dtype; page_table and pos must be int32")
    _native.refuse_tangents("paged_attention", q, k_pages, v_pages, k_pers, v_pers)
    shape = q.shape
    if len(shape) != 3:
        raise ValueError("paged_attention: q must be [batch, heads, head_dim]")
    B, heads, _ = shape
    number, kv_heads, head_dim, page_size, pages, columns, table_stride = _page_numbers("paged_attention", k_pages, v_pages, page_table,
                                                                                        B)
    if kv_heads == 0 or heads % kv_heads != 0:
        raise ValueError(f"heads ({heads}) must be a multiple of kv_heads ({kv_heads})")
    qs = q.stride()
    if shape[2] != head_dim or qs[2] != 1:
        _refuse_shape("q", q, (B, heads, head_dim))
    _check_numbers("pos", pos, B)
    if window is None:
        window = -1
    elif window < 0:
        raise ValueError(f"window_size must be non-negative, got {window}")
    elif window > 0x7FFFFFFF:
        window = -1  # (no sequence is longer)
    n_persistent = 0
    if k_pers is not None and v_pers is not None:
        if not index == k_pers.get_device() == v_pers.get_device():
            _refuse_devices("paged_attention", k_pages, k_pers, v_pers)
        if not dtype is k_pers.dtype is v_pers.dtype:
            raise TypeError("k_pers and v_pers must have the dtype of the pages")
        pers = k_pers.shape
        if len(pers) != 3 or pers[0] != kv_heads or pers[2] != head_dim or v_pers.shape != pers or not k_pers.is_contiguous() \
                or not v_pers.is_contiguous():
            raise ValueError("k_pers and v_pers must be contiguous [kv_heads, n_persistent, head_dim]")
        n_persistent = pers[1]
    elif k_pers is not None or v_pers is not None:
        raise ValueError("k_pers and v_pers go together")
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else torch.empty(B, heads, head_dim, dtype=dtype, device=q.device)
    else:
        if out.get_device() != index:
            _refuse_devices("paged_attention", k_pages, out)
        if out.dtype is not dtype:
            raise TypeError("out must have the dtype of the pages")
        if out.data_ptr() == q.data_ptr() and q.numel():
            raise ValueError("out must not be q")
    os_ = out.stride()
    if out.shape != shape or os_[2] != 1:
        _refuse_shape("out", out, shape)
    if B == 0 or heads == 0:
        return out
    desc = _ATTENTION.pack(number, B, kv_heads, head_dim, page_size, pages, columns, 0, table_stride,
                           k_pages.data_ptr(), v_pages.data_ptr(), page_table.data_ptr(), heads, n_persistent, window, scale,
                           q.data_ptr(), k_pers.data_ptr() if n_persistent else 0, v_pers.data_ptr() if n_persistent else 0,
                           out.data_ptr(), qs[0], qs[1], os_[0], os_[1], pos.data_ptr())
    lib, device = _native.lib(), k_pages.device
    with _native._on(device):  # (how much depends on the device's SMs)
        nbytes = lib.tmw_paged_attention_scratch_bytes(desc)
    # of this call alone: calls on two streams, or of two captured graphs, have nothing in common
    scratch = torch.empty(nbytes, dtype=torch.uint8, device=device)
    _native.launch(index, lib.tmw_paged_attention, desc, scratch.data_ptr() or None, nbytes)
    return out


class PagedCache:
    """One layer's keys and values in pages, for the calls that take a ``RingCache``: ``TitanMAC.prefill`` and ``decode_step``,
    or ``fill`` and ``decode`` directly.  The layers of a model share one ``page_table [B, columns]`` (int32, on the device)."""

    def __init__(self, page_table: torch.Tensor, pages: int, page_size: int, kv_heads: int, head_dim: int, window: Optional[int],
                 n_persistent: int, dtype: torch.dtype, scale: float = 0.0, inv_freq: Optional[torch.Tensor] = None,
                 interleaved: bool = False):
        if dtype not in _native._DTYPES:
            raise TypeError("dtype must be float32, bfloat16 or float16")
        if window is not None and window < 0:
            raise ValueError(f"window_size must be non-negative, got {window}")
        if pages < 0 or page_size <= 0 or kv_heads <= 0 or head_dim <= 0 or n_persistent < 0:
            raise ValueError("a paged cache needs pages of at least one token, heads and their dimensions")
        _native._require_cuda(page_table)
        self.page_table, self.page_size, self.window, self.scale = page_table, page_size, window, scale
        self.kv_heads, self.head_dim, self.n_persistent, self.dtype = kv_heads, head_dim, n_persistent, dtype
        self.inv_freq, self.interleaved = inv_freq, interleaved
        self.device = page_table.device
        self.geometry = ("paged", page_table.shape[0], kv_heads, head_dim, window, n_persistent, dtype)  # no RingCache's
        self.k_pages = torch.zeros((pages, kv_heads, page_size, head_dim), dtype=dtype, device=self.device)
        self.v_pages = torch.zeros_like(self.k_pages)
        self.k_pers = torch.zeros((kv_heads, n_persistent, head_dim), dtype=dtype, device=self.device)
        self.v_pers = torch.zeros_like(self.k_pers)

    def set_persistent(self, k_pers: torch.Tensor, v_pers: torch.Tensor) -> None:
        """``[kv_heads, Np, dh]`` keys/values of the persistent rows (identical for every sequence, not rotated)."""
        self.k_pers.copy_(k_pers)
        self.v_pers.copy_(v_pers)

    def append(self, k: torch.Tensor, v: torch.Tensor, start: torch.Tensor, counts: Optional[torch.Tensor] = None,
               q: Optional[torch.Tensor] = None, q_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
        """``paged_append`` with this cache's rotation."""
        return paged_append(k, v, self.k_pages, self.v_pages, self.page_table, start, counts, q, q_out, self.inv_freq,
                            self.interleaved)

    def attend(self, q: torch.Tensor, pos: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """``paged_attention`` of queries that are rotated already."""
        pers = (self.k_pers, self.v_pers) if self.n_persistent else (None, None)
        return paged_attention(q, self.k_pages, self.v_pages, self.page_table, pos, self.window, *pers, self.scale, out)

    def fill(self, k: torch.Tensor, v: torch.Tensor, t0: int = 0, counts: Optional[torch.Tensor] = None) -> None:
        """Rows ``k, v [B, kv_heads, rows, dh]`` as tokens ``t0 ..`` of every sequence, the first ``counts[b]`` of them."""
        if t0 < 0:
            raise ValueError("t0 must not be negative")
        self.append(k, v, torch.full((k.shape[0],), t0, dtype=torch.int32, device=self.device), counts)

    def decode(self, q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor, pos: torch.Tensor,
               out: Optional[torch.Tensor] = None, seen: Optional[torch.Tensor] = None) -> torch.Tensor:
        """One step: ``q [B, heads, dh]``, ``k_new, v_new [B, kv_heads, dh]``, ``pos [B] int32`` (index of the new token; -1: no
        sequence in this row).  Appends, rotates if the cache does, and attends, at ``seen [B]`` instead of ``pos`` if it is
        given (the caller's way of declaring a row wrong: -2)."""
        if self.inv_freq is None:
            self.append(k_new.unsqueeze(2), v_new.unsqueeze(2), pos)
        else:
            # (the row of a missing sequence is read by nothing but its own attention: zeros, not what memory held)
            turned = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
            self.append(k_new.unsqueeze(2), v_new.unsqueeze(2), pos, q=q.unsqueeze(2), q_out=turned.unsqueeze(2))
            q = turned
        return self.attend(q, pos if seen is None else seen, out)
