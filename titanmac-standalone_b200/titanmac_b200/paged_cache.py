"""Keys and values in pages that sequences share a pool of (``tmw_paged_append``, ``tmw_paged_attention`` and what goes with them).

``RingCache`` keeps ``window + 1`` slots for every sequence of a fixed batch.  Here a sequence has as many pages of ``page_size``
tokens as it needs, anywhere in the pool: token ``t`` of sequence ``b`` is in slot ``t % page_size`` of page
``page_table[b, t // page_size]``.  Who hands out pages writes the table (on the device, in place if the calls are captured in a
graph); entries that no token needs may hold anything.  Sequences may share pages that nobody writes to, a batch may hold rows
without a sequence (``start`` / ``pos`` of -1), query heads may share key heads, and keys and queries can be rotated by their
positions on the way into the cache.

Pages hold the model's type, or 8 bits: ``int8`` or ``float8_e4m3fn`` codes with an fp32 scale for every token and key head, half the
memory and half the traffic.  ``scales``, a pair ``(k_scales, v_scales)`` of ``[pages, kv_heads, page_size]``, goes with such pages
wherever these go; a code stands for itself times its row's scale.  A row is written with ``scale = max(max |x| / largest, 2^-100)``,
``largest`` 127 or 448, and the codes nearest to ``x / scale``; one with a NaN or an infinity reads as NaN.  Beside values that are all
zeros others may be up to 2^18 (scales 2^112 apart): beyond that the attention may leave the zeros out of its sum of weights.

Drafted tokens: ``paged_append`` takes several rows of a sequence, with ``positions`` if they form a tree, ``paged_tree_attention``
attends with all of them at once, and ``paged_keep`` moves the accepted ones together.

Serving only: no gradient flows through these calls (inputs that require one are taken as they are; forward-mode derivatives are
refused).

What the device finds wrong - a position or a page outside the table or the pool - makes NaN of what depends on it, touches nothing
else and is raised by ``_native.poll_status``.
"""

from __future__ import annotations

import struct
from typing import NamedTuple, Optional, Tuple

import torch

from . import _native

# tmw_pages; behind it the fields of tmw_paged_append_desc, of tmw_paged_attention_desc and so on
_APPEND = struct.Struct("@8iq3Q 4i 4Q 12q 3Q")
_ATTENTION = struct.Struct("@8iq3Q 3if 4Q 4q Q")
_READ = struct.Struct("@8iq3Q 2i 2Q 6q 2Q")
_TREE = struct.Struct("@8iq3Q 4ifi 4Q 6q 4Q")
_KEEP = struct.Struct("@8iq3Q 2i 3Q")
_SCALES = struct.Struct("@2i 4Q")  # tmw_page_scales
_FORMATS = {torch.int8: 1, torch.float8_e4m3fn: 2}
MAX_NODES = 64

Scales = Tuple[torch.Tensor, torch.Tensor]


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
    dtype = _native._DTYPES.get(k_pages.dtype, -1)  # (-1: of 8 bits)
    if dtype < 0 and k_pages.dtype not in _FORMATS:
        raise TypeError(f"{name}: pages in float32, bfloat16, float16, int8 or float8_e4m3fn expected")
    return dtype, shape[1], shape[3], shape[2], shape[0], table[1], strides[0]


def _number_of(name: str, dtype: torch.dtype) -> int:
    number = _native._DTYPES.get(dtype)
    if number is None:
        raise TypeError(f"{name}: queries, keys and values in float32, bfloat16 or float16 expected")
    return number


def _check_scales(name: str, scales: Optional[Scales], index: int, shape, what: str) -> Scales:
    if scales is None or len(scales) != 2:
        raise ValueError(f"{name}: pages of 8 bits go with {what}, a pair of tensors")
    _native.refuse_tangents(name, *scales)
    for t in scales:
        if t.get_device() != index:
            _native._require_cuda(t)
            raise ValueError(f"{name}: every tensor must be on one device")
        if t.dtype is not torch.float32:
            raise TypeError(f"{name}: {what} must be float32")
        if t.shape != shape or not t.is_contiguous():
            raise ValueError(f"{name}: {what} must be contiguous {list(shape)}")
    return scales


def _scale_numbers(name: str, k_pages: torch.Tensor, v_pages: torch.Tensor, scales: Optional[Scales],
                   pers_scales: Optional[Scales] = None, pers_shape=None) -> Optional[bytes]:
    """tmw_page_scales of checked scales; None for pages of the model's type."""
    form = _FORMATS.get(k_pages.dtype)
    if v_pages.dtype is not k_pages.dtype:
        raise TypeError(f"{name}: k_pages and v_pages must share one dtype")
    if form is None:
        if scales is not None or pers_scales is not None:
            raise ValueError(f"{name}: scales go with pages of 8 bits")
        return None
    if k_pages.shape[3] % 16 != 0:
        raise ValueError(f"{name}: head_dim must be a multiple of 16 with pages of 8 bits")
    index = k_pages.get_device()
    ks, vs = _check_scales(name, scales, index, k_pages.shape[:3], "scales")
    kp = vp = 0
    if pers_shape is not None:
        kp, vp = (t.data_ptr() for t in _check_scales(name, pers_scales, index, pers_shape, "pers_scales"))
    return _SCALES.pack(form, 0, ks.data_ptr(), vs.data_ptr(), kp, vp)


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
                 interleaved: bool = False, *, scales: Optional[Scales] = None,
                 positions: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """New tokens into the pages: row ``r`` of ``k, v [B, kv_heads, rows, dh]`` (any strides, last axis contiguous) is token
    ``start[b] + r`` of sequence ``b``; rows from ``counts[b]`` on are left out (``start``, ``counts``: int32 ``[B]``).

    ``inv_freq`` (fp32, at most ``dh / 2`` numbers): the first ``2 * len(inv_freq)`` numbers of every key are rotated in pairs,
    pair ``i`` by ``t * inv_freq[i]`` at token ``t``; the pairs are ``(i, i + len(inv_freq))`` or, ``interleaved``,
    ``(2 i, 2 i + 1)``.  ``q [B, heads, rows, dh]`` is rotated likewise into ``q_out`` (may be ``q``; made if None), which is
    returned; its rows that are no new token's are left as they are.  ``positions`` (int32 ``[B, rows]``): what the rows are rotated by
    instead of ``t``.  ``scales``: of pages of 8 bits, written too.  Writes of the same slot twice in one call are the caller's
    to avoid.  Serving only: nothing that is returned or written carries a gradient."""
    index = k_pages.get_device()
    if not 0 <= index == k.get_device() == v.get_device() == v_pages.get_device() == page_table.get_device() == start.get_device():
        _refuse_devices("paged_append", k_pages, k, v, v_pages, page_table, start)
    dtype = k.dtype
    eight = k_pages.dtype in _FORMATS
    if not (dtype is v.dtype and (eight or dtype is k_pages.dtype) and k_pages.dtype is v_pages.dtype
            and torch.int32 is page_table.dtype is start.dtype):
        raise TypeError("paged_append: k, v and the pages must share one dtype; page_table and start must be int32")
    _native.refuse_tangents("paged_append", k, v, k_pages, v_pages, q, inv_freq)
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
    if positions is not None:
        if positions.get_device() != index:
            _refuse_devices("paged_append", k_pages, positions)
        if positions.dtype is not torch.int32 or positions.shape != (B, rows) or not positions.is_contiguous():
            raise TypeError("positions must be contiguous int32 [batch, rows]")
    scaled = None
    if eight or scales is not None:
        scaled = _scale_numbers("paged_append", k_pages, v_pages, scales)
        number = _number_of("paged_append", dtype)
    heads, qs, os_ = 0, (0, 0, 0, 1), (0, 0, 0, 1)
    if q is not None:
        if q.get_device() != index or (q_out is not None and q_out.get_device() != index):
            _refuse_devices("paged_append", k_pages, q, q_out)
        if q.dtype is not dtype or (q_out is not None and q_out.dtype is not dtype):
            raise TypeError("q and q_out must have the dtype of k and v")
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
    if scaled is None and positions is None:
        _native.launch(index, _native.lib().tmw_paged_append, desc)
    else:
        _native.launch(index, _native.lib().tmw_paged_append_scaled, desc, scaled, positions.data_ptr() if positions is not None else None)
    return q_out


def paged_read(k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, start: torch.Tensor, rows: Optional[int] = None,
               counts: Optional[torch.Tensor] = None, dtype: Optional[torch.dtype] = None, *, scales: Optional[Scales] = None,
               k_out: Optional[torch.Tensor] = None, v_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Keys and values back from their pages, ``(k, v)`` of ``[B, kv_heads, rows, dh]``: row ``r`` is token ``start[b] + r``, as keys
    were written (rotated, if they were).  From pages of 8 bits the products of codes and ``scales``, in ``dtype``.  Rows from
    ``counts[b]`` on, and every row where ``start`` is -1, are left as they are in ``k_out`` and ``v_out`` (any strides, last axis contiguous;
    made, of zeros, if None: then ``rows`` and, for pages of 8 bits, ``dtype`` are needed).  For what takes dense keys: a further piece of a
    prompt, another cache."""
    index = k_pages.get_device()
    if not 0 <= index == v_pages.get_device() == page_table.get_device() == start.get_device():
        _refuse_devices("paged_read", k_pages, v_pages, page_table, start)
    if not (k_pages.dtype is v_pages.dtype and torch.int32 is page_table.dtype is start.dtype):
        raise TypeError("paged_read: the pages must share one dtype; page_table and start must be int32")
    _native.refuse_tangents("paged_read", k_pages, v_pages, k_out, v_out)
    if start.dim() != 1:
        raise ValueError("start must be a contiguous vector of one number per sequence")
    B = start.shape[0]
    number, kv_heads, head_dim, page_size, pages, columns, table_stride = _page_numbers("paged_read", k_pages, v_pages, page_table, B)
    _check_numbers("start", start, B)
    if counts is not None:
        if counts.get_device() != index:
            _refuse_devices("paged_read", k_pages, counts)
        if counts.dtype is not torch.int32:
            raise TypeError("counts must be int32")
        _check_numbers("counts", counts, B)
    if (k_out is None) != (v_out is None):
        raise ValueError("k_out and v_out go together")
    if k_out is None:
        if rows is None or rows < 0:
            raise ValueError("paged_read: rows, the number of tokens of a sequence, is needed without k_out and v_out")
        if dtype is None:
            if number < 0:
                raise ValueError("paged_read: pages of 8 bits need the dtype to read them in")
            dtype = k_pages.dtype
        _number_of("paged_read", dtype)
        k_out, v_out = (torch.zeros(B, kv_heads, rows, head_dim, dtype=dtype, device=k_pages.device) for _ in range(2))
    else:
        if not index == k_out.get_device() == v_out.get_device():
            _refuse_devices("paged_read", k_pages, k_out, v_out)
        if k_out.dtype is not v_out.dtype or (dtype is not None and k_out.dtype is not dtype):
            raise TypeError("paged_read: k_out and v_out must share one dtype")
        dtype = k_out.dtype
        if k_out.dim() != 4 or (rows is not None and k_out.shape[2] != rows):
            raise ValueError("k_out must be [batch, kv_heads, rows, head_dim]")
        rows = k_out.shape[2]
    if number >= 0 and dtype is not k_pages.dtype:
        raise TypeError("paged_read: pages of the model's type are read in it")
    shape, ks, vs = (B, kv_heads, rows, head_dim), k_out.stride(), v_out.stride()
    if k_out.shape != shape or ks[3] != 1:
        _refuse_shape("k_out", k_out, shape)
    if v_out.shape != shape or vs[3] != 1:
        _refuse_shape("v_out", v_out, shape)
    scaled = _scale_numbers("paged_read", k_pages, v_pages, scales)
    number = _number_of("paged_read", dtype)
    if B == 0 or rows == 0:
        return k_out, v_out
    desc = _READ.pack(number, B, kv_heads, head_dim, page_size, pages, columns, 0, table_stride, k_pages.data_ptr(), v_pages.data_ptr(),
                      page_table.data_ptr(), rows, 0, k_out.data_ptr(), v_out.data_ptr(), ks[0], ks[1], ks[2], vs[0], vs[1], vs[2],
                      start.data_ptr(), counts.data_ptr() if counts is not None else 0)
    _native.launch(index, _native.lib().tmw_paged_read, desc, scaled)
    return k_out, v_out


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, pos: torch.Tensor,
                    window: Optional[int] = None, k_pers: Optional[torch.Tensor] = None, v_pers: Optional[torch.Tensor] = None,
                    scale: float = 0.0, out: Optional[torch.Tensor] = None, *, scales: Optional[Scales] = None,
                    pers_scales: Optional[Scales] = None) -> torch.Tensor:
    """Attention of the newest token of every sequence, ``q [B, heads, dh]`` at ``pos[b]`` (int32 ``[B]``), whose keys and values
    have been appended: over tokens ``pos - window .. pos`` (None: all up to ``pos``) and the persistent keys
    ``k_pers, v_pers [kv_heads, Np, dh]``.  ``heads`` is a multiple of the pages' ``kv_heads``.  ``pos`` of -1: a sequence without
    tokens; it sees the persistent keys, and is zero without them.  ``out`` must not overlap ``q``.  ``scales``: of pages of 8 bits; the
    persistent keys are then in the same form, ``pers_scales`` a pair of ``[kv_heads, Np]``.  Serving only: the output carries no
    gradient."""
    index = k_pages.get_device()
    if not 0 <= index == q.get_device() == v_pages.get_device() == page_table.get_device() == pos.get_device():
        _refuse_devices("paged_attention", k_pages, q, v_pages, page_table, pos)
    dtype = q.dtype
    held = k_pages.dtype
    eight = held in _FORMATS
    if not (held is v_pages.dtype and (eight or held is dtype) and torch.int32 is page_table.dtype is pos.dtype):
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
    if k_pers is not None or v_pers is not None:
        n_persistent = _check_persistent("paged_attention", k_pages, index, kv_heads, head_dim, k_pers, v_pers)
    scaled = None
    if eight or scales is not None or pers_scales is not None:
        scaled = _scale_numbers("paged_attention", k_pages, v_pages, scales, pers_scales, (kv_heads, n_persistent) if n_persistent else None)
        number = _number_of("paged_attention", dtype)
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else torch.empty(B, heads, head_dim, dtype=dtype, device=q.device)
    else:
        if out.get_device() != index:
            _refuse_devices("paged_attention", k_pages, out)
        if out.dtype is not dtype:
            raise TypeError("out must have the dtype of q")
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
    # (how much depends on the device's SMs)
    nbytes = (_native.ask(index, lib.tmw_paged_attention_scratch_bytes, desc) if scaled is None
              else _native.ask(index, lib.tmw_paged_attention_scaled_scratch_bytes, desc, scaled))
    # of this call alone: calls on two streams, or of two captured graphs, have nothing in common
    scratch = torch.empty(nbytes, dtype=torch.uint8, device=device)
    if scaled is None:
        _native.launch(index, lib.tmw_paged_attention, desc, scratch.data_ptr() or None, nbytes)
    else:
        _native.launch(index, lib.tmw_paged_attention_scaled, desc, scaled, scratch.data_ptr() or None, nbytes)
    return out


def _check_persistent(name: str, k_pages: torch.Tensor, index: int, kv_heads: int, head_dim: int, k_pers: Optional[torch.Tensor],
                      v_pers: Optional[torch.Tensor]) -> int:
    """How many persistent keys there are."""
    if k_pers is None or v_pers is None:
        raise ValueError("k_pers and v_pers go together")
    if not index == k_pers.get_device() == v_pers.get_device():
        _refuse_devices(name, k_pages, k_pers, v_pers)
    if not k_pages.dtype is k_pers.dtype is v_pers.dtype:
        raise TypeError("k_pers and v_pers must have the dtype of the pages")
    pers = k_pers.shape
    if len(pers) != 3 or pers[0] != kv_heads or pers[2] != head_dim or v_pers.shape != pers or not k_pers.is_contiguous() \
            or not v_pers.is_contiguous():
        raise ValueError("k_pers and v_pers must be contiguous [kv_heads, n_persistent, head_dim]")
    return pers[1]


class DraftTree(NamedTuple):
    """What ``paged_tree_attention`` and ``paged_append`` ask of a tree: ``seen [B, nodes]`` (int64, bit ``j`` of entry ``i``: node ``i``
    sees node ``j``) and ``positions [B, nodes]`` (int32)."""

    seen: torch.Tensor
    positions: torch.Tensor


def draft_tree(parents: torch.Tensor, start: torch.Tensor, window: Optional[int] = None) -> DraftTree:
    """``parents [B, nodes]`` (int32 or int64, at most 64 nodes): node ``i``'s parent, an earlier node, or -1 where it follows the cached
    tokens.  ``start [B]``: how many these are.  A node sees its ancestors and itself, with a ``window`` those of its last ``window``
    positions; its position is ``start`` plus how far it is from the root."""
    if parents.dim() != 2 or parents.shape[1] > MAX_NODES or parents.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"parents must be int32 or int64 [batch, nodes], at most {MAX_NODES} nodes")
    B, N = parents.shape
    if start.shape != (B,):
        raise ValueError("start must be a vector of one number per sequence")
    up = parents.long()
    at = torch.arange(N, device=parents.device)
    one = (torch.ones_like(at) << at).expand(B, N)
    if window is not None and window < 0:
        raise ValueError(f"window_size must be non-negative, got {window}")
    # whoever is not an earlier node is nobody; 2^i ancestors more by the i-th step
    up = torch.where((up >= 0) & (up < at), up, torch.full_like(up, -1))
    seen, depth = one, (up >= 0).long()
    steps, reach = 0, up
    while (1 << steps) < N:
        there, of = reach >= 0, reach.clamp(min=0)
        seen = torch.where(there, seen | seen.gather(1, of), seen)
        depth = torch.where(there, depth + depth.gather(1, of), depth)
        reach = torch.where(there, reach.gather(1, of), reach)
        steps += 1
    if window is not None and window < N:
        near = depth[:, None, :] >= depth[:, :, None] - window  # [B, node, seen]
        seen = seen & (near.long() << at).sum(dim=-1)
    return DraftTree(seen.contiguous(), (start.long()[:, None] + depth).to(torch.int32))


def paged_tree_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, start: torch.Tensor,
                         seen: torch.Tensor, counts: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None,
                         window: Optional[int] = None, k_pers: Optional[torch.Tensor] = None, v_pers: Optional[torch.Tensor] = None,
                         scale: float = 0.0, out: Optional[torch.Tensor] = None, *, scales: Optional[Scales] = None,
                         pers_scales: Optional[Scales] = None) -> torch.Tensor:
    """Attention of several drafted tokens of every sequence at once, ``q [B, heads, nodes, dh]`` (any strides, last axis contiguous; at
    most 64 nodes), whose keys and values have been appended as tokens ``start[b] ..``.  Node ``i`` of sequence ``b`` sees the persistent
    keys, the ``start[b]`` tokens in front of the drafts (with a ``window`` those from ``positions[b, i] - window`` on), and the nodes
    whose bits are set in ``seen[b, i]`` (``draft_tree`` makes both of a tree; a row of new tokens one after the other is one too).  A
    sequence has ``counts[b]`` nodes (int32; None: all); rows of ``out`` behind them, and of a sequence with a ``start`` of -1, are left as they
    are (zeros, if ``out`` is made).  A node that sees nothing has zero.  ``out`` must not overlap ``q``; ``scales`` and ``pers_scales`` as
    for ``paged_attention``.  Serving only: the output carries no gradient."""
    index = k_pages.get_device()
    if not 0 <= index == q.get_device() == v_pages.get_device() == page_table.get_device() == start.get_device() == seen.get_device():
        _refuse_devices("paged_tree_attention", k_pages, q, v_pages, page_table, start, seen)
    dtype, held = q.dtype, k_pages.dtype
    eight = held in _FORMATS
    if not (held is v_pages.dtype and (eight or held is dtype) and torch.int32 is page_table.dtype is start.dtype):
        raise TypeError("paged_tree_attention: q and the pages must share one dtype; page_table and start must be int32")
    _native.refuse_tangents("paged_tree_attention", q, k_pages, v_pages, k_pers, v_pers)
    shape = q.shape
    if len(shape) != 4:
        raise ValueError("paged_tree_attention: q must be [batch, heads, nodes, head_dim]")
    B, heads, nodes, _ = shape
    number, kv_heads, head_dim, page_size, pages, columns, table_stride = _page_numbers("paged_tree_attention", k_pages, v_pages,
                                                                                        page_table, B)
    if kv_heads == 0 or heads % kv_heads != 0:
        raise ValueError(f"heads ({heads}) must be a multiple of kv_heads ({kv_heads})")
    if nodes > MAX_NODES:
        raise ValueError(f"paged_tree_attention: at most {MAX_NODES} nodes, got {nodes}")
    qs = q.stride()
    if shape[3] != head_dim or qs[3] != 1:
        _refuse_shape("q", q, (B, heads, nodes, head_dim))
    _check_numbers("start", start, B)
    if seen.dtype is not torch.int64:
        raise TypeError("seen must be int64")
    if seen.shape != (B, nodes) or not seen.is_contiguous():
        raise ValueError("seen must be contiguous [batch, nodes]")
    if counts is not None:
        if counts.get_device() != index:
            _refuse_devices("paged_tree_attention", k_pages, counts)
        if counts.dtype is not torch.int32:
            raise TypeError("counts must be int32")
        _check_numbers("counts", counts, B)
    if window is None or window > 0x7FFFFFFF:  # (no sequence is longer)
        window = -1
    elif window < 0:
        raise ValueError(f"window_size must be non-negative, got {window}")
    elif positions is None:
        raise ValueError("a window goes with the nodes' positions")
    if positions is not None:
        if positions.get_device() != index:
            _refuse_devices("paged_tree_attention", k_pages, positions)
        if positions.dtype is not torch.int32:
            raise TypeError("positions must be int32")
        if positions.shape != (B, nodes) or not positions.is_contiguous():
            raise ValueError("positions must be contiguous [batch, nodes]")
    n_persistent = 0
    if k_pers is not None or v_pers is not None:
        n_persistent = _check_persistent("paged_tree_attention", k_pages, index, kv_heads, head_dim, k_pers, v_pers)
    scaled = None
    if eight or scales is not None or pers_scales is not None:
        scaled = _scale_numbers("paged_tree_attention", k_pages, v_pages, scales, pers_scales,
                                (kv_heads, n_persistent) if n_persistent else None)
        number = _number_of("paged_tree_attention", dtype)
    if out is None:
        out = torch.zeros(B, nodes, heads, head_dim, dtype=dtype, device=q.device).permute(0, 2, 1, 3)
    else:
        if out.get_device() != index:
            _refuse_devices("paged_tree_attention", k_pages, out)
        if out.dtype is not dtype:
            raise TypeError("out must have the dtype of q")
        if out.data_ptr() == q.data_ptr() and q.numel():
            raise ValueError("out must not be q")
    os_ = out.stride()
    if out.shape != shape or os_[3] != 1:
        _refuse_shape("out", out, shape)
    if B == 0 or heads == 0 or nodes == 0:
        return out
    desc = _TREE.pack(number, B, kv_heads, head_dim, page_size, pages, columns, 0, table_stride, k_pages.data_ptr(), v_pages.data_ptr(),
                      page_table.data_ptr(), heads, nodes, n_persistent, window, scale, 0, q.data_ptr(),
                      k_pers.data_ptr() if n_persistent else 0, v_pers.data_ptr() if n_persistent else 0, out.data_ptr(), qs[0], qs[1],
                      qs[2], os_[0], os_[1], os_[2], start.data_ptr(), counts.data_ptr() if counts is not None else 0,
                      positions.data_ptr() if positions is not None else 0, seen.data_ptr())
    lib, device = _native.lib(), k_pages.device
    nbytes = _native.ask(index, lib.tmw_paged_tree_attention_scratch_bytes, desc, scaled)
    scratch = torch.empty(nbytes, dtype=torch.uint8, device=device)  # (of this call alone)
    _native.launch(index, lib.tmw_paged_tree_attention, desc, scaled, scratch.data_ptr() or None, nbytes)
    return out


def paged_keep(k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor, start: torch.Tensor, kept: torch.Tensor,
               counts: torch.Tensor, *, scales: Optional[Scales] = None) -> None:
    """Tokens ``start[b] + kept[b, i]`` become tokens ``start[b] + i``, for ``i < counts[b]``: the accepted path of a drafted tree, its
    keys, values and ``scales`` moved together in their pages.  ``kept`` (int32 ``[B, most]``, at most 64) rises along a row, with
    ``kept[b, i] >= i``; ``start`` of -1: nothing of that sequence moves.  What does not hold is left as it is and raised by
    ``_native.poll_status``."""
    index = k_pages.get_device()
    if not 0 <= index == v_pages.get_device() == page_table.get_device() == start.get_device() == kept.get_device() == counts.get_device():
        _refuse_devices("paged_keep", k_pages, v_pages, page_table, start, kept, counts)
    if not (k_pages.dtype is v_pages.dtype and torch.int32 is page_table.dtype is start.dtype is kept.dtype is counts.dtype):
        raise TypeError("paged_keep: the pages must share one dtype; page_table, start, kept and counts must be int32")
    _native.refuse_tangents("paged_keep", k_pages, v_pages)
    if kept.dim() != 2 or not kept.is_contiguous():
        raise ValueError("kept must be contiguous [batch, most]")
    B, most = kept.shape
    if most > MAX_NODES:
        raise ValueError(f"paged_keep: at most {MAX_NODES} tokens of a sequence, got {most}")
    number, kv_heads, head_dim, page_size, pages, columns, table_stride = _page_numbers("paged_keep", k_pages, v_pages, page_table, B)
    _check_numbers("start", start, B)
    _check_numbers("counts", counts, B)
    scaled = _scale_numbers("paged_keep", k_pages, v_pages, scales)
    if B == 0 or most == 0:
        return
    desc = _KEEP.pack(max(number, 0), B, kv_heads, head_dim, page_size, pages, columns, 0, table_stride, k_pages.data_ptr(),
                      v_pages.data_ptr(), page_table.data_ptr(), most, 0, start.data_ptr(), kept.data_ptr(), counts.data_ptr())
    _native.launch(index, _native.lib().tmw_paged_keep, desc, scaled)


class PagedCache:
    """One layer's keys and values in pages, for the calls that take a ``RingCache``: ``TitanMAC.prefill`` and ``decode_step``,
    or ``fill`` and ``decode`` directly.  ``page_dtype`` (int8 or float8_e4m3fn) holds keys, values and the persistent ones in 8 bits.  The
    layers of a model share one ``page_table [B, columns]`` (int32, on the device)."""

    def __init__(self, page_table: torch.Tensor, pages: int, page_size: int, kv_heads: int, head_dim: int, window: Optional[int],
                 n_persistent: int, dtype: torch.dtype, scale: float = 0.0, inv_freq: Optional[torch.Tensor] = None,
                 interleaved: bool = False, page_dtype: Optional[torch.dtype] = None):
        if dtype not in _native._DTYPES:
            raise TypeError("dtype must be float32, bfloat16 or float16")
        page_dtype = dtype if page_dtype is None else page_dtype
        if page_dtype is not dtype and page_dtype not in _FORMATS:
            raise TypeError("page_dtype must be the dtype, int8 or float8_e4m3fn")
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
        self.k_pages = torch.zeros((pages, kv_heads, page_size, head_dim), dtype=page_dtype, device=self.device)
        self.v_pages = torch.zeros_like(self.k_pages)
        self.k_pers = torch.zeros((kv_heads, n_persistent, head_dim), dtype=page_dtype, device=self.device)
        self.v_pers = torch.zeros_like(self.k_pers)
        self.scales = self.pers_scales = None
        if page_dtype is not dtype:
            if head_dim % 16 != 0:
                raise ValueError("head_dim must be a multiple of 16 with pages of 8 bits")
            self.scales, self.pers_scales = (tuple(torch.ones(t.shape[:-1], dtype=torch.float32, device=self.device) for _ in range(2))
                                             for t in (self.k_pages, self.k_pers))
            self._one_page = torch.zeros((1, 1), dtype=torch.int32, device=self.device)

    def set_persistent(self, k_pers: torch.Tensor, v_pers: torch.Tensor) -> None:
        """``[kv_heads, Np, dh]`` keys/values of the persistent rows (identical for every sequence, not rotated)."""
        if self.scales is None:
            self.k_pers.copy_(k_pers)
            self.v_pers.copy_(v_pers)
        elif self.n_persistent:  # as one page, of tokens from 0 on
            k, v = (t[None].to(device=self.device, dtype=self.dtype).contiguous() for t in (k_pers, v_pers))
            paged_append(k, v, self.k_pers[None], self.v_pers[None], self._one_page, self._one_page[0],
                         scales=tuple(t[None] for t in self.pers_scales))

    def append(self, k: torch.Tensor, v: torch.Tensor, start: torch.Tensor, counts: Optional[torch.Tensor] = None,
               q: Optional[torch.Tensor] = None, q_out: Optional[torch.Tensor] = None,
               positions: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
        """``paged_append`` with this cache's rotation."""
        return paged_append(k, v, self.k_pages, self.v_pages, self.page_table, start, counts, q, q_out, self.inv_freq,
                            self.interleaved, scales=self.scales, positions=positions)

    def read(self, start: torch.Tensor, rows: int, counts: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """``paged_read`` in this cache's dtype."""
        return paged_read(self.k_pages, self.v_pages, self.page_table, start, rows, counts, self.dtype, scales=self.scales)

    def keep(self, start: torch.Tensor, kept: torch.Tensor, counts: torch.Tensor) -> None:
        """``paged_keep`` of this cache's tokens."""
        paged_keep(self.k_pages, self.v_pages, self.page_table, start, kept, counts, scales=self.scales)

    def attend(self, q: torch.Tensor, pos: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """``paged_attention`` of queries that are rotated already."""
        pers = (self.k_pers, self.v_pers) if self.n_persistent else (None, None)
        return paged_attention(q, self.k_pages, self.v_pages, self.page_table, pos, self.window, *pers, self.scale, out,
                               scales=self.scales, pers_scales=self.pers_scales if self.n_persistent else None)

    def attend_tree(self, q: torch.Tensor, start: torch.Tensor, tree: DraftTree, counts: Optional[torch.Tensor] = None,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """``paged_tree_attention`` of queries that are rotated already."""
        pers = (self.k_pers, self.v_pers) if self.n_persistent else (None, None)
        return paged_tree_attention(q, self.k_pages, self.v_pages, self.page_table, start, tree.seen, counts, tree.positions, self.window,
                                    *pers, self.scale, out, scales=self.scales, pers_scales=self.pers_scales if self.n_persistent else None)

    def decode_tree(self, q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor, start: torch.Tensor, tree: DraftTree,
                    counts: Optional[torch.Tensor] = None) -> torch.Tensor:
        """One step of drafted tokens: ``q [B, heads, nodes, dh]``, ``k_new, v_new [B, kv_heads, nodes, dh]`` become tokens ``start[b] ..``
        (-1: no sequence in this row).  Appends, rotates by the tree's positions if the cache does, and attends."""
        if self.inv_freq is None:
            self.append(k_new, v_new, start, counts)
        else:
            turned = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
            q = self.append(k_new, v_new, start, counts, q=q, q_out=turned, positions=tree.positions)
        return self.attend_tree(q, start, tree, counts)

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
