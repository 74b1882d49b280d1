"""Answering from a paged key/value cache: the write of new tokens, attention of the newest token, eviction.

The reference runs whole sequences (``src/streaming_attention/kernel.py:1586-1652``), and :func:`streaming_attention_step`
wants a batch's cache as one tensor.  A server's streams come and go and grow at their own pace, so here the cache is a pool of
pages that every sequence lists in a table of its own:

* ``k_pages``, ``v_pages``: ``[P, H_kv, page, D]``, fp32, fp16, bf16 or ``float8_e4m3fn``; unit stride along ``D``, any other strides
  (a ``[P, page, H_kv, D]`` pool is its ``transpose(1, 2)``);
* ``k_scale``, ``v_scale``: fp32 ``[P, H_kv, page]``, one scale per row and head, for e4m3 pages only;
* ``page_table``: int32 ``[B, M]``; row ``r`` of sequence ``b`` lies in page ``page_table[b, r // page]`` at ``r % page``.  An entry
  outside ``[0, P)`` holds nothing: its rows are masked when read and dropped when written;
* ``lens``: int32 ``[B]``, rows per sequence (what is outside ``[0, M * page]`` is clamped);
* ``weights`` fp32 and ``row_positions`` int32, ``[B, H_kv, M * page]`` (longer is fine): what eviction goes by, the attention weight
  that each cached row has received and its token's position.  They belong to sequences, as the table's rows do.

The calls read lengths and tables on the device, so a decoding step can be captured into a graph and replayed.  They allocate their
workspace with torch on the current stream.  Forward only (inference): outputs have no gradient, and a call under ``jit.trace`` or ``make_fx``,
which it would be missing from, is refused (a compiled function steps out for it).  There is no CPU path.
"""

from __future__ import annotations

import math
import struct
from typing import Optional, Tuple

import torch

from .. import _lib
from .kernel import _clamp_i32


_pack_write = _lib.packer(_lib.PagedWriteParams).pack
_pack_attention = _lib.packer(_lib.PagedAttentionParams).pack
_pack_evict = _lib.packer(_lib.PagedEvictParams).pack
_NO_SCALES = (0,) * 8


def _pages(what, k_pages, v_pages, page_table, lens, k_scale, v_scale, written=False):
    """The checked cache: the numbers of the C ABI's ``kb_paged_cache``, the device's index and the rows that a table names.  (A few microseconds
    of calls that take about ten: every property of a tensor is asked for once, devices by their index.)"""
    if not (k_pages.is_cuda and v_pages.is_cuda):
        raise RuntimeError(f"{what}: the tensors must live on a CUDA device (there is no CPU path)")
    _lib.refuse_recording(what)
    index, shape, dtype = k_pages.get_device(), k_pages.shape, k_pages.dtype
    assert len(shape) == 4 and v_pages.shape == shape and v_pages.dtype == dtype, "k_pages and v_pages are [P, H_kv, page, D]"
    assert v_pages.get_device() == page_table.get_device() == lens.get_device() == index
    P, H_kv, page, D = shape
    ks, vs = k_pages.stride(), v_pages.stride()
    assert page >= 1 and (ks[3] == vs[3] == 1 or 0 in shape), "rows of the pages are dense"
    assert not (k_pages.is_neg() or v_pages.is_neg()), "the pages' memory holds their numbers, not the negated ones"
    table_shape, lens_shape = page_table.shape, lens.shape
    assert len(table_shape) == 2 and len(lens_shape) == 1 and page_table.dtype == lens.dtype == torch.int32
    B, M = table_shape
    assert lens_shape[0] == B, "one table row and one length per sequence"
    f8 = dtype == torch.float8_e4m3fn
    assert (k_scale is not None) == (v_scale is not None) == f8, "8-bit pages, and only those, come with scales"
    scales, code = _NO_SCALES, _lib.KB_E4M3
    if f8:
        assert k_scale.shape == v_scale.shape == shape[:3] and k_scale.dtype == v_scale.dtype == torch.float32
        assert k_scale.get_device() == v_scale.get_device() == index and not (k_scale.is_neg() or v_scale.is_neg())
        scales = k_scale.data_ptr(), v_scale.data_ptr(), *k_scale.stride(), *v_scale.stride()
    else:
        code = _lib.dtype_code(dtype)
    if written and (0 in ks or 0 in vs or (f8 and 0 in scales)):
        for name, s in (("k_pages", ks), ("v_pages", vs), ("k_scale", scales[2:5]), ("v_scale", scales[5:]))[: 4 if f8 else 2]:
            assert (s[0] or P <= 1) and (s[1] or H_kv <= 1) and (s[2] or page <= 1), f"{name} is written: every page, head and row has memory of its own"
    cache = (k_pages.data_ptr(), v_pages.data_ptr(), *ks[:3], *vs[:3], *scales, page_table.data_ptr(), *page_table.stride(), lens.data_ptr(), lens.stride(0),
             B, H_kv, D, P, M, page, code)
    return cache, index, M * page


def _per_row(name, x, dtype, B, H_kv, rows, index):
    """Pointer and strides of ``weights`` or ``row_positions``."""
    shape, strides = x.shape, x.stride()
    assert x.dtype == dtype and x.get_device() == index and not (dtype.is_floating_point and x.is_neg()) and len(shape) == 3 and shape[0] == B and shape[1] == H_kv, f"{name} is [B, H_kv, M * page]"
    assert shape[2] >= rows and (strides[2] == 1 or shape[2] <= 1), f"{name} has an entry for every row, side by side"
    assert (strides[0] or B <= 1) and (strides[1] or H_kv <= 1), f"{name} is written: every sequence and head has entries of its own"
    return x.data_ptr(), strides[0], strides[1]


def _launch(entry, sizes, block, at, like):
    """Launch with a workspace of the bytes that ``sizes`` asks for, on the device of ``like`` (int32); its address and size go to ``at`` of the
    packed ``block``."""
    lib = _lib.load()
    n = getattr(lib, sizes)(block)
    if n:
        workspace = like.new_empty((n + 3) // 4)
        block = block[:at] + _POINTER_AND_SIZE.pack(workspace.data_ptr(), n) + block[at + 16:]
    _lib.check(_lib.launch_packed(getattr(lib, entry), block, like.device), entry)


_POINTER_AND_SIZE = struct.Struct("=QQ")
_NONE3 = (0, 0, 0)


def paged_cache_write(
    k: torch.Tensor,
    v: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    page_table: torch.Tensor,
    lens: torch.Tensor,
    new_lens: Optional[torch.Tensor] = None,
    positions: Optional[torch.Tensor] = None,
    weights: Optional[torch.Tensor] = None,
    row_positions: Optional[torch.Tensor] = None,
    k_scale: Optional[torch.Tensor] = None,
    v_scale: Optional[torch.Tensor] = None,
) -> None:
    """Write new tokens into their rows, in place.

    ``k``, ``v``: ``[B, H_kv, T, D]``, any strides, of the pages' type, or fp32, fp16 or bf16 for e4m3 pages: every row is
    then scaled so that its largest magnitude maps to 448.  ``lens`` counts the new tokens already: token ``t < new_lens[b]``
    (int32 ``[B]``, None for ``T``) goes to row ``lens[b] - new_lens[b] + t``.  The entries of ``weights`` that belong to written rows become
    0, those of ``row_positions`` the tokens' ``positions`` (int32 ``[B, T]``, None for the rows themselves; once rows have been evicted these are no
    longer the tokens' positions, and new tokens need their own to be the newest).  Rows outside the table
    are dropped; two tokens of one call must not share a row of a page.
    """
    cache, index, rows = _pages("paged_cache_write", k_pages, v_pages, page_table, lens, k_scale, v_scale, True)
    shape, dtype = k.shape, k.dtype
    if k.is_neg() or v.is_neg():  # (the sign is a mark on the tensor, which memory does not show)
        k, v = k.resolve_neg(), v.resolve_neg()
    assert len(shape) == 4 and v.shape == shape and v.dtype == dtype and k.get_device() == v.get_device() == index
    B, H_kv, T, D = shape
    pages_shape, lens_shape = k_pages.shape, lens.shape
    assert B == lens_shape[0] and H_kv == pages_shape[1] and D == pages_shape[3], "k and v are [B, H_kv, T, D]"
    assert k_scale is not None or dtype == k_pages.dtype, "k and v have the pages' type"
    new = at = (0, 0, 0)
    if new_lens is not None:
        assert new_lens.shape == lens_shape and new_lens.dtype == torch.int32 and new_lens.get_device() == index
        new = new_lens.data_ptr(), new_lens.stride(0)
    if positions is not None:
        assert positions.shape == (B, T) and positions.dtype == torch.int32 and positions.get_device() == index
        at = positions.data_ptr(), *positions.stride()
    block = _pack_write(
        *cache, k.data_ptr(), *k.stride(), v.data_ptr(), *v.stride(), new[0], new[1], *at,
        *(_NONE3 if weights is None else _per_row("weights", weights, torch.float32, B, H_kv, rows, index)),
        *(_NONE3 if row_positions is None else _per_row("row_positions", row_positions, torch.int32, B, H_kv, rows, index)),
        T, _lib.dtype_code(dtype))
    _lib.check(_lib.launch_packed(_lib.load().kb_paged_write, block, k_pages.device), "kb_paged_write")


def paged_attention(
    q: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    page_table: torch.Tensor,
    lens: torch.Tensor,
    context_size: Optional[int] = None,
    back_contexts: int = 0,
    sm_scale: Optional[float] = None,
    return_lse: bool = False,
    k_scale: Optional[torch.Tensor] = None,
    v_scale: Optional[torch.Tensor] = None,
    weights: Optional[torch.Tensor] = None,
):
    """Attention of the newest token of every sequence, the one in row ``lens[b] - 1``, over the sequence's cached rows.

    ``q``: ``[B, H, D]``, ``H`` a multiple of ``H_kv``, of the pages' type (fp32, fp16 or bf16 for e4m3 pages).  With ``context_size`` the
    operator's mask applies (``kernel.py:1540-1542``): the token sees its own chunk and ``back_contexts`` chunks before it, counted in rows
    (not in tokens: an eviction leaves rows in another order, and a window after one is a window of rows).
    Returns ``o`` ``[B, H, D]`` and, on request, the base-2 log-sum-exp ``[B, H]``; both are 0 for a sequence that sees
    no row.  With ``weights``, the softmax weight of every row that is seen, summed over the query heads of its key/value
    head, is added to ``weights`` in place; that takes 4 bytes of workspace per query head and row that a token can see (of the window, or of the table).

    Sums are held in fp32.  16-bit and e4m3 caches: weights are rounded to 16 bits before they are multiplied with ``v``.  fp32 caches of head dim 64
    and 128 are multiplied on the tensor cores in three parts, as exactly as in fp32; an infinity in a row counts as a NaN there, and so does a number
    within 2^-12 of fp32's largest.  The row of an infinite value, whose scale in e4m3 pages is infinite, makes its heads NaN, and leaves the
    log-sum-exp and weights alone.  (Value scales from 2^-80 to 2^88 lose nothing; smaller ones alone cost the outputs accuracy, larger ones the other two.)
    """
    cache, index, rows = _pages("paged_attention", k_pages, v_pages, page_table, lens, k_scale, v_scale)
    shape, dtype, pages_shape = q.shape, q.dtype, k_pages.shape
    assert len(shape) == 3 and q.get_device() == index, "q is [B, H, D]"
    B, H, D = shape
    H_kv = pages_shape[1]
    assert B == lens.shape[0] and D == pages_shape[3], "q is [B, H, D]"
    assert H_kv >= 1 and H % H_kv == 0, "query heads share the key/value heads evenly"
    assert k_scale is not None or dtype == k_pages.dtype, "q has the pages' type"
    assert context_size is None or context_size >= 1
    assert back_contexts >= 0
    strides = q.stride()
    if strides[2] != 1 or strides[0] % 2 or strides[1] % 2 or q.data_ptr() % 4 or q.is_neg():
        q = q.resolve_neg().contiguous()  # (the tensor-core kernel takes pairs of elements)
        strides = q.stride()
    o = torch.empty_like(q) if q.is_contiguous() else q.new_empty(shape)
    lse = lens.new_empty((B, H), dtype=torch.float32) if return_lse or weights is not None else None
    block = _pack_attention(
        *cache, q.data_ptr(), *strides, o.data_ptr(), 0 if lse is None else lse.data_ptr(),
        *(_NONE3 if weights is None else _per_row("weights", weights, torch.float32, B, H_kv, rows, index)), 0, 0,
        H, _lib.dtype_code(dtype), 0 if context_size is None else _clamp_i32(context_size), 0 if context_size is None else _clamp_i32(back_contexts),
        1.0 / math.sqrt(D) if sm_scale is None else float(sm_scale))
    _launch("kb_paged_attention", "kb_paged_attention_workspace_bytes", block, _lib.PagedAttentionParams.workspace.offset, lens)
    return (o, lse) if return_lse else o


def paged_cache_evict(
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    page_table: torch.Tensor,
    lens: torch.Tensor,
    weights: torch.Tensor,
    row_positions: torch.Tensor,
    budget: int,
    recent: int = 0,
    k_scale: Optional[torch.Tensor] = None,
    v_scale: Optional[torch.Tensor] = None,
    out: Optional[Tuple[torch.Tensor, torch.Tensor, torch.Tensor]] = None,
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Cut every sequence down to ``budget`` rows per head; returns ``(lens, weights, row_positions)``, updated in place.

    The rows whose position is among the newest ``recent`` stay (``row_positions`` above the head's largest minus ``recent``; where these are more
    than ``budget``, the newest of them), then those that have received most attention; of equals the lower row.  Every head keeps rows of its own.  Kept rows below the budget do not move; the kept
    rows behind it fill, in order, the places that came free, so that afterwards rows ``0 .. budget - 1`` are the sequence and its later pages are
    free.  Rows are then no longer in the order of their tokens, which attention without a window does not depend on
    (rotary embedding has been applied before the write).  Rows without a page are passed over, and nothing moves into one: as many rows stay
    as the first ``budget`` places have pages for.

    ``out``: a ``(lens, weights, row_positions)`` to be written instead, not overlapping the given ones (entries of
    the rows that remain; the pages change all the same).  Sequences that share pages need copies of their own first.
    """
    cache, index, rows = _pages("paged_cache_evict", k_pages, v_pages, page_table, lens, k_scale, v_scale, True)
    assert budget >= 1 and recent >= 0, "at least one row stays"
    B, H_kv = lens.shape[0], k_pages.shape[1]
    w = _per_row("weights", weights, torch.float32, B, H_kv, rows, index)
    p = _per_row("row_positions", row_positions, torch.int32, B, H_kv, rows, index)
    if out is None:
        out = (lens, weights, row_positions)
        w_out, p_out = w, p
    else:
        assert len(out) == 3 and out[0].shape == lens.shape and out[0].dtype == torch.int32 and out[0].get_device() == index
        assert out[0].stride(0) or B <= 1, "out[0] is written: every sequence has a length of its own"
        w_out = _per_row("out[1]", out[1], torch.float32, B, H_kv, rows, index)
        p_out = _per_row("out[2]", out[2], torch.int32, B, H_kv, rows, index)
    block = _pack_evict(*cache, *w, *p, *w_out, *p_out, out[0].data_ptr(), out[0].stride(0), 0, 0, _clamp_i32(budget), _clamp_i32(recent))
    _launch("kb_paged_evict", "kb_paged_evict_workspace_bytes", block, _lib.PagedEvictParams.workspace.offset, lens)
    return out
