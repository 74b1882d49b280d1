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
workspace with torch on the current stream.  Forward only (inference).  There is no CPU path.
"""

from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from .. import _lib
from .kernel import _clamp_i32


def _pages(what, k_pages, v_pages, page_table, lens, k_scale, v_scale):
    """The checked cache as the C ABI's structure, and its device's index.  (A few microseconds of calls that take about twelve: every
    property of a tensor is asked for once, devices by their index.)"""
    if not (k_pages.is_cuda and v_pages.is_cuda):
        raise RuntimeError(f"{what}: the tensors must live on a CUDA device (there is no CPU path)")
    index, shape, dtype = k_pages.get_device(), k_pages.shape, k_pages.dtype
    assert len(shape) == 4 and v_pages.shape == shape and v_pages.dtype == dtype, "k_pages and v_pages are [P, H_kv, page, D]"
    assert v_pages.get_device() == page_table.get_device() == lens.get_device() == index
    P, H_kv, page, D = shape
    ks, vs = k_pages.stride(), v_pages.stride()
    assert page >= 1 and (ks[3] == vs[3] == 1 or 0 in shape), "rows of the pages are dense"
    table_shape, lens_shape = page_table.shape, lens.shape
    assert len(table_shape) == 2 and len(lens_shape) == 1 and page_table.dtype == lens.dtype == torch.int32
    B, M = table_shape
    assert lens_shape[0] == B, "one table row and one length per sequence"
    f8 = dtype == torch.float8_e4m3fn
    assert (k_scale is not None) == (v_scale is not None) == f8, "8-bit pages, and only those, come with scales"
    c = _lib.PagedCache()
    c.k, c.v = k_pages.data_ptr(), v_pages.data_ptr()
    c.k_stride[:], c.v_stride[:] = ks[:3], vs[:3]
    if f8:
        assert k_scale.shape == v_scale.shape == shape[:3] and k_scale.dtype == v_scale.dtype == torch.float32
        assert k_scale.get_device() == v_scale.get_device() == index
        c.k_scale, c.v_scale = k_scale.data_ptr(), v_scale.data_ptr()
        c.k_scale_stride[:], c.v_scale_stride[:] = k_scale.stride(), v_scale.stride()
    c.page_table, c.lens, c.lens_stride = page_table.data_ptr(), lens.data_ptr(), lens.stride(0)
    c.table_stride[:] = page_table.stride()
    c.B, c.H_kv, c.D, c.P, c.M, c.page = B, H_kv, D, P, M, page
    c.dtype = _lib.KB_E4M3 if f8 else _lib.dtype_code(dtype)
    return c, index


def _per_row(name, x, dtype, c, index):
    """Pointer and strides of ``weights`` or ``row_positions``."""
    shape, strides = x.shape, x.stride()
    assert x.dtype == dtype and x.get_device() == index and len(shape) == 3 and shape[0] == c.B and shape[1] == c.H_kv, f"{name} is [B, H_kv, M * page]"
    assert shape[2] >= c.M * c.page and (strides[2] == 1 or shape[2] <= 1), f"{name} has an entry for every row, side by side"
    assert (strides[0] or shape[0] <= 1) and (strides[1] or shape[1] <= 1), f"{name} is written: every sequence and head has entries of its own"
    return x.data_ptr(), strides[:2]


def _workspace(p, n, like):
    """``n`` bytes on the device of ``like`` (int32); the caller holds them until the launch has been made."""
    w = like.new_empty((n + 3) // 4)
    p.workspace, p.workspace_bytes = w.data_ptr(), n
    return w


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
    0, those of ``row_positions`` the tokens' ``positions`` (int32 ``[B, T]``, None for the rows themselves).  Rows outside the table
    are dropped; two tokens of one call must not share a row of a page.
    """
    c, index = _pages("paged_cache_write", k_pages, v_pages, page_table, lens, k_scale, v_scale)
    shape, dtype = k.shape, k.dtype
    assert len(shape) == 4 and v.shape == shape and v.dtype == dtype and k.get_device() == v.get_device() == index
    B, H_kv, T, D = shape
    assert B == c.B and H_kv == c.H_kv and D == c.D, "k and v are [B, H_kv, T, D]"
    assert k_scale is not None or dtype == k_pages.dtype, "k and v have the pages' type"
    p = _lib.PagedWriteParams()
    p.cache = c
    p.k, p.v = _lib.tensor4(k), _lib.tensor4(v)
    p.T, p.dtype = T, _lib.dtype_code(dtype)
    if new_lens is not None:
        assert new_lens.shape == lens.shape and new_lens.dtype == torch.int32 and new_lens.get_device() == index
        p.new_lens, p.new_lens_stride = new_lens.data_ptr(), new_lens.stride(0)
    if positions is not None:
        assert positions.shape == (B, T) and positions.dtype == torch.int32 and positions.get_device() == index
        p.positions = positions.data_ptr()
        p.positions_stride[:] = positions.stride()
    if weights is not None:
        p.weights, p.weights_stride[:] = _per_row("weights", weights, torch.float32, c, index)
    if row_positions is not None:
        p.row_positions, p.row_positions_stride[:] = _per_row("row_positions", row_positions, torch.int32, c, index)
    _lib.check(_lib.launch(_lib.load().kb_paged_write, p, k_pages.device), "kb_paged_write")


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
    operator's mask applies (``kernel.py:1540-1542``): the token sees its own chunk and ``back_contexts`` chunks before it, counted in rows.
    Returns ``o`` ``[B, H, D]`` and, on request, the base-2 log-sum-exp ``[B, H]``; both are 0 for a sequence that sees
    no row.  With ``weights``, the softmax weight of every row that is seen, summed over the query heads of its key/value
    head, is added to ``weights`` in place.

    Sums are held in fp32.  16-bit and e4m3 caches: weights are rounded to 16 bits before they are multiplied with ``v``.  fp32 caches of head dim 64
    and 128 are multiplied on the tensor cores in three parts, as exactly as in fp32; an infinity in a row counts as a NaN there.
    """
    c, index = _pages("paged_attention", k_pages, v_pages, page_table, lens, k_scale, v_scale)
    shape, dtype = q.shape, q.dtype
    assert len(shape) == 3 and q.get_device() == index, "q is [B, H, D]"
    B, H, D = shape
    assert B == c.B and D == c.D, "q is [B, H, D]"
    assert c.H_kv >= 1 and H % c.H_kv == 0, "query heads share the key/value heads evenly"
    assert k_scale is not None or dtype == k_pages.dtype, "q has the pages' type"
    assert context_size is None or context_size >= 1
    assert back_contexts >= 0
    strides = q.stride()
    if strides[2] != 1 or strides[0] % 2 or strides[1] % 2 or q.data_ptr() % 4:
        q = q.contiguous()  # (the tensor-core kernel takes pairs of elements)
        strides = q.stride()
    p = _lib.PagedAttentionParams()
    p.cache = c
    o = torch.empty_like(q) if q.is_contiguous() else q.new_empty(shape)
    lse = lens.new_empty((B, H), dtype=torch.float32) if return_lse or weights is not None else None
    p.q, p.o = q.data_ptr(), o.data_ptr()
    p.q_stride[:] = strides
    if lse is not None:
        p.lse = lse.data_ptr()
    if weights is not None:
        p.weights, p.weights_stride[:] = _per_row("weights", weights, torch.float32, c, index)
    p.H, p.dtype = H, _lib.dtype_code(dtype)
    if context_size is not None:
        p.context_size, p.back_contexts = _clamp_i32(context_size), _clamp_i32(back_contexts)
    p.sm_scale = 1.0 / math.sqrt(D) if sm_scale is None else float(sm_scale)
    lib = _lib.load()
    workspace = _workspace(p, lib.kb_paged_attention_workspace_bytes(p), lens)
    _lib.check(_lib.launch(lib.kb_paged_attention, p, k_pages.device), "kb_paged_attention")
    del workspace
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

    The rows whose position is among the newest ``recent`` stay (``row_positions`` above the head's largest minus ``recent``), then those
    that have received most attention; of equals the lower row.  Every head keeps rows of its own.  Kept rows below the budget do not move; the kept
    rows behind it fill, in order, the places that came free, so that afterwards rows ``0 .. budget - 1`` are the sequence and its later pages are
    free.  Rows are then no longer in the order of their tokens, which attention without a window does not depend on
    (rotary embedding has been applied before the write).

    ``out``: a ``(lens, weights, row_positions)`` to be written instead, not overlapping the given ones (entries of
    the rows that remain; the pages change all the same).  Sequences that share pages need copies of their own first.
    """
    c, index = _pages("paged_cache_evict", k_pages, v_pages, page_table, lens, k_scale, v_scale)
    assert budget >= 1 and recent >= 0, "at least one row stays"
    p = _lib.PagedEvictParams()
    p.cache = c
    p.budget, p.recent = _clamp_i32(budget), _clamp_i32(recent)
    if out is None:
        out = (lens, weights, row_positions)
    else:
        assert len(out) == 3 and out[0].shape == lens.shape and out[0].dtype == torch.int32 and out[0].get_device() == index
    p.lens_out, p.lens_out_stride = out[0].data_ptr(), out[0].stride(0)
    p.weights, p.weights_stride[:] = _per_row("weights", weights, torch.float32, c, index)
    p.row_positions, p.row_positions_stride[:] = _per_row("row_positions", row_positions, torch.int32, c, index)
    p.weights_out, p.weights_out_stride[:] = _per_row("out[1]", out[1], torch.float32, c, index)
    p.row_positions_out, p.row_positions_out_stride[:] = _per_row("out[2]", out[2], torch.int32, c, index)
    lib = _lib.load()
    workspace = _workspace(p, lib.kb_paged_evict_workspace_bytes(p), lens)
    _lib.check(_lib.launch(lib.kb_paged_evict, p, k_pages.device), "kb_paged_evict")
    del workspace
    return out
