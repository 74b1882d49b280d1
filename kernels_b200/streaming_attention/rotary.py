"""Rotary position embedding with positions on several axes.

The reference leaves rotary embedding to its callers; :func:`qkv_rope_projection` applies one table of positions, the same
for every sequence.  Tokens of a video or an image stand on several axes (time, height, width), and the
newest tokens of a batch of streams stand at positions of their own.  Here every token brings its position on each axis,
and every axis turns its own band of the frequencies.

One kernel (``kb_rotary``), differentiable in ``q`` and ``k``: the gradient is the same kernel turning the other way.  What traces,
compiles or intercepts operators meets it as ``kernels_b200::rotary_embedding``.  A
backward pass can be captured into a CUDA graph as any of torch's can, while no eager graph of the same leaves is alive.
There is no CPU path.
"""

from __future__ import annotations

from typing import Optional, Sequence, Tuple

import torch

from .. import _lib


_pack = _lib.packer(_lib.RotaryParams).pack


def _rotate(q, k, positions, inv_freq, ends, inverse):
    if q.is_neg() or inv_freq.is_neg() or (k is not None and k.is_neg()):  # the sign is a mark on the tensor, which memory does not show
        q, k, inv_freq = (x if x is None else x.resolve_neg() for x in (q, k, inv_freq))
    shape = q.shape
    B, H, T, D = shape
    q_out, k_out = torch.empty_like(q, memory_format=torch.contiguous_format), None
    keys, keys_to, H_kv = (0, 0, 0, 0, 0), 0, 0
    if k is not None:
        k_shape = k.shape
        k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
        if 0 not in k_shape:
            keys, keys_to, H_kv = (k.data_ptr(), *k.stride()), k_out.data_ptr(), k_shape[1]
    strides = positions.stride()
    if len(strides) == 2:
        strides = strides[0], 0, strides[1]
    block = _pack(q.data_ptr(), *q.stride(), *keys, q_out.data_ptr(), keys_to, positions.data_ptr(), *strides, inv_freq.data_ptr(),
                  B, H, H_kv, T, D, ends[-1], len(ends), *ends, *(0,) * (8 - len(ends)),
                  positions.dtype == torch.int64, _lib.dtype_code(q.dtype), inverse)
    _lib.check(_lib.launch_packed(_lib.load().kb_rotary, block, q.device), "kb_rotary")
    return q_out, k_out


@torch.library.custom_op("kernels_b200::rotary_embedding", mutates_args=(), device_types=("cuda",))
def _rotary_op(
    q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, inv_freq: torch.Tensor, ends: Sequence[int], inverse: bool
) -> Tuple[torch.Tensor, torch.Tensor]:
    q_out, k_out = _rotate(q, k, positions, inv_freq, ends, inverse)
    return q_out, q.new_empty(0) if k_out is None else k_out


@torch.library.register_fake("kernels_b200::rotary_embedding")
def _rotary_op_abstract(q, k, positions, inv_freq, ends, inverse):
    q_out, k_out = (None if x is None else torch.empty_like(x, memory_format=torch.contiguous_format) for x in (q, k))
    return q_out, q.new_empty(0) if k_out is None else k_out


def _op(q, k, *rest):
    """The operator, where something looks into the call: the others go past the dispatcher, which takes 30 microseconds."""
    q_out, k_out = torch.ops.kernels_b200.rotary_embedding(q, k, *rest)
    return q_out, None if k is None else k_out


def _op_setup(ctx, inputs, output):
    _, _, positions, inv_freq, ctx.ends, ctx.inverse = inputs
    ctx.save_for_backward(positions, inv_freq)


def _op_backward(ctx, dq, dk):
    return _gradients(ctx, dq, dk, _op)


def _gradients(ctx, dq, dk, go):
    positions, inv_freq = ctx.saved_tensors
    turn = lambda q, k: go(q, k, positions, inv_freq, ctx.ends, not ctx.inverse)  # noqa: E731
    need_q, need_k = ctx.needs_input_grad[:2]
    if need_q:
        dq, dk = turn(dq, dk if need_k else None)
    else:
        dq, dk = None, turn(dk, None)[0]
    return dq, dk, None, None, None, None


torch.library.register_autograd("kernels_b200::rotary_embedding", _op_backward, setup_context=_op_setup)


def _rotate_or_op(q, k, *rest):
    return (_op if _lib.looked_into(q, k) else _rotate)(q, k, *rest)


def _keep(ctx, inputs):
    _, _, positions, inv_freq, ctx.ends, ctx.inverse = inputs
    ctx.save_for_backward(positions, inv_freq)
    ctx.save_for_forward(positions, inv_freq)


def _turn(*inputs):
    """:func:`_rotate` with gradients."""
    special = _lib.transforms_active() or _lib.looked_into(*inputs[:2])
    return (_RotaryEmbeddingTransformed if special else _RotaryEmbedding).apply(*inputs)


_turn_uncompiled = torch.compiler.disable(_turn)


class _RotaryEmbedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, *inputs):
        _keep(ctx, inputs)
        return _rotate(*inputs)

    @staticmethod
    def backward(ctx, dq, dk):
        # (turned by the same function where gradients are to have gradients)
        return _gradients(ctx, dq, dk, _turn if torch.is_grad_enabled() else _rotate_or_op)

    @staticmethod
    def jvp(ctx, tq, tk, *_):
        positions, inv_freq = ctx.saved_tensors
        turn = lambda x: None if x is None else _turn(x, None, positions, inv_freq, ctx.ends, ctx.inverse)[0]  # noqa: E731
        return turn(tq), turn(tk)


class _RotaryEmbeddingTransformed(_RotaryEmbedding):
    """The form that functorch's transforms ask for (a call of it takes 20 microseconds more), and that calls the operator where something looks into it."""

    @staticmethod
    def forward(q, k, positions, inv_freq, ends, inverse):
        return _rotate_or_op(q, k, positions, inv_freq, ends, inverse)

    @staticmethod
    def setup_context(ctx, inputs, output):
        _keep(ctx, inputs)


def rotary_embedding(
    q: torch.Tensor,
    k: Optional[torch.Tensor],
    positions: torch.Tensor,
    inv_freq: torch.Tensor,
    sections: Optional[Sequence[int]] = None,
):
    """``(q', k')``: pair ``d`` of every head (elements ``d`` and ``d + R``, ``d < R``) turned by ``positions[axis(d)] *
    inv_freq[d]``; contiguous, in the inputs' type.  Differentiable in ``q`` and ``k``.

    ``q``: ``[B, H, T, D]``, ``k``: ``[B, H_kv, T, D]`` or None (then ``k'`` is None), fp32, fp16 or bf16, any strides.
    ``positions``: int32 or int64, ``[A, B, T]``, or ``[A, T]`` for the same positions in every sequence; any whole numbers, far
    ones too: the angle is formed modulo a turn before it is rounded.  ``inv_freq``: float64 ``[R]``, radians per step, ``R <= D / 2``;
    elements from ``2 R`` on are copied.  ``sections``: how many frequencies each of the ``A`` axes (at most 8) takes, in order,
    ``R`` in all; None for one axis.
    """
    if not q.is_cuda:
        raise RuntimeError("rotary_embedding: the tensors must live on a CUDA device (there is no CPU path)")
    shape, pos_shape, index, dtype = q.shape, positions.shape, q.get_device(), q.dtype
    assert len(shape) == 4 and len(pos_shape) in (2, 3), "q is [B, H, T, D], positions are [A, T] or [A, B, T]"
    B, _, T, D = shape
    if k is not None:
        k_shape = k.shape
        assert len(k_shape) == 4 and k_shape[0] == B and k_shape[2] == T and k_shape[3] == D and k.dtype == dtype and k.get_device() == index
    assert positions.dtype in (torch.int32, torch.int64) and positions.get_device() == index
    assert pos_shape[-1] == T and (len(pos_shape) == 2 or pos_shape[1] == B), "positions are [A, T] or [A, B, T]"
    assert inv_freq.ndim == 1 and inv_freq.dtype == torch.float64 and inv_freq.get_device() == index
    R = inv_freq.shape[0]
    assert not inv_freq.requires_grad, "the frequencies have no gradient"
    assert 1 <= R <= D // 2, "as many frequencies as there are pairs, at most"
    sections = (R,) if sections is None else sections
    ends, end = [], 0
    for n in sections:
        end += int(n)
        ends.append(end)
    assert 1 <= len(ends) <= 8 and len(ends) == pos_shape[0], "one section of frequencies per axis, at most 8"
    assert end == R and min(sections) >= 0, "the sections share out inv_freq"
    inv_freq = inv_freq.contiguous()
    looked_into = _lib.looked_into(q, k)
    if _lib.forward_ad_active() or (looked_into and _lib.transforms_active()):
        # (the function's gradients: the operator has none of these; a compiled caller steps out for them)
        return (_turn_uncompiled if torch.compiler.is_compiling() else _turn)(q, k, positions, inv_freq, ends, False)
    if looked_into:
        return _op(q, k, positions, inv_freq, ends, False)
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        return (_RotaryEmbeddingTransformed if _lib.transforms_active() else _RotaryEmbedding).apply(q, k, positions, inv_freq, ends, False)
    return _rotate(q, k, positions, inv_freq, ends, False)
