"""Rotary positions with several axes (time, height, width) on MI355X.

The reference rotates row ``s`` by table row ``s`` (model.py:41-67); text and
image tokens of one prompt instead carry a position per axis. ``sections``
says how many of a row's ``head_dim / 2`` rotated pairs (rotate-half: elements
``i`` and ``i + head_dim / 2``) each axis has, in order, and the tables are the
ones ``precompute_rope`` makes, looked up at each axis' position. One section
is RoPE at arbitrary positions. ``apply_rope_axes`` rotates q and k in one
launch and is differentiable; ``write_to_paged_cache_rope`` (``paged``) rotates
on the way into a page pool.
"""

from __future__ import annotations

from typing import Optional, Sequence, Tuple

import torch

from . import _lib


def check_sections(sections, head_dim: int) -> Tuple[int, ...]:
    """``sections`` as a tuple (``None``: one axis), or ValueError."""
    if head_dim < 2 or head_dim % 2 != 0:
        raise ValueError(f"head_dim must be even for RoPE, got {head_dim}")
    if sections is None:
        return (head_dim // 2,)
    sections = tuple(int(n) for n in sections)
    if not 1 <= len(sections) <= _lib.MAX_ROPE_AXES:
        raise ValueError(f"sections must name 1 to {_lib.MAX_ROPE_AXES} axes, got {len(sections)}")
    if any(n < 1 for n in sections) or sum(sections) != head_dim // 2:
        raise ValueError(f"sections must be positive and add up to head_dim / 2 = {head_dim // 2}, got {sections}")
    return sections


def check_tables(cos, sin, head_dim: int) -> None:
    if cos.dim() != 2 or cos.shape != sin.shape or cos.shape[1] != head_dim or cos.shape[0] == 0:
        raise ValueError(f"cos/sin must be [rope_len, {head_dim}] of one shape, got {tuple(cos.shape)} and "
                         f"{tuple(sin.shape)}")


def check_axis_positions(positions, axes: int, batch: int, seq_len: int) -> torch.Tensor:
    """Positions as an integer tensor ``[axes, batch or 1, seq_len]``, or ValueError."""
    t = positions if isinstance(positions, torch.Tensor) else torch.as_tensor(positions)
    if t.dtype.is_floating_point or t.dtype.is_complex or t.dtype == torch.bool:
        raise ValueError(f"positions must be integers, got {t.dtype}")
    shape = tuple(t.shape)
    if axes == 1 and t.dim() == 1:
        t = t[None, None]
    elif axes == 1 and t.dim() == 2:
        t = t[None]
    elif t.dim() == 2:
        t = t[:, None]
    if t.dim() != 3 or t.shape[0] != axes or t.shape[1] not in (1, batch) or t.shape[2] != seq_len:
        raise ValueError(f"positions must be [axes={axes}, seq={seq_len}] or [{axes}, batch={batch}, {seq_len}], "
                         f"got {shape}")
    return t


def device_positions(t: torch.Tensor, device) -> Tuple[torch.Tensor, Tuple[int, int, int], int]:
    """``check_axis_positions``'s tensor in device memory as int32 or int64
    (others become int64), its strides (0 over a shared batch) and whether it
    is int64. An int32 or int64 tensor already there is used as is."""
    if t.dtype not in (torch.int32, torch.int64):
        t = t.to(torch.int64)
    t = t.to(device)
    return t, (t.stride(0), t.stride(1) if t.shape[1] > 1 else 0, t.stride(2)), int(t.dtype == torch.int64)


def rows_of(x: torch.Tensor) -> torch.Tensor:
    """x with dense rows (its other strides are the kernel's to walk)."""
    return x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous()


def strides3(x: Optional[torch.Tensor]):
    return (_lib.c_i64 * 3)(*(x.stride()[:3] if x is not None else (0, 0, 0)))


def sections4(sections: Sequence[int]):
    return (_lib.c_i32 * _lib.MAX_ROPE_AXES)(*sections)


def _launch(q, k, positions, cos, sin, sections, inverse: bool):
    q = rows_of(q)
    k = None if k is None else rows_of(k)
    batch, heads, seq, d = q.shape
    q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    k_out = None if k is None else torch.empty(k.shape, dtype=k.dtype, device=k.device)
    if batch * seq == 0:
        return q_out, k_out
    pos, stride, i64 = device_positions(positions, q.device)
    args = _lib.RopeAxesArgs(
        _lib.ptr(q), _lib.ptr(k), _lib.ptr(q_out), _lib.ptr(k_out), strides3(q), strides3(k), _lib.ptr(pos),
        (_lib.c_i64 * 3)(*stride), i64, len(sections), sections4(sections), _lib.ptr(cos), _lib.ptr(sin), cos.shape[0],
        batch, heads, 0 if k is None else k.shape[1], seq, d, int(inverse), _lib.dtype_tag(q))
    with torch.cuda.device(q.device):
        _lib.check(_lib.lib().pf_rope_axes(args, _lib.stream_of(q)), "apply_rope_axes")
    return q_out, k_out


class _RopeAxesFn(torch.autograd.Function):
    """The rotation is linear: its backward is the transposed rotation, which
    is differentiable in turn."""

    @staticmethod
    def forward(ctx, q, k, positions, cos, sin, sections, inverse):
        ctx.save_for_backward(positions, cos, sin)
        ctx.sections, ctx.inverse = sections, inverse
        ctx.set_materialize_grads(False)
        return _launch(q, k, positions, cos, sin, sections, inverse)

    @staticmethod
    def backward(ctx, dq, dk):
        positions, cos, sin = ctx.saved_tensors
        if not ctx.needs_input_grad[0]:
            dq = None
        if not ctx.needs_input_grad[1]:
            dk = None
        if dq is not None:
            dq, dk = _RopeAxesFn.apply(dq, dk, positions, cos, sin, ctx.sections, not ctx.inverse)
        elif dk is not None:
            dk, _ = _RopeAxesFn.apply(dk, None, positions, cos, sin, ctx.sections, not ctx.inverse)
        return dq, dk, None, None, None, None, None


def apply_rope_axes(
    q: torch.Tensor,
    k: Optional[torch.Tensor],
    positions,
    cos: torch.Tensor,
    sin: torch.Tensor,
    sections: Optional[Sequence[int]] = None,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Rotate q and k by positions with several axes, in one launch.

    With ``p = positions[axis of pair i]`` each pair ``(x[i], x[i + head_dim /
    2])`` becomes what ``apply_rope`` makes of it with table row ``p``
    (model.py:60-67), in float32 and rounded once.

    Args:
        q: ``[batch, num_heads, seq, head_dim]``, any even head_dim.
        k: ``[batch, num_kv_heads, seq, head_dim]`` in q's dtype, or ``None``.
            Both are read with their own strides: the transposed view of a
            projection is not copied.
        positions: integers ``[axes, seq]`` or ``[axes, batch, seq]`` (one
            axis: also ``[seq]`` or ``[batch, seq]``); int32 and int64 tensors
            on the device are read as they are. A token with a position outside
            the tables on any axis gives zeros (and zero gradients).
        cos, sin: ``[rope_len, head_dim]`` tables (``precompute_rope``); no
            gradient flows to them.
        sections: the rotated pairs of each axis (1 to 4 axes), positive and
            ``head_dim / 2`` in all; ``None``: one axis.

    Returns:
        ``(q_rot, k_rot)``, dense, in q's dtype; ``k_rot`` is ``None`` without
        k. Differentiable in q and k.
    """
    out = _lib.calls().rope_axes(q, k, positions, cos, sin, sections)
    if out is not None:
        return out
    if q.dim() != 4 or (k is not None and k.dim() != 4):
        raise ValueError("q and k must be rank-4 [batch, heads, seq, head_dim] arrays")
    batch, _, seq, head_dim = q.shape
    if k is not None and (k.shape[0] != batch or k.shape[2] != seq or k.shape[3] != head_dim):
        raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)} must share batch, seq and head_dim")
    if q.shape[1] == 0 or (k is not None and k.shape[1] == 0):
        raise ValueError("q and k must have heads")
    if k is not None and k.dtype != q.dtype:
        raise ValueError(f"q and k must share a dtype, got {q.dtype} and {k.dtype}")
    sections = check_sections(sections, head_dim)
    check_tables(cos, sin, head_dim)
    positions = check_axis_positions(positions, len(sections), batch, seq)
    _lib.require_device(q, *([] if k is None else [k]))
    _lib.dtype_tag(q)
    cos, sin = (t.detach().to(device=q.device, dtype=torch.float32).contiguous() for t in (cos, sin))
    return _RopeAxesFn.apply(q, k, positions.to(q.device), cos, sin, sections, False)


__all__ = ["apply_rope_axes"]
