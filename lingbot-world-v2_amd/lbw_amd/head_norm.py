"""Per-head RMSNorm of q and k with the position rotation in the same pass, and its gradient.

Beside ``qk_norm_rope`` (the Wan blocks' norm over the whole row, on one dense grid): every head is
normalised by itself, q and k may have different head counts (grouped heads), and each token brings its
own position on one to four axes, as sequences packed one after another need. With
y = x rsqrt(mean_d x^2 + eps) w per head, the first 2 * pairs values of y turn by pairs -- (2i, 2i + 1)
interleaved, or (i, i + pairs) in split halves -- pair i by ``angles[pos[token, axis of i], i]``; the
result is scaled and rounded to bf16 once, from fp32.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Sequence

import torch

from . import _lib

__all__ = ["AxisRope", "axis_rope", "qk_head_norm_rope", "qk_head_norm_rope_"]

MAX_AXES = 4


@dataclass(frozen=True)
class AxisRope:
    """A rotation table on a device: ``table`` fp32 ``[positions, pairs, 2]`` (cos, sin), the pairs of
    each axis, and how the values pair."""
    table: torch.Tensor
    axes: tuple
    interleaved: bool


def axis_rope(angles: torch.Tensor, axes: Sequence[int] | None = None, *, interleaved: bool = True,
              device=None) -> AxisRope:
    """Table of ``angles`` ``[positions, pairs]`` (radians; ``wan_rope_freqs`` gives such a table). The
    first ``axes[0]`` pairs turn with a token's first position, the next ``axes[1]`` with its
    second, ... (``rope.axis_split(pairs)`` for the video models' frame, height and width); None: one
    axis. Cosines and sines are taken in 64 bits. Made once, used by every call."""
    if angles.dim() != 2 or not angles.dtype.is_floating_point:
        raise ValueError(f"angles must be floating [positions, pairs], got {tuple(angles.shape)} "
                         f"{angles.dtype}")
    pairs = angles.shape[1]
    axes = (pairs,) if axes is None else tuple(int(a) for a in axes)
    if not 1 <= len(axes) <= MAX_AXES or min(axes) < 0 or sum(axes) != pairs:
        raise ValueError(f"axes {axes}: 1 to {MAX_AXES} counts that add up to {pairs} pairs")
    if not interleaved and pairs % 8:
        raise ValueError(f"split halves need a multiple of 8 pairs, got {pairs}")
    a = angles.detach().to(device=angles.device if device is None else device, dtype=torch.float64)
    return AxisRope(torch.stack((a.cos(), a.sin()), -1).float().contiguous(), axes,
                    bool(interleaved))


def _rows(name, t, like=None):
    if t.dim() != 3 or t.dtype != torch.bfloat16 or t.stride(2) != 1:
        raise ValueError(f"{name} must be bf16 [tokens, heads, D] with a contiguous head dim, got "
                         f"{tuple(t.shape)} {t.dtype} strides {t.stride()}")
    if like is not None and t.shape != like.shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(like.shape)}")


# The ops check what they are given (and raise RuntimeError); a call they refuse is looked over once more
# here, for a ValueError that names the argument. A call that passes pays for one set of checks.
def _check(q, k, wq, wk, rope, pos):
    _rows("q", q)
    _rows("k", k)
    T, hq, D = q.shape
    if k.shape[0] != T or k.shape[2] != D or k.shape[1] < 1 or hq % k.shape[1]:
        raise ValueError(f"k {tuple(k.shape)} does not fit q {tuple(q.shape)}: the same tokens and "
                         "head dim, and a head count that divides q's")
    if 2 * rope.table.shape[1] > D:
        raise ValueError(f"{rope.table.shape[1]} pairs do not fit a head of {D}")
    if rope.table.device != q.device:
        raise ValueError("the rotation table is on another device")
    if (wq is None) != (wk is None):
        raise ValueError("wq and wk: both or neither")
    if pos.dim() == 1:
        pos = pos[:, None]
    if pos.dtype != torch.int32 or tuple(pos.shape) != (T, len(rope.axes)):
        raise ValueError(f"pos must be int32 [{T}, {len(rope.axes)}], got {tuple(pos.shape)} "
                         f"{pos.dtype}")


def qk_head_norm_rope(q, k, wq, wk, rope: AxisRope, pos, eps: float = 1e-6, *,
                      q_scale: float = 1.0, k_scale: float = 1.0):
    """New ``(q', k')`` of q ``[tokens, heads, D]`` and k ``[tokens, kv_heads, D]`` (bf16; strided views
    with a contiguous head dim are fine, e.g. column blocks of a fused projection; D 32, 64, 128 or
    256). ``wq``, ``wk``: ``[D]`` weights, both bf16 or both fp32, or None. ``pos``: int32
    ``[tokens, axes]`` (``[tokens]`` for one axis) on q's device; a position outside the table turns its
    pairs into NaN. Differentiable in q, k, wq and wk (first derivatives, reverse mode; the same bits every
    run)."""
    try:
        return _lib.ops().head_norm_rope(q, k, wq, wk, rope.table, rope.axes, rope.interleaved, pos,
                                         eps, q_scale, k_scale)
    except (RuntimeError, NotImplementedError):
        _check(q, k, wq, wk, rope, pos)
        raise


def qk_head_norm_rope_(q, k, wq, wk, rope: AxisRope, pos, eps: float = 1e-6, *, q_out, k_out,
                       v=None, v_out=None, rows=None, q_scale: float = 1.0, k_scale: float = 1.0):
    """Write form: into ``q_out`` and ``k_out`` (q itself, k itself, or apart from the inputs), with v
    copied to ``v_out`` when given. With ``rows`` (int32 ``[tokens]`` on q's device) token t is the
    newest one of sequence t: its k and v go to row ``rows[t]`` of the caches ``k_out``, ``v_out``
    ``[tokens, capacity, kv_heads, D]`` (strided views are fine), and are not written where that row
    is outside the cache. Outputs may interleave with other tensors of the call, not share an element with
    one. Not differentiable: raises while gradients are recorded and one of the tensors, weights included,
    requires one (``torch.no_grad`` takes it). Returns ``(q_out, k_out)``."""
    try:
        _lib.ops().head_norm_rope_(q, k, wq, wk, rope.table, rope.axes, rope.interleaved, pos, eps,
                                   q_scale, k_scale, q_out, k_out, v, v_out, rows)
    except (RuntimeError, NotImplementedError):
        _check(q, k, wq, wk, rope, pos)
        _check_out(q, k, q_out, k_out, v, v_out, rows)
        raise
    return q_out, k_out


def _check_out(q, k, q_out, k_out, v, v_out, rows):
    _rows("q_out", q_out, q)
    if (v is None) != (v_out is None):
        raise ValueError("v and v_out: both or neither")
    if v is not None:
        _rows("v", v, k)
    for name, t in (("k_out", k_out), ("v_out", v_out)):
        if t is None:
            continue
        if rows is None:
            _rows(name, t, k)
        elif (t.dim() != 4 or t.dtype != torch.bfloat16 or t.stride(3) != 1
              or (t.shape[0],) + tuple(t.shape[2:]) != tuple(k.shape)):
            raise ValueError(f"{name} must be a bf16 cache [{k.shape[0]}, capacity, {k.shape[1]}, "
                             f"{k.shape[2]}] with a contiguous head dim, got {tuple(t.shape)} "
                             f"{t.dtype} strides {t.stride()}")
    if rows is not None and (rows.dtype != torch.int32 or tuple(rows.shape) != (q.shape[0],)):
        raise ValueError(f"rows must be int32 [{q.shape[0]}], got {tuple(rows.shape)} {rows.dtype}")
