"""Attention over sequences packed one after another, its gradient, and its single-token form.

Beside the chunk attention (``attention``, ``attention_segments``: one window of keys for a chunk of
queries, equal head counts): whole prompts or clips of different lengths in one call without padding,
causal or full, with grouped heads (query head h reads key/value head ``h // (heads // kv_heads)``), a
backward pass for training, and one query token per sequence over a cache for serving.

bf16 in and out, fp32 scores, softmax and sums; head dim 128. Results do not depend on the order in
which workgroups run (no atomics).
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Sequence

import torch

from . import _lib

__all__ = ["PackedPlan", "packed_plan", "attention_packed", "attention_packed_backward",
           "attention_decode"]

HEAD_DIM = 128


@dataclass(frozen=True)
class PackedPlan:
    """The lengths of a packed batch and the kernels' work items for them, on a device. Made once for a
    batch; every layer's call uses it. A graph that captured calls with it needs it alive."""
    q_lens: tuple
    k_lens: tuple
    causal: bool
    q_tokens: int
    k_tokens: int
    q_items: torch.Tensor
    k_items: torch.Tensor
    info: tuple  # q_tokens, k_tokens, and the items' tile counts


def _lens(name, lens) -> tuple:
    if torch.is_tensor(lens):
        if lens.device.type != "cpu":
            raise ValueError(f"{name} must be host values: the work is planned on the host")
        lens = lens.tolist()
    lens = tuple(int(x) for x in lens)
    if any(x < 0 for x in lens):
        raise ValueError(f"{name} has a negative length")
    if sum(lens) > (1 << 31) - 256:
        raise ValueError(f"{name} add up to {sum(lens)} tokens: at most 2^31 - 256")
    return lens


def packed_plan(q_lens: Sequence[int], k_lens: Sequence[int] | None = None, *, causal: bool = True,
                device=None) -> PackedPlan:
    """Plan for sequences of ``q_lens`` query and ``k_lens`` (default: the same) key tokens, packed in
    this order. ``causal``: query i sees keys ``j <= i + k_len - q_len`` (the last query sees all of them,
    as when a prompt continues over cached keys; leading queries of a sequence with fewer keys see
    none), otherwise every key of its sequence. Lengths may be 0."""
    ops = _lib.ops()
    ql = _lens("q_lens", q_lens)
    kl = ql if k_lens is None else _lens("k_lens", k_lens)
    if len(ql) != len(kl):
        raise ValueError(f"{len(ql)} query and {len(kl)} key lengths")
    qi, ki, tiles = ops.packed_plan(torch.tensor(ql, dtype=torch.int32), torch.tensor(kl, dtype=torch.int32),
                             bool(causal))
    device = torch.device("cuda") if device is None else torch.device(device)
    return PackedPlan(ql, kl, bool(causal), sum(ql), sum(kl), qi.to(device), ki.to(device),
                      (sum(ql), sum(kl), *tiles))


# The ops check what they are given (and raise RuntimeError); a call they refuse is looked over once more
# here, for a ValueError that names the argument. A call that passes pays for one set of checks.
def _check(q, k, v, plan):
    for name, t, n in (("q", q, plan.q_tokens), ("k", k, plan.k_tokens), ("v", v, plan.k_tokens)):
        if t.dim() != 3 or t.dtype != torch.bfloat16 or t.shape[2] != HEAD_DIM:
            raise ValueError(f"{name} must be bf16 [tokens, heads, {HEAD_DIM}], got "
                             f"{tuple(t.shape)} {t.dtype}")
        if t.shape[0] != n:
            raise ValueError(f"{name} has {t.shape[0]} tokens, the plan {n}: pass the packed rows only")
    if k.shape != v.shape or k.shape[1] < 1 or q.shape[1] % k.shape[1]:
        raise ValueError(f"k {tuple(k.shape)}, v {tuple(v.shape)}: one shape, with a head count that "
                         f"divides q's {q.shape[1]}")
    if plan.q_items.device != q.device:
        raise ValueError(f"the plan is on {plan.q_items.device}, q on {q.device}")


def _scale(softmax_scale) -> float:
    if softmax_scale is None:
        return 0.0
    s = float(softmax_scale)
    if not s > 0.0 or math.isinf(s):
        raise ValueError(f"softmax_scale {softmax_scale}: positive and finite")
    return s


def attention_packed(q, k, v, plan: PackedPlan, *, softmax_scale: float | None = None,
                     return_lse: bool = False):
    """softmax(scale Q K^T) V of every sequence of ``plan``: q ``[q_tokens, heads, 128]``, k, v
    ``[k_tokens, kv_heads, 128]`` bf16 (strided views are fine, 16-byte rows) -> out like q; scale
    default 1/sqrt(128), at most 1e6. ``return_lse``: also lse fp32 ``[heads, q_tokens]`` (natural log; no gradient
    flows through it). A query that sees no key gives 0, lse -inf and no gradient. Nothing of one
    sequence reaches another, whatever its values; inside a sequence a NaN or infinity may also reach
    rows that do not see it. Differentiable in q, k, v (first derivatives, reverse mode). A training step captured into
    a graph must not share leaves with a live eager graph of another stream: that backward raises."""
    scale = _scale(softmax_scale)
    try:
        out, lse = _lib.ops().attention_packed(q, k, v, plan.q_items, plan.k_items, plan.info, scale,
                                               return_lse)
    except (RuntimeError, NotImplementedError):
        _check(q, k, v, plan)
        raise
    return (out, lse) if return_lse else out


def attention_packed_backward(dout, q, k, v, out, lse, plan: PackedPlan, *,
                              softmax_scale: float | None = None):
    """``(dq, dk, dv)`` of :func:`attention_packed` from its inputs, ``out`` and ``lse``, without
    autograd."""
    scale = _scale(softmax_scale)
    try:
        return _lib.ops().attention_packed_bwd(dout, q, k, v, out, lse, plan.q_items, plan.k_items,
                                               plan.info, scale)
    except (RuntimeError, NotImplementedError):
        _check(q, k, v, plan)
        if (dout.shape != q.shape or out.shape != q.shape
                or tuple(lse.shape) != (q.shape[1], q.shape[0])):
            raise ValueError("dout and out must have q's shape, lse [heads, tokens]") from None
        raise


def attention_decode(q, k_cache, v_cache, lens, *, softmax_scale: float | None = None,
                     num_splits: int = 0, out=None):
    """One query token per sequence: q ``[batch, heads, 128]`` over ``k_cache``, ``v_cache``
    ``[batch, capacity, kv_heads, 128]`` (strided views are fine), keys ``0 .. lens[b] - 1`` of
    sequence b -> ``[batch, heads, 128]`` (into ``out`` when given). ``lens`` int32 ``[batch]`` on q's device
    is read there (no host sync; limited to ``[0, capacity]``); rows behind a length may hold
    anything. A sequence of no keys gives 0. Not differentiable; with ``out`` it raises while gradients are
    recorded and one of the tensors requires one. ``num_splits`` 1: one workgroup per sequence and kv head; n: the whole batch's
    keys cut into ``n * batch`` equal pieces that run side by side; 0: by batch, heads and capacity."""
    s = _scale(softmax_scale)
    try:
        ops = _lib.ops()
        if out is None:
            return ops.attention_decode(q, k_cache, v_cache, lens, s, num_splits)
        ops.attention_decode_out(q, k_cache, v_cache, lens, s, num_splits, out)
        return out
    except (RuntimeError, NotImplementedError):
        _check_decode(q, k_cache, v_cache, lens, num_splits, out)
        raise


def _check_decode(q, k_cache, v_cache, lens, num_splits, out):
    if q.dim() != 3 or q.dtype != torch.bfloat16 or q.shape[2] != HEAD_DIM:
        raise ValueError(f"q must be bf16 [batch, heads, {HEAD_DIM}], got {tuple(q.shape)} {q.dtype}")
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        if (t.dim() != 4 or t.dtype != torch.bfloat16 or t.shape[0] != q.shape[0]
                or t.shape[3] != HEAD_DIM or t.shape != k_cache.shape):
            raise ValueError(f"{name} must be bf16 [{q.shape[0]}, capacity, kv_heads, {HEAD_DIM}], one "
                             f"shape for both, got {tuple(t.shape)} {t.dtype}")
    if k_cache.shape[2] < 1 or q.shape[1] % k_cache.shape[2]:
        raise ValueError(f"{k_cache.shape[2]} kv heads do not divide {q.shape[1]} heads")
    if lens.dtype != torch.int32 or tuple(lens.shape) != (q.shape[0],):
        raise ValueError(f"lens must be int32 [{q.shape[0]}], got {tuple(lens.shape)} {lens.dtype}")
    if not 0 <= num_splits <= 128:
        raise ValueError(f"num_splits {num_splits} not in [0, 128]")
    if out is not None and (out.shape != q.shape or out.dtype != torch.bfloat16 or out.stride(2) != 1):
        raise ValueError("out must be bf16 of q's shape with a contiguous head dim")
