"""A paged key/value cache: appending to it, attention over it, and choosing which of its pages to look at.

Beside the per-sequence caches (``qk_head_norm_rope_`` with ``rows``, ``attention_decode``): pages of a fixed
number of tokens that belong to any sequence, so sequences of different lengths share one pool, and several that go
on from one history share its pages. The caller keeps the page table -- ``table`` int32 ``[batch, width]`` on the
device, entry j the page of a sequence's tokens ``j * page_size ..`` -- and the lengths; both are read on the device,
so a captured step replays with new ones. Entries behind a sequence's length may hold anything. A page outside the
cache is never followed: nothing is written to it, keys from it make a result NaN, and it is selected first.

bf16 data, fp32 sums and softmax; query head h reads key/value head ``h // (heads // kv_heads)``. Results do not
depend on the order in which workgroups run (no atomics on data).
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _lib
from .head_norm import AxisRope
from .packed import HEAD_DIM, _scale

__all__ = ["PagedKV", "paged_kv", "paged_append_", "attention_paged", "paged_select"]


@dataclass(frozen=True)
class PagedKV:
    """``k``, ``v`` bf16 ``[pages, page_size, kv_heads, D]`` (strided views are fine) and, for
    :func:`paged_select`, ``bounds`` bf16 ``[pages, kv_heads, 2, D]``: the smallest and the largest value of each key
    component of a page."""
    k: torch.Tensor
    v: torch.Tensor
    bounds: torch.Tensor | None = None


def paged_kv(pages: int, page_size: int, kv_heads: int, head_dim: int = HEAD_DIM, *, bounds: bool = False,
             device=None) -> PagedKV:
    """A cache of zeros. ``page_size``: a power of two from 16 to 1024. ``head_dim``: 128 (:func:`paged_append_` also fills
    pages of 32, 64 and 256, for readers of one's own). A page holds each head's tokens together, so a head's part of it
    is one block of memory."""
    if pages < 1 or kv_heads < 1 or head_dim < 1:
        raise ValueError(f"a cache of {pages} pages, {kv_heads} heads of {head_dim}")
    if not 16 <= page_size <= 1024 or page_size & (page_size - 1):
        raise ValueError(f"page_size {page_size}: a power of two from 16 to 1024")
    device = torch.device("cuda") if device is None else torch.device(device)
    k, v = (torch.zeros(pages, kv_heads, page_size, head_dim, dtype=torch.bfloat16, device=device).transpose(1, 2)
            for _ in range(2))
    edge = torch.zeros(pages, kv_heads, 2, head_dim, dtype=torch.bfloat16, device=device) if bounds else None
    return PagedKV(k, v, edge)


# The ops check what they are given (and raise RuntimeError); a call they refuse is looked over once more
# here, for a ValueError that names the argument. A call that passes pays for one set of checks.
def _check_cache(cache, heads, D):
    k, v = cache.k, cache.v
    for name, t in (("cache.k", k), ("cache.v", v)):
        if t.dim() != 4 or t.dtype != torch.bfloat16 or t.shape[2:] != (heads, D) or t.shape != k.shape:
            raise ValueError(f"{name} must be bf16 [pages, page_size, {heads}, {D}], one shape for both, got "
                             f"{tuple(t.shape)} {t.dtype}")
    size = k.shape[1]
    if not 16 <= size <= 1024 or size & (size - 1):
        raise ValueError(f"page_size {size}: a power of two from 16 to 1024")
    _check_bounds(cache, heads, D)


def _check_bounds(cache, heads, D):
    e = cache.bounds
    if e is not None and (e.dtype != torch.bfloat16 or tuple(e.shape) != (cache.k.shape[0], heads, 2, D)
                          or not e.is_contiguous()):
        raise ValueError(f"cache.bounds must be contiguous bf16 {(cache.k.shape[0], heads, 2, D)}, got "
                         f"{tuple(e.shape)} {e.dtype}")


def _check_table(table, lens, batch):
    if lens.dtype != torch.int32 or tuple(lens.shape) != (batch,):
        raise ValueError(f"lens must be int32 [{batch}], got {tuple(lens.shape)} {lens.dtype}")
    if table.dtype != torch.int32 or table.dim() != 2 or table.shape[0] != batch:
        raise ValueError(f"table must be int32 [{batch}, width], got {tuple(table.shape)} {table.dtype}")


def paged_append_(cache: PagedKV, q, k, v, table, lens, rope: AxisRope, pos=None, *, starts=None, q_out=None,
                  wq=None, wk=None, eps: float | None = None, q_scale: float = 1.0, k_scale: float = 1.0):
    """New tokens, q ``[tokens, heads, D]``, k, v ``[tokens, kv_heads, D]`` (bf16; strided views with a contiguous
    head dim are fine, e.g. column blocks of a fused projection; D 32, 64, 128 or 256): q and k turned by ``rope`` at the
    tokens' positions, k and v put into the cache, its bounds (where it has them) kept up.

    ``lens`` int32 ``[batch]``: the rows that each sequence has so far; the call does not change it. ``starts`` None: one
    token per sequence, token b goes to row ``lens[b]``. Otherwise int32 ``[batch + 1]`` on the device, rising: tokens
    ``starts[b] .. starts[b + 1] - 1`` are sequence b's next ones, as far as there are such tokens (a slice of a longer
    batch may have starts below 0 and past its end); tokens outside all of them are left alone, their ``q_out`` rows too. A row outside the table is not written. ``pos`` int32 ``[tokens, axes]`` (``[tokens]`` for one
    axis); None: a token's row in its sequence's table, for a rotation of one axis (behind a prefix that is not the
    position: give it). A position outside the rotation's table turns
    its pairs into NaN. ``eps`` not None: RMSNorm of every q and k head first, as in :func:`qk_head_norm_rope`, with
    weights ``wq``, ``wk`` or none.

    A page that gets its row 0 starts its bounds anew; rows written over later only widen them. No two sequences of a call,
    nor two entries of a sequence's row of the table, may put tokens into one page (copy a shared page that is not full,
    with its bounds, before a branch goes on in it). Returns the turned q, in ``q_out`` when given (q
    itself, or apart from every other tensor of the call). Not differentiable: raises while gradients are recorded and
    one of the tensors, weights included, requires one (``torch.no_grad`` takes it)."""
    if q_out is None:
        q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    try:
        _lib.ops().paged_append_.default(q, k, v, wq, wk, rope.table, rope.axes, rope.interleaved, pos, eps is not None,
                                 0.0 if eps is None else eps, q_scale, k_scale, table, lens, starts, q_out, cache.k,
                                 cache.v, cache.bounds)
    except (RuntimeError, NotImplementedError):
        _check_append(cache, q, k, v, table, lens, rope, pos, starts, q_out, wq, wk, eps)
        raise
    return q_out


def _check_append(cache, q, k, v, table, lens, rope, pos, starts, q_out, wq, wk, eps):
    for name, t in (("q", q), ("k", k), ("v", v), ("q_out", q_out)):
        if t.dim() != 3 or t.dtype != torch.bfloat16 or (t.shape[2] > 1 and t.stride(2) != 1):
            raise ValueError(f"{name} must be bf16 [tokens, heads, D] with a contiguous head dim, got "
                             f"{tuple(t.shape)} {t.dtype} strides {t.stride()}")
    T, hq, D = q.shape
    if k.shape[0] != T or k.shape[2] != D or k.shape[1] < 1 or hq % k.shape[1] or v.shape != k.shape:
        raise ValueError(f"k {tuple(k.shape)}, v {tuple(v.shape)} do not fit q {tuple(q.shape)}: the same tokens and "
                         "head dim, one head count for both that divides q's")
    if q_out.shape != q.shape:
        raise ValueError(f"q_out must have q's shape, got {tuple(q_out.shape)}")
    if eps is None and (wq is not None or wk is not None):
        raise ValueError("wq and wk belong to the norm: eps is wanted with them")
    if (wq is None) != (wk is None):
        raise ValueError("wq and wk: both or neither")
    if 2 * rope.table.shape[1] > D:
        raise ValueError(f"{rope.table.shape[1]} pairs do not fit a head of {D}")
    if pos is None:
        if len(rope.axes) != 1:
            raise ValueError(f"a rotation on {len(rope.axes)} axes needs pos")
    else:
        p = pos[:, None] if pos.dim() == 1 else pos
        if p.dtype != torch.int32 or tuple(p.shape) != (T, len(rope.axes)):
            raise ValueError(f"pos must be int32 [{T}, {len(rope.axes)}], got {tuple(pos.shape)} {pos.dtype}")
    batch = T if starts is None else lens.numel()
    _check_table(table, lens, batch)
    if starts is not None and (starts.dtype != torch.int32 or tuple(starts.shape) != (batch + 1,)):
        raise ValueError(f"starts must be int32 [{batch + 1}], got {tuple(starts.shape)} {starts.dtype}")
    _check_cache(cache, k.shape[1], D)


def attention_paged(q, cache: PagedKV, table, lens, *, selected=None, prefix_table=None, prefix_len=None,
                    softmax_scale: float | None = None, num_splits: int = 0, out=None):
    """One query token per sequence over its pages: q ``[batch, heads, 128]``, keys ``0 .. lens[b] - 1`` of sequence b
    (``lens`` int32 ``[batch]`` on q's device, limited to what the table's row holds) -> ``[batch, heads, 128]`` (into
    ``out`` when given). A sequence of no keys gives 0. Rows behind a length may hold anything.

    ``prefix_table`` int32 ``[pages]``: keys that come before every sequence's own, ``prefix_len`` of them (an int, or
    one int32 on the device, limited to the pages; None: all). They are read once for the whole batch (unless they are
    few); table and lens then describe what each sequence has behind them. Several tokens of one sequence are as many rows of q, table and lens.

    ``selected`` int32 ``[batch, kv_heads, n]`` (from :func:`paged_select`): a key/value head attends to the table entries
    that its list names, up to the first negative one; entries at or past the length name no keys, one that is named twice
    counts twice. It applies to the sequences' own keys, not to a prefix.

    Scores that are all -infinity give NaN.

    The lengths are on the device, so the work is cut by what the table and the prefix can hold: where lengths stay far
    below that, give the columns that they can reach (``table[:, :n]`` is taken as it is).

    Not differentiable; with ``out`` it raises while gradients are recorded and one of the tensors requires one.
    ``num_splits`` as in :func:`attention_decode`; the keys of a list or prefix are cut into so many pieces."""
    s = _scale(softmax_scale)
    keys = -1
    if prefix_len is not None and not torch.is_tensor(prefix_len):
        keys, prefix_len = int(prefix_len), None
        if keys < 0:
            raise ValueError(f"prefix_len {keys} is negative")
    try:
        ops = _lib.ops()
        if out is None:
            return ops.attention_paged.default(q, cache.k, cache.v, table, lens, selected, prefix_table, prefix_len, keys, s,
                                       num_splits)
        ops.attention_paged_out.default(q, cache.k, cache.v, table, lens, selected, prefix_table, prefix_len, keys, s,
                                num_splits, out)
        return out
    except (RuntimeError, NotImplementedError):
        _check_attention(q, cache, table, lens, selected, prefix_table, prefix_len, keys, num_splits, out)
        raise


def _check_query(q, heads):
    if q.dim() != 3 or q.dtype != torch.bfloat16 or q.shape[2] != HEAD_DIM:
        raise ValueError(f"q must be bf16 [batch, heads, {HEAD_DIM}], got {tuple(q.shape)} {q.dtype}")
    if heads < 1 or q.shape[1] % heads:
        raise ValueError(f"{heads} kv heads do not divide {q.shape[1]} heads")


def _check_attention(q, cache, table, lens, selected, prefix_table, prefix_len, keys, num_splits, out):
    heads = cache.k.shape[2] if cache.k.dim() == 4 else 0
    _check_query(q, heads)
    _check_cache(cache, heads, HEAD_DIM)
    _check_table(table, lens, q.shape[0])
    if not 0 <= num_splits <= 128:
        raise ValueError(f"num_splits {num_splits} not in [0, 128]")
    if selected is not None and (selected.dtype != torch.int32 or selected.dim() != 3
                                 or tuple(selected.shape[:2]) != (q.shape[0], heads)):
        raise ValueError(f"selected must be int32 [{q.shape[0]}, {heads}, pages], got {tuple(selected.shape)} "
                         f"{selected.dtype}")
    if prefix_table is None:
        if prefix_len is not None or keys >= 0:
            raise ValueError("prefix_len without prefix_table")
    elif prefix_table.dtype != torch.int32 or prefix_table.dim() != 1:
        raise ValueError(f"prefix_table must be int32 [pages], got {tuple(prefix_table.shape)} {prefix_table.dtype}")
    elif keys > prefix_table.shape[0] * cache.k.shape[1]:
        raise ValueError(f"prefix_len {keys}: {prefix_table.shape[0]} pages of {cache.k.shape[1]} tokens")
    if prefix_len is not None and (prefix_len.dtype != torch.int32 or prefix_len.numel() != 1):
        raise ValueError(f"prefix_len must be an int or one int32, got {tuple(prefix_len.shape)} {prefix_len.dtype}")
    if out is not None and (out.shape != q.shape or out.dtype != torch.bfloat16 or out.stride(2) != 1):
        raise ValueError("out must be bf16 of q's shape with a contiguous head dim")


def paged_select(q, cache: PagedKV, table, lens, count: int, *, first: int = 1, last: int = 1):
    """The pages that each key/value head's queries should look at: int32 ``[batch, kv_heads, count]``, table entries in
    ascending order, -1 behind them, for ``attention_paged(..., selected=)``. A sequence's ``first`` first and ``last``
    last pages are always among them; the others are those with the highest score, the largest that any query head of
    the group could reach with a key inside the page's bounds (ties: the lower entry). Scores are summed in 64 bits, so
    the choice is the same on every run. A page whose bounds are not finite counts among the highest. Sequences of no more
    than ``count`` pages get all of theirs. q ``[batch, heads, 128]``, the cache with its bounds."""
    if cache.bounds is None:
        raise ValueError("the cache has no bounds: paged_kv(..., bounds=True)")
    page_size, heads = cache.k.shape[1:3] if cache.k.dim() == 4 else (0, 0)
    try:
        return _lib.ops().paged_select.default(q, cache.bounds, table, lens, page_size, count, first, last)
    except (RuntimeError, NotImplementedError):
        _check_query(q, heads)
        _check_cache(cache, heads, HEAD_DIM)
        _check_table(table, lens, q.shape[0])
        if count < 1 or first < 0 or last < 0 or first + last > count:
            raise ValueError(f"count {count} with the {first} first and {last} last pages") from None
        raise
