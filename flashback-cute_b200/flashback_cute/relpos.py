"""Attention with a learned relative position bias (no counterpart in the reference).

Query i and key j of a sequence with sq queries and sk keys are r = j - (i + sk - sq) positions apart (bottom-right
aligned, like causal masking). A learned table of shape (num_buckets, heads) holds one number per bucket of r and head:

    S = scale * Q K^T + table[bucket(r), head],   P = softmax(S),   O = P V

  flashback_attn_relpos_func, flashback_attn_relpos_varlen_func   forward, and first-order gradients of q, k, v and the table
  flashback_attn_relpos_decode                                    a few new tokens per sequence against a cache of keys and values
  flashback_relpos_bias                                            the bias as a tensor (heads, sq, sk), differentiable

Buckets (`bucket_starts`): bidirectional, the first half of the table is for r <= 0 and the second for r > 0, both by
n = |r|; otherwise the whole table goes by n = max(-r, 0). Of the nb buckets of a side, distances below e = nb // 2 have one
each; bucket e + t takes the distances with log(n / e) / log(max_distance / e) * (nb - e) >= t, the last one everything
beyond. The comparison is done in whole numbers, so that a distance on a border belongs to the upper bucket on every machine.
"""

from __future__ import annotations

import ctypes
import functools
import inspect
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .interface import _Geom, _stat, _validate

_raw = _lib.raw


@functools.lru_cache(maxsize=256)
def bucket_starts(side: int, max_distance: int) -> tuple:
    """First distance of the buckets 1, 2, ..., side - 1 of a side, ascending (a bucket that no distance falls in starts
    where the next one does)."""
    e = side // 2
    m = side - e
    starts = list(range(1, e))
    for t in range(m):
        bound = max_distance ** t * e ** m  # bucket e + t: n ** m * e ** t >= bound
        lo, hi = e, max_distance
        while lo < hi:
            mid = (lo + hi) // 2
            if mid ** m * e ** t >= bound:
                hi = mid
            else:
                lo = mid + 1
        starts.append(lo)
    return tuple(starts)


@functools.lru_cache(maxsize=256)
def _starts_array(side: int, max_distance: int):
    s = bucket_starts(side, max_distance)
    return (ctypes.c_int32 * len(s))(*s)


class _Buckets:
    """The bucket function of one call: what the C structure needs besides the table."""

    __slots__ = ("num", "two", "starts")

    def __init__(self, num: int, two: bool, max_distance: int):
        self.num, self.two = num, two
        self.starts = _starts_array(num // 2 if two else num, max_distance)

    def bind(self, table: Optional[torch.Tensor]) -> _lib.FbRelpos:
        return _lib.relpos(table, self.num, self.two, self.starts)


def _buckets(num: int, two: bool, max_distance: int) -> _Buckets:
    max_distance = int(max_distance)
    if not 2 <= num <= _lib.RELPOS_MAX_BUCKETS or (two and (num < 4 or num % 2)):
        raise ValueError(f"bias_table needs 2 to {_lib.RELPOS_MAX_BUCKETS} buckets, even and at least 4 when bidirectional")
    if not (num // 2 if two else num) // 2 < max_distance < 2 ** 30:
        raise ValueError("max_distance must be larger than half the buckets of a side (and below 2**30)")
    return _Buckets(num, two, max_distance)


def _check_table(table: torch.Tensor, heads: int, like: torch.Tensor) -> None:
    if table.dim() != 2 or table.shape[1] != heads:
        raise ValueError(f"bias_table must have shape (num_buckets, {heads}), one column per query head")
    if table.dtype != like.dtype:
        raise TypeError("bias_table must share the dtype of q, k, v")
    if table.device != like.device:
        raise ValueError("bias_table must be on the device of q, k, v")


def _check_shapes(q, k, v, rows: bool) -> None:
    """Shapes and devices of q, k, v beyond what `_validate` looks at. rows: packed (total, heads, d) instead of dense."""
    dim = 3 if rows else 4
    if not q.dim() == k.dim() == v.dim() == dim:
        raise ValueError("q, k, v must have %d dimensions" % dim)
    if k.shape != v.shape or (not rows and q.shape[0] != k.shape[0]):
        raise ValueError("k and v must have the same shape, and q, k, v the same batch size")
    if not q.device == k.device == v.device:
        raise ValueError("q, k, v must be on one device")


def _rows(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """`t` in a layout the kernels take (unit stride on head_dim, batch folded into rows, positive strides that are multiples
    of 8 elements, 16-byte aligned), copied only if needed."""
    if t is None or t.numel() == 0 or (_lib.rows_ok(t) and _raw(t).stride(-3) > 0 and _raw(t).stride(-2) > 0):
        return t
    return torch.empty(t.shape, dtype=t.dtype, device=t.device).copy_(t)


class _RelposAttnFunc(torch.autograd.Function):
    """(q, k, v, table) -> (out, lse); backward gives dq, dk, dv and the table's gradient. First order only."""

    @staticmethod
    def forward(q, k, v, table, cu_q, cu_k, max_q, max_k, scale, causal, buckets):
        q, k, v = map(_rows, (q, k, v))
        out, lse = torch.empty(q.shape, dtype=q.dtype, device=q.device), _stat(q, cu_q)
        g = _Geom(q, k, cu_q, cu_k, max_q, max_k, scale, causal)
        if g.empty:
            return out.zero_(), lse.fill_(float("-inf"))
        _lib.relpos_fwd(g.prob, buckets.bind(table), q, k, v, out, lse)
        return out, lse

    @staticmethod
    def setup_context(ctx, inputs, output):
        q, k, v, table, cu_q, cu_k, max_q, max_k, scale, causal, buckets = inputs
        out, lse = output
        ctx.mark_non_differentiable(lse)
        ctx.save_for_backward(q, k, v, table, out, lse, cu_q, cu_k)
        ctx.geom, ctx.buckets = (max_q, max_k, scale, causal), buckets

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, _dlse):
        q, k, v, table, out, lse, cu_q, cu_k = ctx.saved_tensors
        want = ctx.needs_input_grad[:4]
        new = lambda t, wanted: torch.empty(t.shape, dtype=t.dtype, device=t.device) if wanted else None  # noqa: E731
        grads = [new(t, w) for t, w in zip((q, k, v, table), want)]
        q, k, v, out, dout = map(_rows, (q, k, v, out, dout))
        g = _Geom(q, k, cu_q, cu_k, *ctx.geom)
        if g.empty:
            grads = [t if t is None else t.zero_() for t in grads]
        elif any(want):
            dpsum = _stat(q, cu_q)
            _lib.bwd_row_stats(g.prob, out, dout, None, None, dpsum, None)
            _lib.relpos_bwd(g.prob, ctx.buckets.bind(table), q, k, v, dout, lse, dpsum, *grads)
        return (*grads, *((None,) * 7))


class _RelposBiasFunc(torch.autograd.Function):
    """table (num_buckets, heads) -> bias (heads, sq, sk). Linear: derivatives of any order, both modes."""

    @staticmethod
    def forward(table, sq, sk, buckets):
        out = torch.empty(table.shape[1], sq, sk, dtype=table.dtype, device=table.device)
        if out.numel():
            _lib.relpos_bias(buckets.bind(table), out)
        return out

    @staticmethod
    def setup_context(ctx, inputs, output):
        _, ctx.sq, ctx.sk, ctx.buckets = inputs

    @staticmethod
    def backward(ctx, grad):
        return _RelposBiasGradFunc.apply(grad, ctx.buckets), None, None, None

    @staticmethod
    def jvp(ctx, table_dot, *_):
        return _RelposBiasFunc.forward(_raw(table_dot), ctx.sq, ctx.sk, ctx.buckets)


class _RelposBiasGradFunc(torch.autograd.Function):
    """The transpose of _RelposBiasFunc: (heads, sq, sk) summed by bucket, (num_buckets, heads)."""

    @staticmethod
    def forward(grad, buckets):
        grad = grad.contiguous()
        if grad.data_ptr() % 16:
            grad = grad.clone()
        dtable = torch.empty(buckets.num, grad.shape[0], dtype=grad.dtype, device=grad.device)
        if grad.numel() == 0:
            return dtable.zero_()
        _lib.relpos_bias_grad(buckets.bind(None), grad, dtable)
        return dtable

    @staticmethod
    def setup_context(ctx, inputs, output):
        grad, ctx.buckets = inputs
        ctx.sizes = grad.shape[1:]

    @staticmethod
    def backward(ctx, grad2):
        return _RelposBiasFunc.apply(grad2, *ctx.sizes, ctx.buckets), None

    @staticmethod
    def jvp(ctx, grad_dot, *_):
        return _RelposBiasGradFunc.forward(_raw(grad_dot), ctx.buckets)


for _fn in (_RelposAttnFunc, _RelposBiasFunc, _RelposBiasGradFunc):  # see interface.py
    _fn.forward.__signature__ = inspect.signature(_fn.forward)


def flashback_attn_relpos_func(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    bias_table: torch.Tensor,
    max_distance: int = 128,
    softmax_scale: Optional[float] = None,
    causal: bool = False,
    bidirectional: Optional[bool] = None,
) -> torch.Tensor:
    """Softmax attention with a learned relative position bias: q (b, sq, hq, d), k/v (b, sk, hkv, d), bias_table
    (num_buckets, hq) of the same dtype (bfloat16, float16 or float32; float32 runs on CUDA cores). bidirectional: whether
    keys behind their query have buckets of their own; by default unless `causal`. Differentiable once, in q, k, v and
    bias_table."""
    _validate(q, k, v)
    _check_shapes(q, k, v, rows=False)
    _check_table(bias_table, q.shape[2], q)
    b = _buckets(bias_table.shape[0], (not causal) if bidirectional is None else bool(bidirectional), max_distance)
    if softmax_scale is None:
        softmax_scale = q.shape[-1] ** -0.5
    return _RelposAttnFunc.apply(q, k, v, bias_table, None, None, None, None, softmax_scale, causal, b)[0]


def flashback_attn_relpos_varlen_func(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    bias_table: torch.Tensor,
    cu_seqlens_q: torch.Tensor,
    cu_seqlens_k: torch.Tensor,
    max_seqlen_q: int,
    max_seqlen_k: int,
    max_distance: int = 128,
    softmax_scale: Optional[float] = None,
    causal: bool = False,
    bidirectional: Optional[bool] = None,
) -> torch.Tensor:
    """The same for packed sequences: q (total_q, hq, d), k/v (total_k, hkv, d), cu_seqlens int32 (b+1,)."""
    _validate(q, k, v)
    _check_shapes(q, k, v, rows=True)
    _check_table(bias_table, q.shape[1], q)
    for cu in (cu_seqlens_q, cu_seqlens_k):
        if cu.dtype != torch.int32:
            raise TypeError("cu_seqlens_q and cu_seqlens_k must be int32")
        if cu.dim() != 1 or cu.numel() < 2 or cu.numel() != cu_seqlens_q.numel() or cu.device != q.device or not cu.is_contiguous():
            raise ValueError("cu_seqlens_q and cu_seqlens_k must be contiguous, of one length (batch + 1) and on the device of q")
    b = _buckets(bias_table.shape[0], (not causal) if bidirectional is None else bool(bidirectional), max_distance)
    if softmax_scale is None:
        softmax_scale = q.shape[-1] ** -0.5
    return _RelposAttnFunc.apply(
        q, k, v, bias_table, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k, softmax_scale, causal, b
    )[0]


def _cache_ok(t: torch.Tensor) -> bool:
    return t.stride(3) == 1 and t.data_ptr() % 16 == 0 and all(t.stride(i) >= 0 and t.stride(i) % 8 == 0 for i in range(3))


def flashback_attn_relpos_decode(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    cache_seqlens: Optional[torch.Tensor],
    bias_table: torch.Tensor,
    max_distance: int = 128,
    softmax_scale: Optional[float] = None,
    bidirectional: bool = False,
) -> torch.Tensor:
    """Attention of the newest tokens of every sequence: q (b, sq, hq, d) against caches (b, s, hkv, d) that already hold
    their keys and values. cache_seqlens, int32 (b,) on the device of q: keys per sequence, the new tokens included (None: s each; values are
    clamped to [0, s]). Causal: token t of sequence i sits at position cache_seqlens[i] - sq + t. Cache rows at or behind a
    sequence's length are not read. bfloat16 or float16; meant for one to a few tokens (every 16 or 32 (token, head) pairs of a kv head read the
    cache once). No autograd graph."""
    _validate(q, k_cache, v_cache)
    _check_shapes(q, k_cache, v_cache, rows=False)
    _check_table(bias_table, q.shape[2], q)
    if q.dtype == torch.float32:
        raise TypeError("decoding takes float16 or bfloat16")
    if cache_seqlens is not None:
        if cache_seqlens.dtype != torch.int32:
            raise TypeError("cache_seqlens must be int32")
        if cache_seqlens.shape != q.shape[:1] or cache_seqlens.device != q.device or not cache_seqlens.is_contiguous():
            raise ValueError("cache_seqlens must be contiguous, of shape (batch,) and on the device of q")
    b = _buckets(bias_table.shape[0], bool(bidirectional), max_distance)
    if softmax_scale is None:
        softmax_scale = q.shape[-1] ** -0.5
    with torch.no_grad():
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        if out.numel() == 0 or k_cache.numel() == 0:
            return out.zero_()
        if not (_cache_ok(k_cache) and _cache_ok(v_cache)):
            raise ValueError("caches need unit stride on head_dim, strides that are multiples of 8 elements and 16-byte alignment")
        if not _cache_ok(q):
            q = torch.empty(q.shape, dtype=q.dtype, device=q.device).copy_(q)
        _lib.relpos_decode(b.bind(bias_table), q, k_cache, v_cache, cache_seqlens, out, softmax_scale)
    return out


def flashback_relpos_bias(
    bias_table: torch.Tensor, seqlen_q: int, seqlen_k: int, max_distance: int = 128, bidirectional: bool = True
) -> torch.Tensor:
    """The bias as a tensor (heads, seqlen_q, seqlen_k) of the table's dtype (bfloat16, float16 or float32): entry (h, i, j) is
    bias_table[bucket(j - (i + seqlen_k - seqlen_q)), h]. For attention that the fused functions do not take (other head
    sizes, masks of its own) and for looking at what was learned. Differentiable in bias_table, any order and mode."""
    if bias_table.dim() != 2 or bias_table.shape[1] == 0:
        raise ValueError("bias_table must have shape (num_buckets, heads)")
    if bias_table.dtype not in (torch.float16, torch.bfloat16, torch.float32):
        raise TypeError("bias_table must be float16, bfloat16 or float32")
    if not bias_table.is_cuda:
        raise NotImplementedError("flashback_cute (B200 build) has no CPU path: tensors must be CUDA tensors")
    if not (0 <= seqlen_q <= 1 << 20 and 0 <= seqlen_k <= 1 << 30):
        raise ValueError("seqlen_q must be at most 2**20 and seqlen_k at most 2**30")
    b = _buckets(bias_table.shape[0], bool(bidirectional), max_distance)
    return _RelposBiasFunc.apply(bias_table, int(seqlen_q), int(seqlen_k), b)
