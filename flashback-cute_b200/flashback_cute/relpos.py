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
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from .interface import _validate

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


@functools.lru_cache(maxsize=None)  # (kept: argument templates hold the arrays' addresses)
def _starts_array(side: int, max_distance: int):
    s = bucket_starts(side, max_distance)
    return (ctypes.c_int32 * len(s))(*s)


def _check_buckets(num: int, two: bool, max_distance: int) -> None:
    if not 2 <= num <= _lib.RELPOS_MAX_BUCKETS or (two and (num < 4 or num % 2)):
        raise ValueError(f"bias_table needs 2 to {_lib.RELPOS_MAX_BUCKETS} buckets, even and at least 4 when bidirectional")
    if not (num // 2 if two else num) // 2 < max_distance < 2 ** 30:
        raise ValueError("max_distance must be larger than half the buckets of a side (and below 2**30)")


def _bias(table_shape, table_stride, two: bool, max_distance: int) -> _lib.FbRelpos:
    """The C structure, without the table's address. The array of bucket starts lives as long as the process."""
    num = table_shape[0]
    starts = _starts_array(num // 2 if two else num, max_distance)
    return _lib.FbRelpos(None, table_stride[0], table_stride[1], num, int(two), ctypes.addressof(starts))


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


def _check_cu_seqlens(cu_q, cu_k, q) -> None:
    for cu in (cu_q, cu_k):
        if cu.dtype != torch.int32:
            raise TypeError("cu_seqlens_q and cu_seqlens_k must be int32")
        if cu.dim() != 1 or cu.numel() < 2 or cu.numel() != cu_q.numel() or cu.device != q.device or not cu.is_contiguous():
            raise ValueError("cu_seqlens_q and cu_seqlens_k must be contiguous, of one length (batch + 1) and on the device of q")


def _numbers(max_distance, scale):
    """The options as Python numbers. Plans are found by their values: a tensor among them would be found by its identity, whatever it holds by then."""
    return int(max_distance), None if scale is None else float(scale)


class _Plans:
    """Plans by geometry, a bounded number of them: shapes, strides, types and options, never addresses."""

    def __init__(self, most: int = 1024):
        self.most, self.plans = most, {}
        self.get = self.plans.get

    def add(self, key, plan):
        if len(self.plans) >= self.most:
            self.plans.clear()
        self.plans[key] = plan
        return plan


def _strides_ok(shape, stride) -> bool:
    """Rows x heads x head_dim as the kernels take it: unit stride on head_dim, batch folded into rows, positive strides that are
    multiples of 8 elements. A tensor without elements is never read."""
    if 0 in shape:
        return True
    if stride[-1] != 1 or stride[-2] <= 0 or stride[-3] <= 0 or stride[-2] % 8 or stride[-3] % 8:
        return False
    return len(shape) == 3 or shape[0] <= 1 or stride[0] == shape[1] * stride[1]


def _plain(t: torch.Tensor) -> torch.Tensor:
    """A copy in the standard layout (torch's .contiguous() may keep odd strides of dimensions of size 1)."""
    return torch.empty(t.shape, dtype=t.dtype, device=t.device).copy_(t)


def _plain_strides(shape):
    s = [1]
    for n in reversed(shape[1:]):
        s.append(s[-1] * n)
    return tuple(reversed(s))


def _raw_ptr(t: torch.Tensor) -> int:
    return _raw(t).data_ptr()


def _address():
    """data_ptr, through torch.func's wrappers where a transform is active (tensors made inside one are wrappers themselves)."""
    return _raw_ptr if torch._C._are_functorch_transforms_active() else torch.Tensor.data_ptr


_F, _B = _lib.FbRelposFwdArgs, _lib.FbRelposBwdArgs
_FW = {n: _lib.word(_F, n, "ptr") for n in ("q", "k", "v", "out", "out_low")}
_FW.update(table=_lib.word(_F, "bias", "table"), lse=_lib.word(_F, "lse"), shift=_lib.word(_F, "shift"), cu_q=_lib.word(_F, "prob", "cu_seqlens_q"), cu_k=_lib.word(_F, "prob", "cu_seqlens_k"))
_BW = {n: _lib.word(_B, n, "ptr") for n in ("q", "k", "v", "out", "dout", "out_low", "dq", "dk", "dv")}
_BW.update(table=_lib.word(_B, "bias", "table"), lse=_lib.word(_B, "lse"), shift=_lib.word(_B, "shift"), cu_q=_lib.word(_B, "prob", "cu_seqlens_q"), cu_k=_lib.word(_B, "prob", "cu_seqlens_k"),
           dtable=_lib.word(_B, "dtable"), work=_lib.word(_B, "workspace"))


class _AttnPlan:
    """Everything about one geometry of the attention calls that does not depend on the data: the arguments' checks, templates."""

    def __init__(self, q, k, v, table, cu_q, cu_k, max_q, max_k, max_distance, scale, causal, two):
        _validate(q, k, v)
        _check_shapes(q, k, v, rows=cu_q is not None)
        _check_table(table, q.shape[-2], q)
        if cu_q is not None:
            _check_cu_seqlens(cu_q, cu_k, q)
        q_shape, k_shape, table_shape, dtype, device = tuple(q.shape), tuple(k.shape), tuple(table.shape), q.dtype, q.device
        q_stride, k_stride, v_stride, table_stride = q.stride(), k.stride(), v.stride(), table.stride()
        batch = None if cu_q is None else cu_q.shape[0] - 1
        two = (not causal) if two is None else two
        _check_buckets(table_shape[0], two, max_distance)
        scale = q_shape[-1] ** -0.5 if scale is None else scale
        self.q_shape, self.dtype, self.device, self.index = q_shape, dtype, device, device.index
        self.heads = q_shape[-2]
        packed = batch is not None
        if packed:
            total_q, total_k, b, sq, sk = q_shape[0], k_shape[0], batch, max_q, max_k
        else:
            b, sq, sk = q_shape[0], q_shape[1], k_shape[1]
            total_q, total_k = b * sq, b * sk
        self.total_q, self.stat_bytes = total_q, 4 * self.heads * total_q
        self.empty = 0 in q_shape or 0 in k_shape or 0 in (sq, sk)  # nothing is read, whatever the layouts
        self.copies = not (self.empty or (_strides_ok(q_shape, q_stride) and _strides_ok(k_shape, k_stride) and _strides_ok(k_shape, v_stride)))
        self.low = dtype != torch.float32
        if self.copies or self.empty:
            return
        cu = 16 if packed else None  # an address to come: a problem with cu_seqlens is a packed one
        prob = _lib.FbProblem(
            _lib._DTYPES[dtype], b, self.heads, k_shape[-2], q_shape[-1], sq, sk, int(causal), total_q, total_k, cu, cu, scale,
            _lib.DEFAULT_FLAGS | (_lib.FB_FLAG_ZERO_REST if packed else 0),
        )
        bias = _bias(table_shape, table_stride, two, max_distance)
        t = lambda stride: _lib.FbTensor(None, stride[-3], stride[-2])  # noqa: E731
        o, k = t(_plain_strides(q_shape)), t(_plain_strides(k_shape))
        self.fwd = _lib.template(_F(prob, bias, t(q_stride), t(k_stride), t(v_stride), o, o, None))
        self.bwd = _lib.template(_B(prob, bias, t(q_stride), t(k_stride), t(v_stride), o, o, o, None, o, k, k, None, self.heads, 1, None))
        self.work = _lib.load().fb_relpos_workspace_bytes(ctypes.byref(prob), table_shape[0]) // 4

    def forward(self, q, k, v, table, cu_q, cu_k, train: bool):
        """(out, low, stats); the last two are None unless `train` (low: never for float32). stats: the rows' log-sum-exps and shifts."""
        out = torch.empty(self.q_shape, dtype=self.dtype, device=self.device)
        low = stats = None
        if train:
            stats = torch.empty((2, self.heads, self.total_q), dtype=torch.float32, device=self.device)
            if self.low:
                low = torch.empty(self.q_shape, dtype=self.dtype, device=self.device)
        if self.empty:
            return out.zero_(), low, stats
        ptr, w, i = _address(), self.fwd[:], _FW
        w[i["q"]], w[i["k"]], w[i["v"]], w[i["table"]], w[i["out"]] = ptr(q), ptr(k), ptr(v), ptr(table), ptr(out)
        if stats is not None:
            w[i["lse"]] = at = ptr(stats)
            w[i["shift"]] = at + self.stat_bytes
        if low is not None:
            w[i["out_low"]] = ptr(low)
        if cu_q is not None:
            w[i["cu_q"]], w[i["cu_k"]] = ptr(cu_q), ptr(cu_k)
        _lib.call_words("fb_relpos_fwd", w, self.index)
        return out, low, stats

    def backward(self, q, k, v, table, cu_q, cu_k, out, low, stats, dout, want):
        """[dq, dk, dv, dtable], None where not wanted."""
        grads = [torch.empty(t.shape, dtype=self.dtype, device=self.device) if x else None for t, x in zip((q, k, v, table), want)]
        if self.empty:
            return [t if t is None else t.zero_() for t in grads]
        ptr = _address()
        if ptr(dout) % 16 or not dout.is_contiguous() or dout.stride() != _plain_strides(self.q_shape):
            dout = _plain(dout)
        work = torch.empty(self.work, dtype=torch.float32, device=self.device)
        w, i = self.bwd[:], _BW
        w[i["q"]], w[i["k"]], w[i["v"]], w[i["table"]], w[i["out"]] = ptr(q), ptr(k), ptr(v), ptr(table), ptr(out)
        at = ptr(stats)
        w[i["dout"]], w[i["lse"]], w[i["shift"]], w[i["work"]] = ptr(dout), at, at + self.stat_bytes, ptr(work)
        if low is not None:
            w[i["out_low"]] = ptr(low)
        if cu_q is not None:
            w[i["cu_q"]], w[i["cu_k"]] = ptr(cu_q), ptr(cu_k)
        for name, t in zip(("dq", "dk", "dv", "dtable"), grads):
            if t is not None:
                w[i[name]] = ptr(t)
        _lib.call_words("fb_relpos_bwd", w, self.index)
        return grads


_attn_plans = _Plans()


class _RelposAttnFunc(torch.autograd.Function):
    """(q, k, v, table) -> out; backward gives dq, dk, dv and the table's gradient. First order only."""

    @staticmethod
    def forward(ctx, q, k, v, table, cu_q, cu_k, plan):
        out, low, stats = plan.forward(q, k, v, table, cu_q, cu_k, True)
        ctx.save_for_backward(q, k, v, table, cu_q, cu_k, out, low, stats)
        ctx.plan = plan
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, table, cu_q, cu_k, out, low, stats = ctx.saved_tensors
        return (*ctx.plan.backward(q, k, v, table, cu_q, cu_k, out, low, stats, dout, ctx.needs_input_grad[:4]), None, None, None)


class _RelposAttnTransformed(torch.autograd.Function):
    """The same for torch.func transforms, which ask for setup_context (and for intermediates as outputs)."""

    @staticmethod
    def forward(q, k, v, table, cu_q, cu_k, plan):
        return plan.forward(q, k, v, table, cu_q, cu_k, True)

    @staticmethod
    def setup_context(ctx, inputs, output):
        q, k, v, table, cu_q, cu_k, ctx.plan = inputs
        ctx.mark_non_differentiable(*(t for t in output[1:] if t is not None))
        ctx.save_for_backward(q, k, v, table, cu_q, cu_k, *output)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, *_):
        q, k, v, table, cu_q, cu_k, out, low, stats = map(_raw, ctx.saved_tensors)
        return (*ctx.plan.backward(q, k, v, table, cu_q, cu_k, out, low, stats, _raw(dout), ctx.needs_input_grad[:4]), None, None, None)


def _attention(q, k, v, table, cu_q, cu_k, max_q, max_k, max_distance, scale, causal, two):
    max_distance, scale = _numbers(max_distance, scale)
    causal = bool(causal)
    if two is not None:
        two = bool(two)
    if cu_q is not None:
        max_q, max_k = int(max_q), int(max_k)
    for again in (True, False):
        key = (
            q.shape, k.shape, v.shape, table.shape, q.stride(), k.stride(), v.stride(), table.stride(),
            q.dtype, k.dtype, v.dtype, table.dtype, q.device, k.device, v.device, table.device, max_distance, scale, causal, two, _lib.DEFAULT_FLAGS,
        )
        if cu_q is not None:
            key += (cu_q.shape, cu_k.shape, cu_q.dtype, cu_k.dtype, cu_q.device, cu_k.device, cu_q.stride(), cu_k.stride(), max_q, max_k)
        plan = _attn_plans.get(key)
        if plan is None:
            plan = _attn_plans.add(key, _AttnPlan(q, k, v, table, cu_q, cu_k, max_q, max_k, max_distance, scale, causal, two))
        if not plan.copies:
            break
        assert again, "the standard layout is one that the kernels take"
        q, k, v = (t if _strides_ok(t.shape, t.stride()) else _Plain.apply(t) for t in (q, k, v))
    transformed, ptr = torch._C._are_functorch_transforms_active(), _address()
    if (ptr(q) | ptr(k) | ptr(v)) % 16:
        return _attention(*(_Plain.apply(t) if ptr(t) % 16 else t for t in (q, k, v)), table, cu_q, cu_k, max_q, max_k, max_distance, scale, causal, two)
    if transformed:
        return _RelposAttnTransformed.apply(q, k, v, table, cu_q, cu_k, plan)[0]
    if (torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or table.requires_grad)) or forward_ad._current_level >= 0:
        return _RelposAttnFunc.apply(q, k, v, table, cu_q, cu_k, plan)
    return plan.forward(q, k, v, table, cu_q, cu_k, False)[0]


class _Plain(torch.autograd.Function):
    """Copy into the standard layout."""

    @staticmethod
    def forward(t):
        return _plain(t)

    @staticmethod
    def setup_context(ctx, inputs, output):
        pass

    @staticmethod
    def backward(ctx, g):
        return g

    @staticmethod
    def jvp(ctx, t):
        return t.clone()


class _BiasSpec:
    """Bucket function and template of flashback_relpos_bias for one geometry."""

    def __init__(self, table, sq, sk, two, max_distance):
        if table.dim() != 2 or table.shape[1] == 0:
            raise ValueError("bias_table must have shape (num_buckets, heads)")
        if table.dtype not in (torch.float16, torch.bfloat16, torch.float32):
            raise TypeError("bias_table must be float16, bfloat16 or float32")
        if not table.is_cuda:
            raise NotImplementedError("flashback_cute (B200 build) has no CPU path: tensors must be CUDA tensors")
        if not (0 <= sq <= 1 << 20 and 0 <= sk <= 1 << 30):
            raise ValueError("seqlen_q must be at most 2**20 and seqlen_k at most 2**30")
        table_shape, table_stride, dtype, device = tuple(table.shape), table.stride(), table.dtype, table.device
        _check_buckets(table_shape[0], two, max_distance)
        self.num, self.heads, self.dtype, self.device, self.index = table_shape[0], table_shape[1], dtype, device, device.index
        self.shape = (self.heads, sq, sk)
        lib, code = _lib.load(), _lib._DTYPES[dtype]
        self.fill = _lib.template(_lib.FbRelposBiasArgs(code, self.heads, sq, sk, _bias(table_shape, table_stride, two, max_distance), None))
        self.grad = _lib.template(_lib.FbRelposBiasGradArgs(code, self.heads, sq, sk, _bias(table_shape, table_stride, two, max_distance), None, None, self.heads, 1, None))
        self.work = lib.fb_relpos_bias_workspace_bytes(code, self.heads, sq, sk, self.num) // 4
        self.stride, self.options = table_stride, (sq, sk, two, max_distance)

    def forward(self, table):
        if table.stride() != self.stride:  # (tangents and second-order cotangents come in layouts of their own)
            return _bias_spec(table, *self.options).forward(table)
        out = torch.empty(self.shape, dtype=self.dtype, device=self.device)
        if out.numel():
            ptr, w = _address(), self.fill[:]
            w[_FILL_TABLE], w[_FILL_OUT] = ptr(table), ptr(out)
            _lib.call_words("fb_relpos_bias", w, self.index)
        return out

    def backward(self, grad):
        ptr = _address()
        if not grad.is_contiguous() or ptr(grad) % 16:
            grad = _plain(grad)
        dtable = torch.empty((self.num, self.heads), dtype=self.dtype, device=self.device)
        if grad.numel() == 0:
            return dtable.zero_()
        work = torch.empty(self.work, dtype=torch.float32, device=self.device)
        w = self.grad[:]
        w[_GRAD_IN], w[_GRAD_OUT], w[_GRAD_WORK] = ptr(grad), ptr(dtable), ptr(work)
        _lib.call_words("fb_relpos_bias_grad", w, self.index)
        return dtable


_FILL_TABLE, _FILL_OUT = _lib.word(_lib.FbRelposBiasArgs, "bias", "table"), _lib.word(_lib.FbRelposBiasArgs, "out")
_GRAD_IN, _GRAD_OUT, _GRAD_WORK = (_lib.word(_lib.FbRelposBiasGradArgs, n) for n in ("grad", "dtable", "workspace"))
_bias_specs = _Plans()


def _bias_spec(table, sq, sk, two, max_distance):
    key = (table.shape, table.stride(), table.dtype, table.device, sq, sk, two, max_distance)
    spec = _bias_specs.get(key)
    if spec is None:
        spec = _bias_specs.add(key, _BiasSpec(table, sq, sk, two, max_distance))
    return spec


class _RelposBiasFunc(torch.autograd.Function):
    """table (num_buckets, heads) -> bias (heads, sq, sk). Linear: derivatives of any order, both modes."""

    @staticmethod
    def forward(table, spec):
        return spec.forward(table)

    @staticmethod
    def setup_context(ctx, inputs, output):
        ctx.spec = inputs[1]

    @staticmethod
    def backward(ctx, grad):
        if torch.is_grad_enabled() and grad.requires_grad or torch._C._are_functorch_transforms_active():
            return _RelposBiasGradFunc.apply(grad, ctx.spec), None
        return ctx.spec.backward(grad), None

    @staticmethod
    def jvp(ctx, table_dot, _):
        return ctx.spec.forward(_raw(table_dot))


class _RelposBiasEager(torch.autograd.Function):
    """The same outside torch.func transforms, in the form that costs less per call (no setup_context)."""

    @staticmethod
    def forward(ctx, table, spec):
        ctx.spec = spec
        return spec.forward(table)

    @staticmethod
    def backward(ctx, grad):
        if torch.is_grad_enabled() and grad.requires_grad:
            return _RelposBiasGradFunc.apply(grad, ctx.spec), None
        return ctx.spec.backward(grad), None


class _RelposBiasGradFunc(torch.autograd.Function):
    """The transpose of _RelposBiasFunc: (heads, sq, sk) summed by bucket, (num_buckets, heads)."""

    @staticmethod
    def forward(grad, spec):
        return spec.backward(grad)

    @staticmethod
    def setup_context(ctx, inputs, output):
        ctx.spec = inputs[1]

    @staticmethod
    def backward(ctx, grad2):
        return _RelposBiasFunc.apply(grad2, ctx.spec), None

    @staticmethod
    def jvp(ctx, grad_dot, _):
        return ctx.spec.backward(_raw(grad_dot))


for _fn in (_RelposAttnTransformed, _Plain, _RelposBiasFunc, _RelposBiasGradFunc):  # see interface.py
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
    keys behind their query have buckets of their own; by default unless `causal`. An entry of -inf, or at or below -2^100 (the
    lowest bfloat16 or float32 value), hides its pairs; a row that sees nothing gives zeros. Differentiable once, in q, k, v
    and bias_table (a second derivative raises)."""
    return _attention(q, k, v, bias_table, None, None, None, None, max_distance, softmax_scale, causal, bidirectional)


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
    """The same for packed sequences: q (total_q, hq, d), k/v (total_k, hkv, d), cu_seqlens int32 (b+1,). Rows that belong to no
    sequence (behind cu_seqlens[b]) are not read; their results and gradients are zeros."""
    return _attention(
        q, k, v, bias_table, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k, max_distance, softmax_scale, causal, bidirectional
    )


_D = _lib.FbRelposDecodeArgs
_DW = {n: _lib.word(_D, n, "ptr") for n in ("q", "k", "v")}
_DW.update(table=_lib.word(_D, "bias", "table"), lens=_lib.word(_D, "lens"), out=_lib.word(_D, "out"), work=_lib.word(_D, "workspace"))


class _DecodePlan:
    def __init__(self, q, k, v, lens, table, max_distance, scale, two):
        _validate(q, k, v)
        _check_shapes(q, k, v, rows=False)
        _check_table(table, q.shape[2], q)
        if q.dtype == torch.float32:
            raise TypeError("decoding takes float16 or bfloat16")
        if lens is not None:
            if lens.dtype != torch.int32:
                raise TypeError("cache_seqlens must be int32")
            if lens.shape != q.shape[:1] or lens.device != q.device or not lens.is_contiguous():
                raise ValueError("cache_seqlens must be contiguous, of shape (batch,) and on the device of q")
        q_shape, k_shape, table_shape, dtype = tuple(q.shape), tuple(k.shape), tuple(table.shape), q.dtype
        table_stride = table.stride()
        q_stride, k_stride, v_stride = (tuple(0 if n == 1 else s for n, s in zip(t.shape[:3], t.stride())) + t.stride()[3:] for t in (q, k, v))  # (of one entry: any)
        _check_buckets(table_shape[0], two, max_distance)
        if q_shape[2] // k_shape[2] * table_shape[0] > _lib.DECODE_MAX_TABLE:
            raise ValueError(f"decoding takes at most {_lib.DECODE_MAX_TABLE} table entries per kv head: (heads_q / heads_kv) * num_buckets")
        ok = lambda s: s[3] == 1 and all(x >= 0 and x % 8 == 0 for x in s[:3])  # noqa: E731
        if not (ok(k_stride) and ok(v_stride)):
            raise ValueError("caches need unit stride on head_dim and strides that are multiples of 8 elements")
        self.copy_q = not ok(q_stride)
        self.empty = 0 in q_shape or 0 in k_shape
        cache = lambda s: _lib.FbCache(None, *s[:3])  # noqa: E731
        args = _D(_lib._DTYPES[dtype], q_shape[0], q_shape[2], k_shape[2], q_shape[3], q_shape[1], k_shape[1], q_shape[-1] ** -0.5 if scale is None else scale,
                  _bias(table_shape, table_stride, two, max_distance), cache(_plain_strides(q_shape) if self.copy_q else q_stride), cache(k_stride), cache(v_stride))
        self.words = _lib.template(args)
        self.work = _lib.load().fb_relpos_decode_workspace_bytes(ctypes.byref(args)) // 4


_decode_plans = _Plans()


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
    clamped to [0, s]). (hq / hkv) * num_buckets is at most 4096. Causal: token t of sequence i sits at position cache_seqlens[i] - sq + t. Cache rows at or behind a
    sequence's length are not read. bfloat16 or float16; meant for one to a few tokens (every 16 or 32 (token, head) pairs of a kv head read the
    cache once). No autograd graph."""
    max_distance, softmax_scale = _numbers(max_distance, softmax_scale)
    bidirectional = bool(bidirectional)
    if q.data_ptr() % 16:  # a copy in the standard layout, with the plan of that layout (a clone may have strides of its own)
        with torch.no_grad():
            q = _plain(q)
    key = (
        q.shape, k_cache.shape, v_cache.shape, bias_table.shape, q.stride(), k_cache.stride(), v_cache.stride(), bias_table.stride(),
        q.dtype, k_cache.dtype, v_cache.dtype, bias_table.dtype, q.device, k_cache.device, v_cache.device, bias_table.device,
        max_distance, softmax_scale, bidirectional,
    )
    if cache_seqlens is not None:
        key += (cache_seqlens.shape, cache_seqlens.stride(), cache_seqlens.dtype, cache_seqlens.device)
    plan = _decode_plans.get(key)
    if plan is None:
        plan = _decode_plans.add(key, _DecodePlan(q, k_cache, v_cache, cache_seqlens, bias_table, max_distance, softmax_scale, bidirectional))
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if plan.empty:
        return out.zero_()
    if (k_cache.data_ptr() | v_cache.data_ptr()) % 16:
        raise ValueError("caches need 16-byte alignment")
    if plan.copy_q:
        with torch.no_grad():
            q = _plain(q)
    w, i = plan.words[:], _DW
    w[i["q"]], w[i["k"]], w[i["v"]], w[i["table"]], w[i["out"]] = q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), bias_table.data_ptr(), out.data_ptr()
    if cache_seqlens is not None:
        w[i["lens"]] = cache_seqlens.data_ptr()
    if plan.work:
        work = torch.empty(plan.work, dtype=torch.float32, device=q.device)
        w[i["work"]] = work.data_ptr()
    _lib.call_words("fb_relpos_decode", w, q.device.index)
    return out


def flashback_relpos_bias(
    bias_table: torch.Tensor, seqlen_q: int, seqlen_k: int, max_distance: int = 128, bidirectional: bool = True
) -> torch.Tensor:
    """The bias as a tensor (heads, seqlen_q, seqlen_k) of the table's dtype (bfloat16, float16 or float32): entry (h, i, j) is
    bias_table[bucket(j - (i + seqlen_k - seqlen_q)), h]. For attention that the fused functions do not take (other head
    sizes, masks of its own) and for looking at what was learned. Differentiable in bias_table, any order and mode."""
    seqlen_q, seqlen_k, max_distance, two = int(seqlen_q), int(seqlen_k), int(max_distance), bool(bidirectional)
    spec = _bias_spec(bias_table, seqlen_q, seqlen_k, two, max_distance)
    if forward_ad._current_level >= 0 or torch._C._are_functorch_transforms_active():
        return _RelposBiasFunc.apply(bias_table, spec)
    if torch.is_grad_enabled() and bias_table.requires_grad:
        return _RelposBiasEager.apply(bias_table, spec)
    return spec.forward(bias_table)
