"""Test double for the biased attention's C calls, used by the CPU tests of its host side only.

`library()` replaces `_lib.call_words` by a function that takes the argument structure apart as the library would (addresses and
strides of CPU memory) and fills the outputs from the oracle, so that checks, plans, copies and the autograd glue run without a GPU.
"""

import ctypes
from contextlib import contextmanager

import torch
from torch._functorch.pyfunctorch import temporarily_clear_interpreter_stack

from flashback_cute import _lib, relpos
from oracle import relpos_oracle as orc

TYPES = {0: torch.bfloat16, 1: torch.float16, 2: torch.float32}


def memory(ptr, shape, strides, dtype):
    """The tensor of `shape` and `strides` (elements) at address `ptr`; None for a null pointer."""
    if not ptr:
        return None
    n = 1 + sum((m - 1) * s for m, s in zip(shape, strides))
    raw = (ctypes.c_char * (n * dtype.itemsize)).from_address(ptr)
    return torch.frombuffer(raw, dtype=dtype).as_strided(shape, strides)


def _seq(t, rows, heads, d, dtype):
    return memory(t.ptr, (rows, heads, d), (t.row_stride, t.head_stride, 1), dtype)


def _table(bias, heads, dtype):
    return memory(bias.table, (bias.num_buckets, heads), (bias.bucket_stride, bias.head_stride), dtype)


class Calls(list):
    """(entry point, argument structure) of every call made."""

    def __call__(self, name, words, device):
        struct = {"fb_relpos_fwd": _lib.FbRelposFwdArgs, "fb_relpos_bwd": _lib.FbRelposBwdArgs, "fb_relpos_decode": _lib.FbRelposDecodeArgs,
                  "fb_relpos_bias": _lib.FbRelposBiasArgs, "fb_relpos_bias_grad": _lib.FbRelposBiasGradArgs}[name]
        a = struct.from_buffer_copy(words.tobytes())
        self.append((name, a))
        with temporarily_clear_interpreter_stack():  # the library knows nothing of torch.func
            getattr(self, name, lambda a: None)(a)

    def _attention(self, a, dout=None):
        p, dtype = a.prob, TYPES[a.prob.dtype]
        q = _seq(a.q, p.total_q, p.heads_q, p.head_dim, dtype)
        k, v = (_seq(t, p.total_k, p.heads_kv, p.head_dim, dtype) for t in (a.k, a.v))
        if p.cu_seqlens_q:
            lens = [memory(cu, (p.batch + 1,), (1,), torch.int32).diff().tolist() for cu in (p.cu_seqlens_q, p.cu_seqlens_k)]
            lens = [[min(n, most) for n in ns] for ns, most in zip(lens, (p.seqlen_q, p.seqlen_k))]
        else:
            lens = [[p.seqlen_q] * p.batch, [p.seqlen_k] * p.batch]
        used_q, used_k = sum(lens[0]), sum(lens[1])
        far = self.far
        table = _table(a.bias, p.heads_q, dtype)
        do = None if dout is None else _seq(dout, p.total_q, p.heads_q, p.head_dim, dtype)[:used_q]
        return orc.attention(q[:used_q], k[:used_k], v[:used_k], table, far, bool(a.bias.bidirectional), p.softmax_scale, bool(p.causal), do, *lens), used_q, used_k

    far = 128  # max_distance of the calls

    def fb_relpos_fwd(self, a):
        p, dtype = a.prob, TYPES[a.prob.dtype]
        r, n, _ = self._attention(a)
        out = _seq(a.out, p.total_q, p.heads_q, p.head_dim, dtype)
        out[:n] = r.out.to(dtype)
        if p.flags & _lib.FB_FLAG_ZERO_REST:
            out[n:] = 0

    def fb_relpos_bwd(self, a):
        p, dtype = a.prob, TYPES[a.prob.dtype]
        r, nq, nk = self._attention(a, a.dout)
        for t, g, n, heads, rows in ((a.dq, r.dq, nq, p.heads_q, p.total_q), (a.dk, r.dk, nk, p.heads_kv, p.total_k), (a.dv, r.dv, nk, p.heads_kv, p.total_k)):
            if t.ptr:
                out = _seq(t, rows, heads, p.head_dim, dtype)
                out[:n] = g.to(dtype)
                if p.flags & _lib.FB_FLAG_ZERO_REST:
                    out[n:] = 0
        if a.dtable:
            memory(a.dtable, (a.bias.num_buckets, p.heads_q), (a.dtable_bucket_stride, a.dtable_head_stride), dtype).copy_(r.dt.to(dtype))

    def fb_relpos_decode(self, a):
        dtype, b, sq, sk, hq, hkv, d = TYPES[a.dtype], a.batch, a.seqlen_q, a.seqlen_k, a.heads_q, a.heads_kv, a.head_dim
        strides = lambda t: (t.batch_stride, t.row_stride, t.head_stride, 1)  # noqa: E731
        q = memory(a.q.ptr, (b, sq, hq, d), strides(a.q), dtype)
        k, v = (memory(t.ptr, (b, sk, hkv, d), strides(t), dtype) for t in (a.k, a.v))
        lens = memory(a.lens, (b,), (1,), torch.int32).tolist() if a.lens else [sk] * b
        out = memory(a.out, (b, sq, hq, d), (sq * hq * d, hq * d, d, 1), dtype)
        for i, n in enumerate(lens):
            out[i] = orc.attention(q[i:i + 1], k[i:i + 1, :n], v[i:i + 1, :n], _table(a.bias, hq, dtype), self.far, bool(a.bias.bidirectional), a.softmax_scale, True).out[0].to(dtype)

    which = None  # (sq, sk) buckets of the bias tensor's calls

    def fb_relpos_bias(self, a):
        dtype = TYPES[a.dtype]
        out = memory(a.out, (a.heads, a.seqlen_q, a.seqlen_k), (a.seqlen_q * a.seqlen_k, a.seqlen_k, 1), dtype)
        out.copy_(_table(a.bias, a.heads, dtype).t()[:, self.which])

    def fb_relpos_bias_grad(self, a):
        dtype = TYPES[a.dtype]
        grad = memory(a.grad, (a.heads, a.seqlen_q, a.seqlen_k), (a.seqlen_q * a.seqlen_k, a.seqlen_k, 1), dtype)
        out = memory(a.dtable, (a.bias.num_buckets, a.heads), (a.dtable_bucket_stride, a.dtable_head_stride), dtype)
        for h in range(a.heads):
            out[:, h] = torch.zeros(a.bias.num_buckets, dtype=torch.float64).index_add_(0, self.which.flatten(), grad[h].double().flatten()).to(dtype)


@contextmanager
def library():
    """Calls on CPU tensors inside the block go to the double; gives the list of them."""
    calls = Calls()
    keep = _lib.call_words, relpos._validate
    _lib.call_words, relpos._validate = calls, lambda q, k, v: None
    try:
        yield calls
    finally:
        _lib.call_words, relpos._validate = keep
