"""CPU tests of the biased attention's host side (checks, plans, copies, autograd glue) with the library replaced by a double."""

import ctypes
import math
from types import SimpleNamespace

import pytest
import torch

from flashback_cute import _lib, flashback_attn_relpos_decode, flashback_attn_relpos_func, flashback_attn_relpos_varlen_func, flashback_relpos_bias, relpos
from oracle import relpos_oracle as orc
from tests import relpos_double as double

BF16 = torch.bfloat16


def _mk(shape, seed, dtype=BF16):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _decode_want(q, k, v, table):
    return orc.attention(q, k, v, table, 128, False, q.shape[-1] ** -0.5, True).out.to(q.dtype)


# ---------------------------------------------------------------------------------------------
# decoding: layouts of q
# ---------------------------------------------------------------------------------------------
def odd_queries():
    """Queries of strides that the kernel takes at an address that it does not take (8 bytes off), dense and not."""
    one = _mk((3, 1, 8, 72), 0)[..., 4:68]                                     # a slice of wider heads
    fused = _mk((2 * 3 * 12 * 64 + 4,), 1)[4:].view(2, 3, 12, 64)[:, :, :8]    # the query heads of a fused buffer
    dense = _mk((2 * 3 * 8 * 64 + 4,), 2)[4:].view(2, 3, 8, 64)
    turned = _mk((2 * 8 * 3 * 64 + 4,), 3)[4:].view(2, 8, 3, 64).transpose(1, 2)
    same = _mk((8 * 64 + 4,), 4)[4:].view(1, 1, 8, 64).expand(3, 2, 8, 64)     # one query for every sequence and token
    return dict(one=one, fused=fused, dense=dense, turned=turned, same=same)


@pytest.mark.parametrize("which", list(odd_queries()))
def test_decode_takes_queries_at_any_address(which):
    q = odd_queries()[which]
    assert q.data_ptr() % 16 == 8
    k, v, table = _mk((q.shape[0], 9, 4, 64), 10), _mk((q.shape[0], 9, 4, 64), 11), _mk((32, 8), 12)
    with double.library() as calls:
        got = flashback_attn_relpos_decode(q, k, v, None, table)
        again = flashback_attn_relpos_decode(_mk(q.shape, 13), k, v, None, table)  # the plans of other layouts stay what they are
    assert all(a.q.ptr % 16 == 0 for _, a in calls)
    assert torch.equal(got, _decode_want(q, k, v, table))
    assert torch.equal(again, _decode_want(_mk(q.shape, 13), k, v, table))


# ---------------------------------------------------------------------------------------------
# options that are tensors and change between calls
# ---------------------------------------------------------------------------------------------
def test_options_count_by_their_value():
    """Lengths, scales, distances and sizes handed over as 0-dim tensors, changed in place: the call uses what they hold."""
    longest, scale, far = torch.tensor(40), torch.tensor(0.125), torch.tensor(128)
    q, k, v, table = _mk((160, 8, 64), 0), _mk((160, 4, 64), 1), _mk((160, 4, 64), 2), _mk((32, 8), 3)
    cu = torch.tensor([0, 40, 60], dtype=torch.int32)
    qd, kd = _mk((2, 1, 8, 64), 4), _mk((2, 9, 4, 64), 5)
    spec = relpos._BiasSpec
    with double.library() as calls:
        for n, c, f in ((40, 0.125, 128), (100, 1.0, 64)):
            longest.fill_(n), scale.fill_(c), far.fill_(f)
            cu[1:] = torch.tensor([n, n + 20])
            calls.far = f
            flashback_attn_relpos_varlen_func(q, k, v, table, cu, cu, longest, longest, max_distance=far, softmax_scale=scale, causal=torch.tensor(True))
            flashback_attn_relpos_decode(qd, kd, kd, None, table, max_distance=far, softmax_scale=scale)
            fwd, dec = calls[-2][1], calls[-1][1]
            assert (fwd.prob.seqlen_q, fwd.prob.seqlen_k, fwd.prob.softmax_scale, fwd.prob.causal) == (n, n, c, 1)
            assert dec.softmax_scale == c
            starts = relpos.bucket_starts(32, f)
            for a in (fwd, dec):
                assert tuple((ctypes.c_int32 * 31).from_address(a.bias.starts)) == starts
    # the sizes of the bias tensor: the look-up, with the plan's device check out of the way
    made = []
    relpos._BiasSpec = lambda table, sq, sk, two, far: made.append((sq, sk, two, far)) or SimpleNamespace(forward=lambda t: (sq, sk, far))
    try:
        size = torch.tensor(5)
        for n in (5, 9):
            size.fill_(n), far.fill_(100 + n)
            assert flashback_relpos_bias(table, size, size, max_distance=far) == (n, n, 100 + n)
        assert all(type(x) in (int, bool) for m in made for x in m)
    finally:
        relpos._BiasSpec = spec
        relpos._bias_specs.plans.clear()


# ---------------------------------------------------------------------------------------------
# sequences of length zero
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("b", [1, 2, 3])
@pytest.mark.parametrize("sq,sk", [(0, 5), (5, 0), (0, 0)])
def test_dense_batches_of_empty_sequences(b, sq, sk, monkeypatch):
    """No loop of copies (torch's strides of an empty tensor are not those of rows folded into the batch)."""
    copies, plain = [], relpos._plain
    monkeypatch.setattr(relpos, "_plain", lambda t: copies.append(t) or (plain(t) if len(copies) < 20 else pytest.fail("copies without end")))
    for turned in (False, True):
        mk = lambda s, h, seed: _mk((b, h, s, 64), seed).transpose(1, 2) if turned else _mk((b, s, h, 64), seed)  # noqa: E731
        leaves = [t.requires_grad_() for t in (mk(sq, 4, 0), mk(sk, 2, 1), mk(sk, 2, 2), _mk((32, 4), 3))]
        with double.library() as calls:
            out = flashback_attn_relpos_func(*leaves, causal=True)
            grads = torch.autograd.grad(out, leaves, torch.ones_like(out))
            assert flashback_attn_relpos_decode(leaves[0], leaves[1], leaves[2], None, leaves[3]).shape == out.shape
        assert not calls and out.shape == (b, sq, 4, 64) and (out == 0).all()
        assert all(g.shape == t.shape and (g == 0).all() for g, t in zip(grads, leaves))


# ---------------------------------------------------------------------------------------------
# flags of the binding
# ---------------------------------------------------------------------------------------------
def test_flags_of_the_call_count(monkeypatch):
    """`_lib.DEFAULT_FLAGS` as it is at the call, like the rest of the binding, also for a layout seen before."""
    q, k, table = _mk((1, 5, 4, 64), 0), _mk((1, 5, 2, 64), 1), _mk((32, 4), 2)
    with double.library() as calls:
        for flags in (0, _lib.FB_FLAG_FORCE_SIMT, 0):
            monkeypatch.setattr(_lib, "DEFAULT_FLAGS", flags)
            leaf = q.clone().requires_grad_()
            torch.autograd.grad(flashback_attn_relpos_func(leaf, k, k, table).sum(), leaf)
            assert [a.prob.flags for _, a in calls[-2:]] == [flags, flags]


# ---------------------------------------------------------------------------------------------
# addresses under torch.func
# ---------------------------------------------------------------------------------------------
def test_misaligned_inputs_under_torch_func():
    off = lambda shape, seed: _mk((math.prod(shape) + 4,), seed)[4:].view(shape)  # noqa: E731
    q, k, v, table = off((2, 5, 4, 64), 0), off((2, 6, 2, 64), 1), off((2, 6, 2, 64), 2), _mk((32, 4), 3)
    assert all(t.data_ptr() % 16 == 8 for t in (q, k, v))
    loss = lambda *a: flashback_attn_relpos_func(*a, causal=True).float().sum()  # noqa: E731
    with double.library() as calls:
        got = torch.func.grad(loss, argnums=(0, 1, 2, 3))(q, k, v, table)
        leaves = [t.clone().requires_grad_() for t in (q, k, v, table)]
        want = torch.autograd.grad(loss(*leaves), leaves)
    assert all(t.ptr % 16 == 0 for _, a in calls for t in (a.q, a.k, a.v))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---------------------------------------------------------------------------------------------
# the bias tensor of a broadcast table
# ---------------------------------------------------------------------------------------------
def test_derivatives_of_the_bias_of_a_broadcast_table(monkeypatch):
    """One column for every head (stride 0): tangents and second-order cotangents have layouts of their own."""
    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda t: True))
    column = _mk((8, 1), 0, torch.float32)
    which = orc.buckets(5, 7, 8, 6, True)
    bias = lambda c: flashback_relpos_bias(c.expand(-1, 3), 5, 7, max_distance=6)  # noqa: E731
    way, w = _mk((8, 1), 1, torch.float32), _mk((3, 5, 7), 2, torch.float32).requires_grad_()
    with double.library() as calls:
        calls.which = which
        _, tangent = torch.func.jvp(bias, (column,), (way,))
        assert torch.equal(tangent, way.expand(-1, 3).t()[:, which])
        spread = torch.randn(8, 3)
        leaf = column.expand(-1, 3).detach().requires_grad_()
        assert leaf.stride() == (1, 0)
        first = torch.autograd.grad((flashback_relpos_bias(leaf, 5, 7, max_distance=6) * w).sum(), leaf, create_graph=True)[0]
        assert torch.equal(torch.autograd.grad((first * spread).sum(), w)[0], spread.t()[:, which])


# ---------------------------------------------------------------------------------------------
# packed tensors longer than their sequences
# ---------------------------------------------------------------------------------------------
def test_rows_of_no_sequence_get_zeros(monkeypatch):
    """Results and gradients come from memory that may hold anything; the call asks for zeros in the rows that no sequence has."""
    fresh = torch.empty
    monkeypatch.setattr(torch, "empty", lambda *a, **kw: fresh(*a, **kw).fill_(float("nan")))
    q, k, v, do, table = _mk((50, 4, 64), 0), _mk((50, 2, 64), 1), _mk((50, 2, 64), 2), _mk((50, 4, 64), 3), _mk((32, 4), 4)
    for t in (q, k, v, do):
        t[30:] = float("nan")
    for lens in ([20, 10], [30, 0], [0, 0]):
        cu = torch.tensor([0, lens[0], sum(lens)], dtype=torch.int32)
        leaves = [t.clone().requires_grad_() for t in (q, k, v, table)]
        with double.library():
            out = flashback_attn_relpos_varlen_func(*leaves, cu, cu, max(lens), max(lens), causal=True)
            grads = torch.autograd.grad(out, leaves, do)
        assert all((t[sum(lens):] == 0).all() for t in (out, *grads[:3]))
        assert all(torch.isfinite(t).all() for t in (out, *grads))


# ---------------------------------------------------------------------------------------------
# decoding: strides of dimensions of size one, the table's limit
# ---------------------------------------------------------------------------------------------
def test_decode_strides_of_single_entries_do_not_matter():
    """One sequence or one head out of buffers with odd strides between them."""
    buf = _mk((9 * 4 * 64 + 3,), 0)
    k = buf[: 9 * 4 * 64].as_strided((1, 9, 4, 64), (9 * 4 * 64 + 3, 256, 64, 1))
    one = _mk((2, 9, 64), 1).as_strided((2, 9, 1, 64), (576, 64, 3, 1))
    q, table = _mk((1, 1, 8, 64), 2), _mk((32, 8), 3)
    with double.library() as calls:
        assert torch.equal(flashback_attn_relpos_decode(q, k, k, None, table), _decode_want(q, k, k, table))
        q2 = _mk((2, 1, 8, 64), 4)
        assert torch.equal(flashback_attn_relpos_decode(q2, one, one, None, table), _decode_want(q2, one, one, table))
    assert all(s % 8 == 0 for _, a in calls for t in (a.q, a.k, a.v) for s in (t.batch_stride, t.row_stride, t.head_stride))
    odd = buf.as_strided((2, 3, 4, 64), (771, 256, 64, 1))
    with double.library(), pytest.raises(ValueError):  # between several of them: the kernel's loads need the alignment
        flashback_attn_relpos_decode(q2, odd, odd, None, table)


def test_decode_refuses_tables_beyond_shared_memory():
    k = _mk((1, 3, 1, 64), 0)
    with double.library(), pytest.raises(ValueError, match="4096"):
        flashback_attn_relpos_decode(_mk((1, 1, 64, 64), 1), k, k, None, _mk((128, 64), 2))
