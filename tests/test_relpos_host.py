"""CPU tests of the biased attention's host side (checks, plans, copies, autograd glue) with the library replaced by a double."""

import pytest
import torch

from flashback_cute import flashback_attn_relpos_decode
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
