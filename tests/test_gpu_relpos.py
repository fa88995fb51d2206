"""GPU tests of attention with a learned relative position bias, against the float64 oracle and its bounds
(oracle/relpos_oracle.py derives them: half a step of the type for every rounding, float32 sums)."""

import itertools

import pytest
import torch

from flashback_cute import _lib, flashback_attn_func, flashback_attn_relpos_func, flashback_attn_relpos_varlen_func, flashback_relpos_bias
from oracle import relpos_oracle as orc

pytestmark = pytest.mark.gpu
if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

DEV = "cuda"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _device_status_clean():
    yield
    torch.cuda.synchronize()
    _lib.check_device_status()


def _within(name, got, want, tol):
    """|got - want| <= tol, element by element (smallest denormals of float16 aside: half a step of 2^-24)."""
    assert got.shape == want.shape, name
    assert torch.isfinite(got).all(), name
    over = (got.double() - want).abs() - tol - 2.0 ** -25
    worst = over.max().item() if over.numel() else -1.0
    assert worst <= 0, f"{name}: {worst:.3e} beyond the bound (largest bound {tol.max().item():.3e}, largest value {want.abs().max().item():.3e})"


def _mk(shape, dtype, seed, std=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=DEV) * std).to(dtype)


def _check(dtype, d, hq, hkv, causal, batch, sq, sk, num=32, far=128, two=None, seed=0, table=None, packed=None):
    """Forward and gradients of one dense or packed (`packed`: lists of lengths) problem."""
    two = (not causal) if two is None else two
    if packed:
        q, k, v, do = (_mk((sum(n), h, d), dtype, seed + i) for i, (n, h) in enumerate(zip((packed[0], packed[1], packed[1], packed[0]), (hq, hkv, hkv, hq))))
        cu = [torch.tensor([0, *itertools.accumulate(n)], dtype=torch.int32, device=DEV) for n in packed]
    else:
        q, k, v, do = (_mk((batch, s, h, d), dtype, seed + i) for i, (s, h) in enumerate(((sq, hq), (sk, hkv), (sk, hkv), (sq, hq))))
    table = _mk((num, hq), dtype, seed + 9) if table is None else table
    leaves = [t.clone().requires_grad_() for t in (q, k, v, table)]
    if packed:
        out = flashback_attn_relpos_varlen_func(*leaves, *cu, max(packed[0]), max(packed[1]), max_distance=far, causal=causal, bidirectional=two)
    else:
        out = flashback_attn_relpos_func(*leaves, max_distance=far, causal=causal, bidirectional=two)
    grads = torch.autograd.grad(out, leaves, do)
    ref = orc.attention(q, k, v, table, far, two, d ** -0.5, causal, do, *(packed or (None, None)))
    for name, got, want, tol in zip(("out", "dq", "dk", "dv", "dtable"), (out.detach(), *grads), ref[:5], ref.tol):
        _within(name, got, want, tol)


@pytest.mark.parametrize("sizes", [(1, 1), (1, 300), (128, 128), (129, 65), (200, 333), (300, 97), (64, 640)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("d", [64, 128])
def test_dense_bf16(d, causal, sizes):
    _check(BF16, d, 4, 2, causal, 2, *sizes)


@pytest.mark.parametrize("heads", [(3, 3), (6, 1)])
@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("d", [64, 128])
def test_types_and_heads(d, dtype, heads):
    _check(dtype, d, *heads, True, 2, 150, 211)
    _check(dtype, d, *heads, False, 1, 97, 97)


@pytest.mark.parametrize("num,far,two", [(2, 2, False), (4, 2, True), (8, 5, True), (32, 17, False), (64, 1024, False), (128, 300, True), (128, 65, False)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_buckets(dtype, num, far, two):
    """Few and many buckets, borders closer than a tile and beyond the sequence, also both-sided under a causal mask."""
    _check(dtype, 64, 2, 1, False, 1, 333, 401, num, far, two)
    _check(dtype, 64, 2, 1, True, 1, 401, 333, num, far, two)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("heads", [(4, 4), (4, 1)])
def test_packed(heads, causal, dtype):
    _check(dtype, 64, *heads, causal, None, None, None, packed=([37, 200, 1, 129, 0, 64], [50, 200, 7, 300, 0, 64]))
    _check(dtype, 128, *heads, causal, None, None, None, packed=([300, 1, 0, 257], [290, 1, 5, 257]))


def test_long_rows_share_one_bucket():
    """Blocks far from the diagonal take the path of a single bucket; 1500 rows cross it on both sides."""
    _check(BF16, 64, 2, 1, False, 1, 1500, 1500)
    _check(BF16, 128, 1, 1, True, 1, 1500, 1500, 32, 64)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_entries_that_hide_or_that_nobody_points_at(dtype):
    """-inf in the table hides its pairs (rows that see nothing give zeros); infinities and NaN in entries that only masked
    or absent pairs point at do no harm."""
    hq, num = 2, 32
    table = _mk((num, hq), dtype, 3)
    table[0, 0] = -float("inf")  # the query's own position: the first row sees nothing
    table[5, 1] = -float("inf")
    _check(dtype, 64, hq, 1, True, 1, 200, 200, table=table)
    table = _mk((num, hq), dtype, 4)
    table[num // 2:] = float("nan")  # keys behind the query: masked
    table[num // 2 + 3:, 0] = float("inf")
    _check(dtype, 64, hq, 1, True, 2, 77, 77, two=True, table=table)
    table = _mk((num, hq), dtype, 5)
    table[12:] = float("inf")  # distances from 12 on: longer than any of these sequences
    _check(dtype, 64, hq, 1, True, None, None, None, two=False, far=128, table=table, packed=([7, 1, 12, 3], [7, 1, 12, 3]))


def test_lowest_values_hide():
    """The lowest bfloat16 / float32 value hides like -inf, also where a row sees nothing else; the lowest float16 value is a number."""
    for dtype in (BF16, F32):
        table = _mk((32, 2), dtype, 3)
        table[0, 0] = torch.finfo(dtype).min
        table[7, 1] = torch.finfo(dtype).min
        hidden = table.clone()
        hidden[0, 0] = hidden[7, 1] = -float("inf")
        q, k, v, do = (_mk((1, 150, 2, 64), dtype, i) for i in range(4))
        res = []
        for t in (table, hidden):
            leaves = [x.clone().requires_grad_() for x in (q, k, v, t)]
            out = flashback_attn_relpos_func(*leaves, causal=True)
            res.append((out.detach(), *torch.autograd.grad(out, leaves, do)))
        assert all(torch.equal(a, b) for a, b in zip(*res)) and (res[0][0][:, 0, 0] == 0).all()
    table = _mk((32, 2), F16, 3)
    table[9] = torch.finfo(F16).min
    _check(F16, 64, 2, 1, False, 1, 150, 150, table=table)


@pytest.mark.parametrize("scale", [-0.2, 0.0, 1.5])
def test_scales(scale):
    """Negative, zero and large scales (the row maximum follows the bias and the scaled scores)."""
    q, k, v, do = (_mk((2, 190, 2, 64), BF16, i) for i in range(4))
    leaves = [t.clone().requires_grad_() for t in (q, k, v, _mk((32, 2), BF16, 8))]
    for causal in (False, True):
        out = flashback_attn_relpos_func(*leaves, softmax_scale=scale, causal=causal)
        grads = torch.autograd.grad(out, leaves, do)
        ref = orc.attention(q, k, v, leaves[3], 128, not causal, scale, causal, do)
        for name, got, want, tol in zip(("out", "dq", "dk", "dv", "dtable"), (out.detach(), *grads), ref[:5], ref.tol):
            _within(name, got, want, tol)


def test_broadcast_inputs():
    """One set of keys for every batch entry, one column for every head: gradients are summed by what expanded them."""
    q, k, v, do = _mk((3, 100, 4, 64), BF16, 0), _mk((1, 100, 2, 64), BF16, 1), _mk((1, 100, 2, 64), BF16, 2), _mk((3, 100, 4, 64), BF16, 3)
    column = _mk((32, 1), BF16, 4)
    leaves = [t.clone().requires_grad_() for t in (q, k, v, column)]
    out = flashback_attn_relpos_func(leaves[0], leaves[1].expand(3, -1, -1, -1), leaves[2].expand(3, -1, -1, -1), leaves[3].expand(-1, 4))
    grads = torch.autograd.grad(out, leaves, do)
    ref = orc.attention(q, k.expand(3, -1, -1, -1), v.expand(3, -1, -1, -1), column.expand(-1, 4), 128, True, 0.125, False, do)
    sums = [ref.dq, ref.dk.sum(0, True), ref.dv.sum(0, True), ref.dt.sum(1, True)]
    tols = [ref.tol[1], ref.tol[2].sum(0, True), ref.tol[3].sum(0, True), ref.tol[4].sum(1, True)]
    for name, got, want, tol in zip(("dq", "dk", "dv", "dcolumn"), grads, sums, tols):
        _within(name, got, want, tol * 1.01 + 3 * torch.finfo(BF16).eps / 2 * want.abs())  # torch adds the parts in bfloat16 steps


def test_cuda_core_kernels_agree():
    """The CUDA-core kernels on 16-bit inputs (FB_FLAG_FORCE_SIMT), a second implementation, within the same bounds."""
    flags, _lib.DEFAULT_FLAGS = _lib.DEFAULT_FLAGS, _lib.FB_FLAG_FORCE_SIMT
    from flashback_cute import relpos

    relpos._attn_plans.plans.clear()
    try:
        _check(BF16, 64, 4, 2, True, 1, 77, 90)
        _check(F16, 128, 2, 1, False, None, None, None, packed=([33, 1, 50], [33, 4, 50]))
    finally:
        _lib.DEFAULT_FLAGS = flags
        relpos._attn_plans.plans.clear()


def test_strides_and_offsets():
    """Views: heads before rows, sliced heads, an offset into a larger tensor, a transposed table, a broadcast gradient."""
    b, s, hq, hkv, d = 2, 130, 4, 2, 64
    q = _mk((b, hq, s, d), BF16, 0).transpose(1, 2)
    k = _mk((b, s, hkv + 3, d), BF16, 1)[:, :, 1:1 + hkv]
    v = _mk((b, s, hkv, 2 * d), BF16, 2)[..., d:]
    odd = _mk((s * hkv * b * d + 1,), BF16, 4)[1:].view(b, s, hkv, d)
    table = _mk((hq, 32), BF16, 3).t()
    leaves = [t.requires_grad_() for t in (q, k, v, table)]
    out = flashback_attn_relpos_func(*leaves, causal=True)
    grads = torch.autograd.grad(out.float().sum(), leaves)
    ref = orc.attention(*leaves, 128, False, d ** -0.5, True, torch.ones_like(out))
    for name, got, want, tol in zip(("out", "dq", "dk", "dv", "dtable"), (out.detach(), *grads), ref[:5], ref.tol):
        _within(name, got, want, tol)
    out = flashback_attn_relpos_func(q, odd, odd, table, causal=True)
    ref = orc.attention(q, odd, odd, table, 128, False, d ** -0.5, True)
    _within("out", out.detach(), ref.out, ref.tol[0])


def test_zero_table_is_plain_attention():
    q, k, v = _mk((2, 256, 4, 64), BF16, 0), _mk((2, 256, 2, 64), BF16, 1), _mk((2, 256, 2, 64), BF16, 2)
    got = flashback_attn_relpos_func(q, k, v, torch.zeros(32, 4, dtype=BF16, device=DEV), causal=True)
    want = flashback_attn_func(q, k, v, causal=True)
    assert (got.float() - want.float()).abs().max() <= 2 * torch.finfo(BF16).eps * want.abs().max()


def test_gradient_of_the_table_against_differences():
    """Central differences of <O, dO> in the float32 path along a random direction of the table: the step's square times the third derivative
    and float32 rounding of O over the step are both below 1e-3 of the value here."""
    q, k, v, do = (_mk((1, 90, 2, 64), F32, i) for i in range(4))
    table, way = _mk((32, 2), F32, 5), _mk((32, 2), F32, 6)
    leaf = table.clone().requires_grad_()
    loss = lambda t: (flashback_attn_relpos_func(q, k, v, t).double() * do.double()).sum()  # noqa: E731
    g = torch.autograd.grad(loss(leaf), leaf)[0]
    h = 2.0 ** -6
    diff = (loss(table + h * way) - loss(table - h * way)) / (2 * h)
    want = (g.double() * way.double()).sum()
    assert abs(diff - want) <= 1e-2 * abs(want) + 1e-3 * (g.double() * way.double()).abs().sum()


def test_gradients_asked_for_one_by_one():
    q, k, v, table, do = (_mk(s, BF16, i) for i, s in enumerate([(1, 140, 2, 64), (1, 150, 2, 64), (1, 150, 2, 64), (32, 2), (1, 140, 2, 64)]))
    every = [t.clone().requires_grad_() for t in (q, k, v, table)]
    want = torch.autograd.grad(flashback_attn_relpos_func(*every), every, do)
    for n in range(4):
        some = [t.clone().requires_grad_(i == n) for i, t in enumerate((q, k, v, table))]
        got = torch.autograd.grad(flashback_attn_relpos_func(*some), some[n], do)[0]
        assert torch.equal(got, want[n])


def test_deterministic_and_second_order_refused():
    leaves = [_mk(s, BF16, i).requires_grad_() for i, s in enumerate([(2, 300, 4, 64), (2, 300, 1, 64), (2, 300, 1, 64), (32, 4)])]
    do = _mk((2, 300, 4, 64), BF16, 8)
    runs = [torch.autograd.grad(flashback_attn_relpos_func(*leaves, causal=True), leaves, do) for _ in range(3)]
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, runs[0]))
    g = torch.autograd.grad(flashback_attn_relpos_func(*leaves), leaves, do.requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g[0].float().sum(), leaves[0])


def test_empty():
    table = _mk((32, 2), BF16, 0).requires_grad_()
    q, k = _mk((1, 5, 2, 64), BF16, 1).requires_grad_(), _mk((1, 0, 2, 64), BF16, 2)
    out = flashback_attn_relpos_func(q, k, k, table)
    assert torch.equal(out, torch.zeros_like(out))
    assert all(torch.equal(g, torch.zeros_like(g)) for g in torch.autograd.grad(out, (q, table), torch.ones_like(out)))
    out = flashback_attn_relpos_func(q[:, :0], _mk((1, 3, 2, 64), BF16, 2), _mk((1, 3, 2, 64), BF16, 2), table)
    assert out.shape == (1, 0, 2, 64)


def test_rows_behind_the_last_sequence_stay():
    """Packed tensors longer than the sequences say: the rows behind the last one are not touched."""
    cu = torch.tensor([0, 70, 150], dtype=torch.int32, device=DEV)
    q, out = _mk((200, 2, 64), BF16, 0), torch.full((200, 2, 64), 7.0, dtype=BF16, device=DEV)
    k, table = _mk((200, 2, 64), BF16, 1), _mk((32, 2), BF16, 2)
    from flashback_cute import relpos

    import ctypes

    prob = _lib.problem(q, k, cu, cu, 80, 80, 0.125, True)
    lse = torch.full((2, 200), 7.0, device=DEV)
    bias = relpos._bias(table.shape, table.stride(), False, 128)
    bias.table = table.data_ptr()
    a = _lib.FbRelposFwdArgs(prob, bias, *(_lib.seq_tensor(t) for t in (q, k, k, out)), _lib.seq_tensor(None), lse.data_ptr())
    assert _lib.load().fb_relpos_fwd(ctypes.byref(a), torch.cuda.current_stream().cuda_stream) == 0
    assert (out[150:] == 7.0).all() and (lse[:, 150:] == 7.0).all()
    ref = orc.attention(q[:150], k[:150], k[:150], table, 128, False, 0.125, True, None, [70, 80], [70, 80])
    _within("out", out[:150], ref.out, ref.tol[0])


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_behind_the_last_sequence_may_hold_anything(dtype):
    """Packed tensors with NaN behind the last sequence: neither the outputs nor any gradient of the sequences' rows sees it."""
    for causal, lens in ((True, [70, 80, 101]), (False, [64, 1, 130])):
        total = sum(lens)
        cu = torch.tensor([0, *itertools.accumulate(lens)], dtype=torch.int32, device=DEV)
        full = [_mk((total + 40, h, 64), dtype, i) for i, h in enumerate((4, 2, 2, 4))]
        for t in full:
            t[total:] = float("nan")
        table = _mk((32, 4), dtype, 9)
        leaves = [t.requires_grad_() for t in (*full[:3], table)]
        out = flashback_attn_relpos_varlen_func(*leaves, cu, cu, max(lens), max(lens), causal=causal)
        grads = torch.autograd.grad(out, leaves, full[3])
        q, k, v, do = (t.detach()[:total] for t in full)
        ref = orc.attention(q, k, v, table, 128, not causal, 0.125, causal, do, lens, lens)
        for name, got, want, tol in zip(("out", "dq", "dk", "dv", "dtable"), (out.detach(), *grads), ref[:5], ref.tol):
            _within(name, got[:want.shape[0]], want, tol)


@pytest.mark.parametrize("dtype,d", [(BF16, 128), (F16, 64)])
def test_every_streamed_block_is_a_tail(dtype, d):
    """Short queries under many heads: the dK/dV kernel meets the end of the sequence in every block it streams."""
    for hq, sq, sk, causal in ((8, 52, 15, True), (16, 1, 200, False), (12, 33, 70, True), (16, 63, 300, False)):
        for seed in range(3):
            _check(dtype, d, hq, 1, causal, 2, sq, sk, 64, 91, False, seed)
    _check(dtype, d, 8, 1, True, None, None, None, packed=([5, 60, 1, 33, 100], [5, 60, 1, 33, 100]))


def test_a_broken_sequence_leaves_the_others_alone():
    """NaN in one sequence of a packed batch: the sequences before and behind it are what they are without it."""
    lens = [100, 70, 90]
    cu = torch.tensor([0, *itertools.accumulate(lens)], dtype=torch.int32, device=DEV)
    good = [_mk((260, 2, 64), BF16, i) for i in range(4)]
    table, res = _mk((32, 2), BF16, 9), []
    for broken in (False, True):
        q, k, v, do = (t.clone() for t in good)
        if broken:
            for t in (q, k, v, do):
                t[100:170] = float("nan")
        leaves = [t.requires_grad_() for t in (q, k, v)]
        out = flashback_attn_relpos_varlen_func(*leaves, table, cu, cu, 100, 100, causal=True)
        res.append((out.detach(), *torch.autograd.grad(out, leaves, do)))
    for a, b in zip(*res):
        assert torch.equal(a[:100], b[:100]) and torch.equal(a[170:], b[170:])


def _step(seed, d=64, s=300, causal=True):
    from flashback_cute import flashback_attn_relpos_decode

    leaves = [_mk(x, BF16, seed + i).requires_grad_() for i, x in enumerate([(2, s, 4, d), (2, s, 2, d), (2, s, 2, d), (32, 4)])]
    out = flashback_attn_relpos_func(*leaves, causal=causal)
    grads = torch.autograd.grad(out, leaves, _mk((2, s, 4, d), BF16, seed + 5))
    lens = torch.tensor([s, 17], dtype=torch.int32, device=DEV)
    q, k, v, table = (t.detach() for t in leaves)
    one = flashback_attn_relpos_decode(q[:, -1:], k, v, lens, table)
    long_k = _mk((1, 20000, 2, d), BF16, seed + 6)
    many = flashback_attn_relpos_decode(q[:1, -1:], long_k, long_k, None, table)
    bias = flashback_relpos_bias(leaves[3], 200, 333)
    return [out.detach(), *grads, one, many, bias.detach(), torch.autograd.grad(bias, leaves[3], _mk((4, 200, 333), BF16, seed + 7))[0]]


def test_several_streams_at_once():
    """The same work on four streams at once (CTAs of different kernels and calls share the SMs), against one after the other."""
    want = [_step(10 * i, 128 if i % 2 else 64, 300 + 50 * i, i < 2) for i in range(4)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    for _ in range(3):
        got = [None] * 4
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = _step(10 * i, 128 if i % 2 else 64, 300 + 50 * i, i < 2)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_workspaces_may_hold_anything():
    """Outputs and workspaces come from memory full of NaN: nothing is read before it is written, nothing is left unwritten."""
    want = _step(3)
    for _ in range(2):
        torch.cuda.synchronize()
        poison = [torch.full((n,), float("nan"), device=DEV) for n in (1 << 24, 1 << 20, 1 << 18, 1 << 16, 1 << 14, 1 << 12, 128, 64)]
        poison += [torch.full((n,), float("nan"), device=DEV) for n in (1 << 20, 1 << 18, 1 << 16, 1 << 14, 1 << 12, 128, 64) for _ in range(8)]
        del poison
        assert all(torch.equal(a, b) for a, b in zip(_step(3), want))


def test_several_threads_at_once():
    """Calls from several host threads: plans, argument templates and the library's look-ups are shared between them."""
    import concurrent.futures

    want = [_step(7 * i, s=180 + i) for i in range(4)]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            got = [_step(7 * i, s=180 + i) for _ in range(3)]
            torch.cuda.current_stream().synchronize()
        return got

    with concurrent.futures.ThreadPoolExecutor(4) as pool:
        for i, runs in enumerate(pool.map(work, range(4))):
            for r in runs:
                assert all(torch.equal(a, b) for a, b in zip(r, want[i]))


def test_two_captured_graphs():
    """Two graphs over the same buffers, replayed in turn and with eager calls between: each has workspaces of its own."""
    bufs = [_mk(x, BF16, i) for i, x in enumerate([(2, 150, 4, 64), (2, 150, 2, 64), (2, 150, 2, 64), (32, 4), (2, 150, 4, 64)])]

    def step(causal):
        leaves = [t.detach().requires_grad_() for t in bufs[:4]]
        out = flashback_attn_relpos_func(*leaves, causal=causal)
        return (out.detach(), *torch.autograd.grad(out, leaves, bufs[4]))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(True), step(False)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for causal in (True, False):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append(step(causal))
        graphs.append(g)
    for round_ in range(3):
        for i in range(5):
            bufs[i].copy_(_mk(bufs[i].shape, BF16, 40 * round_ + i))
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        for got, causal in zip(outs, (True, False)):
            assert all(torch.equal(a, b) for a, b in zip(got, step(causal)))


def test_under_torch_func():
    shapes = [(1, 70, 2, 64), (1, 70, 2, 64), (1, 70, 2, 64), (32, 2)]
    x = [_mk(s, BF16, i) for i, s in enumerate(shapes)]
    got = torch.func.grad(lambda *a: flashback_attn_relpos_func(*a).float().sum(), argnums=(0, 1, 2, 3))(*x)
    leaves = [t.clone().requires_grad_() for t in x]
    want = torch.autograd.grad(flashback_attn_relpos_func(*leaves).float().sum(), leaves)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with pytest.raises(RuntimeError):  # no forward mode
        torch.func.jvp(lambda t: flashback_attn_relpos_func(*x[:3], t), (x[3],), (x[3],))


def test_captured_and_replayed_on_a_side_stream():
    """Forward and backward captured into one graph, replayed with new inputs in the same buffers; equal to an eager run."""
    shapes = [(2, 257, 4, 64), (2, 257, 2, 64), (2, 257, 2, 64), (32, 4), (2, 257, 4, 64)]
    bufs = [_mk(s, BF16, i) for i, s in enumerate(shapes)]

    def step():
        leaves = [t.detach().requires_grad_() for t in bufs[:4]]
        out = flashback_attn_relpos_func(*leaves, causal=True)
        return (out.detach(), *torch.autograd.grad(out, leaves, bufs[4]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = step()
    for i, s in enumerate(shapes):
        bufs[i].copy_(_mk(s, BF16, 20 + i))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, step()))


# ---------------------------------------------------------------------------------------------
# the bias as a tensor
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("sizes", [(1, 1), (1, 4099), (17, 3), (33, 2050), (130, 257), (300, 300)])
@pytest.mark.parametrize("two", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_bias_tensor_and_its_gradient(dtype, two, sizes):
    sq, sk = sizes
    for num, far, heads in ((32, 128, 3), (128, 1500, 2), (4, 7, 1)):
        table = _mk((num, heads), dtype, 0).requires_grad_()
        which = orc.buckets(sq, sk, num, far, two).to(DEV)
        bias = flashback_relpos_bias(table, sq, sk, max_distance=far, bidirectional=two)
        assert torch.equal(bias.detach(), table.detach().t()[:, which])
        grad = _mk(bias.shape, dtype, 1)
        got = torch.autograd.grad(bias, table, grad)[0]
        want, size = (torch.zeros(num, heads, dtype=torch.float64, device=DEV) for _ in range(2))
        for h in range(heads):
            want[:, h].index_add_(0, which.flatten(), grad[h].double().flatten())
            size[:, h].index_add_(0, which.flatten(), grad[h].double().abs().flatten())
        # float32 sums along a diagonal (at most 512 rows in a row), over the warps and a run of neighbours; then 64 bits; one rounding
        u = torch.finfo(dtype).eps / 2
        _within("dtable", got, want, (512 / 8 + 8 + 5 + 8) * 2.0 ** -24 * size * (1 + u) + u * want.abs())


def test_bias_tensor_views_and_derivatives():
    table = _mk((3, 32), F32, 0).t().requires_grad_()
    bias = flashback_relpos_bias(table, 40, 50)
    g = torch.autograd.grad(bias.sum(), table, create_graph=True)[0]  # a broadcast gradient
    which = orc.buckets(40, 50, 32, 128, True).to(DEV)
    assert torch.equal(g.detach(), torch.bincount(which.flatten(), minlength=32).float()[:, None].expand(-1, 3))
    w = _mk((3, 40, 50), F32, 1).requires_grad_()
    first = torch.autograd.grad((flashback_relpos_bias(table, 40, 50) * w).sum(), table, create_graph=True)[0]
    way = _mk((32, 3), F32, 2)
    second = torch.autograd.grad((first * way).sum(), w)[0]
    assert torch.equal(second, way.t()[:, which])
    _, tangent = torch.func.jvp(lambda t: flashback_relpos_bias(t, 40, 50), (table.detach(),), (way,))
    assert torch.equal(tangent, way.t()[:, which])


def test_bias_tensor_empty():
    table = _mk((32, 2), BF16, 0).requires_grad_()
    bias = flashback_relpos_bias(table, 0, 5)
    assert bias.shape == (2, 0, 5)
    assert torch.equal(torch.autograd.grad(bias.sum(), table)[0], torch.zeros_like(table))


# ---------------------------------------------------------------------------------------------
# new tokens against a cache
# ---------------------------------------------------------------------------------------------
def _decode_ref(q, k, v, lens, table, far, two, scale):
    out, tol = torch.zeros(q.shape, dtype=torch.float64, device=DEV), torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    for b, n in enumerate(lens):
        n = min(max(n, 0), k.shape[1])
        r = orc.attention(q[b:b + 1], k[b:b + 1, :n], v[b:b + 1, :n], table, far, two, scale, True)
        out[b], tol[b] = r.out[0], r.tol[0][0]
    return out, tol


def _check_decode(dtype, d, hq, hkv, sq, s, lens, num=32, far=128, two=False, seed=0):
    from flashback_cute import flashback_attn_relpos_decode

    b = len(lens)
    q, k, v = _mk((b, sq, hq, d), dtype, seed), _mk((b, s, hkv, d), dtype, seed + 1), _mk((b, s, hkv, d), dtype, seed + 2)
    table = _mk((num, hq), dtype, seed + 3)
    for i, n in enumerate(lens):  # rows that must not be read
        k[i, max(n, 0):], v[i, max(n, 0):] = float("nan"), float("nan")
    got = flashback_attn_relpos_decode(q, k, v, torch.tensor(lens, dtype=torch.int32, device=DEV), table, max_distance=far, bidirectional=two)
    want, tol = _decode_ref(q, k, v, lens, table, far, two, d ** -0.5)
    _within("out", got, want, tol)


@pytest.mark.parametrize("sq", [1, 2, 5])
@pytest.mark.parametrize("heads", [(4, 4), (8, 1), (12, 4)])
@pytest.mark.parametrize("dtype,d", [(BF16, 64), (BF16, 128), (F16, 64), (F16, 128)])
def test_decode(dtype, d, heads, sq):
    _check_decode(dtype, d, *heads, sq, 700, [700, 1, 0, 3, 16, 17, 64, 65, 511, 640, 900, -4])


@pytest.mark.parametrize("num,far,two", [(2, 2, False), (64, 2000, False), (32, 60, True), (128, 300, False)])
def test_decode_buckets(num, far, two):
    _check_decode(BF16, 128, 8, 2, 3, 2300, [2300, 100, 1555], num, far, two)


def test_decode_one_slice_and_many():
    """One slice per sequence (the kernel writes the output itself), and more slices than keys."""
    _check_decode(BF16, 64, 32, 8, 1, 300, [300 - 7 * i for i in range(40)])
    _check_decode(BF16, 64, 160, 160, 1, 90, [90 - i for i in range(16)])
    _check_decode(F16, 128, 1, 1, 1, 9001, [9001, 5])


def test_decode_many_rows():
    """More (token, head) pairs per kv head than one operand holds."""
    _check_decode(BF16, 64, 16, 1, 7, 400, [400, 3, 129])
    _check_decode(F16, 128, 40, 1, 2, 150, [150, 31])


def test_decode_agrees_with_the_prompt_path():
    """The last tokens of a prompt, computed as a prompt and token by token against a growing cache."""
    from flashback_cute import flashback_attn_relpos_decode

    q, k, v, table = _mk((2, 200, 8, 64), BF16, 0), _mk((2, 256, 2, 64), BF16, 1), _mk((2, 256, 2, 64), BF16, 2), _mk((32, 8), BF16, 3)
    whole = flashback_attn_relpos_func(q, k[:, :200].contiguous(), v[:, :200].contiguous(), table, causal=True)
    tol = orc.attention(q, k[:, :200], v[:, :200], table, 128, False, 0.125, True).tol[0]
    for t in (0, 1, 63, 64, 150, 199):
        lens = torch.full((2,), t + 1, dtype=torch.int32, device=DEV)
        one = flashback_attn_relpos_decode(q[:, t:t + 1], k, v, lens, table)
        assert ((one[:, 0].double() - whole[:, t].double()).abs() <= 2 * tol[:, t]).all()


def test_decode_views_and_no_lengths():
    """Caches as views of one tensor (keys and values side by side, heads before rows); no lengths: every row counts."""
    from flashback_cute import flashback_attn_relpos_decode

    kv = _mk((3, 2, 4, 333, 64), BF16, 1)  # (b, k or v, heads, rows, d)
    k, v = kv[:, 0].transpose(1, 2), kv[:, 1].transpose(1, 2)
    q, table = _mk((3, 8, 2, 64), BF16, 0).transpose(1, 2), _mk((8, 32), BF16, 3).t()
    got = flashback_attn_relpos_decode(q, k, v, None, table)
    want, tol = _decode_ref(q, k, v, [333] * 3, table, 128, False, 0.125)
    _within("out", got, want, tol)
    with pytest.raises(ValueError):
        flashback_attn_relpos_decode(q, k.transpose(2, 3).contiguous().transpose(2, 3), v, None, table)
    with pytest.raises(TypeError):
        flashback_attn_relpos_decode(q.float(), k.float(), v.float(), None, table.float())
    with pytest.raises(TypeError):
        flashback_attn_relpos_decode(q, k, v, torch.zeros(3, dtype=torch.int64, device=DEV), table)
    with pytest.raises(ValueError):
        flashback_attn_relpos_decode(q, k, v, torch.zeros(2, dtype=torch.int32, device=DEV), table)


def test_decode_captured_with_growing_lengths():
    """One graph, replayed while the lengths grow: a generation loop."""
    from flashback_cute import flashback_attn_relpos_decode

    q, k, v, table = _mk((4, 1, 8, 128), BF16, 0), _mk((4, 512, 2, 128), BF16, 1), _mk((4, 512, 2, 128), BF16, 2), _mk((32, 8), BF16, 3)
    lens = torch.full((4,), 300, dtype=torch.int32, device=DEV)
    flashback_attn_relpos_decode(q, k, v, lens, table)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = flashback_attn_relpos_decode(q, k, v, lens, table)
    for _ in range(3):
        lens += 37
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, flashback_attn_relpos_decode(q, k, v, lens, table))


def test_decode_empty():
    from flashback_cute import flashback_attn_relpos_decode

    q, k, table = _mk((2, 1, 4, 64), BF16, 0), _mk((2, 0, 4, 64), BF16, 1), _mk((32, 4), BF16, 3)
    assert torch.equal(flashback_attn_relpos_decode(q, k, k, None, table), torch.zeros_like(q))
    assert flashback_attn_relpos_decode(q[:0], _mk((0, 5, 4, 64), BF16, 1), _mk((0, 5, 4, 64), BF16, 1), None, table).shape == (0, 1, 4, 64)


# ---------------------------------------------------------------------------------------------
# offsets that pass 32 bits, long rows
# ---------------------------------------------------------------------------------------------
def test_decode_offsets_beyond_32_bits():
    """A cache of more than 2^31 elements; the last kv head of the last rows against the oracle's formula."""
    from flashback_cute import flashback_attn_relpos_decode

    s, hkv, d = 1_060_000, 16, 128
    assert s * hkv * d > 2 ** 31
    k, v = (torch.empty(1, s, hkv, d, dtype=BF16, device=DEV).normal_() for _ in range(2))
    q, table = _mk((1, 1, hkv, d), BF16, 0), _mk((32, hkv), BF16, 1)
    got = flashback_attn_relpos_decode(q, k, v, None, table)
    which = torch.full((1, s), 31, device=DEV)
    which[0, -200:] = orc.buckets(1, 200, 32, 128, False)[0].to(DEV)
    for h in (0, hkv - 1):
        w = lambda t: t[0, :, h].double()  # noqa: E731
        r = orc.head(w(q), w(k), w(v), table[:, h].double(), which, d ** -0.5, True, 2.0 ** -8)
        _within("out", got[0, :, h], r.out, r.tol_out)


def test_bias_tensor_offsets_beyond_32_bits():
    n, heads = 16_411, 8
    assert n * n * heads > 2 ** 31
    table = _mk((32, heads), BF16, 0).requires_grad_()
    bias = flashback_relpos_bias(table, n, n, bidirectional=False)
    row = orc.buckets(1, n, 32, 128, False)[0].to(DEV)  # the last query's
    assert torch.equal(bias[heads - 1, -1].detach(), table.detach()[:, heads - 1][row])
    grad = torch.zeros_like(bias)
    grad[heads - 1, -1] = 1
    got = torch.autograd.grad(bias, table, grad)[0]
    want = torch.zeros(32, heads, device=DEV)
    want[:, heads - 1] = torch.bincount(row, minlength=32).float()
    assert torch.equal(got, want.to(BF16))


def test_long_sequence():
    """32768 keys: the last 256 queries' outputs and gradients, and the last keys' (no earlier query sees them)."""
    s, n = 32768, 256
    q, k, v, do = (_mk((1, s, 1, 64), BF16, i) for i in range(4))
    do[:, :-n] = 0  # then only these queries have gradients
    leaves = [t.requires_grad_() for t in (q, k, v, _mk((32, 1), BF16, 7))]
    out = flashback_attn_relpos_func(*leaves, causal=True)
    grads = torch.autograd.grad(out, leaves, do)
    which = torch.full((n, s), 31, device=DEV)
    which[:, -n - 200:] = orc.buckets(n, n + 200, 32, 128, False).to(DEV)
    w = lambda t, m=s: t.detach()[0, -m:, 0].double()  # noqa: E731
    r = orc.head(w(q, n), w(k), w(v), leaves[3].detach()[:, 0].double(), which, 0.125, True, 2.0 ** -8, w(do, n))
    _within("out", out.detach()[0, -n:, 0], r.out, r.tol_out)
    for name, got, want, tol in (("dq", grads[0][0, -n:, 0], r.dq, r.tol_dq), ("dk", grads[1][0, :, 0], r.dk, r.tol_dk), ("dv", grads[2][0, :, 0], r.dv, r.tol_dv),
                                 ("dtable", grads[3][:, 0], r.dt, r.tol_dt + 2.0 ** -8 * (r.dt.abs() + r.tol_dt))):
        _within(name, got, want, tol)


def test_decode_queries_at_any_address():
    """Queries 8 bytes off an aligned address: slices of wider heads, of a fused buffer, transposed, one for all."""
    from flashback_cute import flashback_attn_relpos_decode
    from tests.test_relpos_host import odd_queries

    for q in odd_queries().values():
        flat = q.as_strided((q.untyped_storage().nbytes() // 2,), (1,), 0).to(DEV)
        q = flat.as_strided(q.shape, q.stride(), q.storage_offset())
        assert q.data_ptr() % 16 == 8
        k, v, table = _mk((q.shape[0], 90, 4, 64), BF16, 1), _mk((q.shape[0], 90, 4, 64), BF16, 2), _mk((32, 8), BF16, 3)
        lens = [90, 31, 2][:q.shape[0]]
        got = flashback_attn_relpos_decode(q, k, v, torch.tensor(lens, dtype=torch.int32, device=DEV), table)
        want, tol = _decode_ref(q, k, v, lens, table, 128, False, 0.125)
        _within("out", got, want, tol)


def test_empty_sequences_in_batches():
    """Two dense sequences of length zero: queries, keys, both."""
    for sq, sk in ((0, 5), (5, 0), (0, 0)):
        leaves = [t.requires_grad_() for t in (_mk((2, sq, 4, 64), BF16, 0), _mk((2, sk, 2, 64), BF16, 1), _mk((2, sk, 2, 64), BF16, 2), _mk((32, 4), BF16, 3))]
        out = flashback_attn_relpos_func(*leaves)
        assert out.shape == (2, sq, 4, 64) and (out == 0).all()
        assert all((g == 0).all() for g in torch.autograd.grad(out, leaves, torch.ones_like(out)))


def test_misaligned_inputs_under_torch_func():
    off = lambda shape, seed: torch.cat([_mk((4,), BF16, 0), _mk(shape, BF16, seed).flatten()])[4:].view(shape)  # noqa: E731
    x = (off((2, 50, 4, 64), 0), off((2, 60, 2, 64), 1), off((2, 60, 2, 64), 2), _mk((32, 4), BF16, 3))
    assert x[0].data_ptr() % 16 == 8
    got = torch.func.grad(lambda *a: flashback_attn_relpos_func(*a).float().sum(), argnums=(0, 1, 2, 3))(*x)
    leaves = [t.clone().requires_grad_() for t in x]
    want = torch.autograd.grad(flashback_attn_relpos_func(*leaves).float().sum(), leaves)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_bias_tensor_of_a_broadcast_table():
    column, way = _mk((32, 1), F32, 0), _mk((32, 1), F32, 1)
    which = orc.buckets(40, 50, 32, 128, True).to(DEV)
    _, tangent = torch.func.jvp(lambda c: flashback_relpos_bias(c.expand(-1, 3), 40, 50), (column,), (way,))
    assert torch.equal(tangent, way.expand(-1, 3).t()[:, which])
    leaf, w, spread = column.expand(-1, 3).detach().requires_grad_(), _mk((3, 40, 50), F32, 2).requires_grad_(), _mk((32, 3), F32, 3)
    first = torch.autograd.grad((flashback_relpos_bias(leaf, 40, 50) * w).sum(), leaf, create_graph=True)[0]
    assert torch.equal(torch.autograd.grad((first * spread).sum(), w)[0], spread.t()[:, which])


def test_decode_long_caches_of_mid_sized_batches():
    """148 to 295 (sequence, kv head) pairs and caches beyond 8192 rows; most sequences short."""
    for b, hkv, s, long in ((24, 8, 8200, 8200), (37, 4, 9001, 3000), (40, 7, 16500, 5000)):
        _check_decode(BF16, 64, hkv, hkv, 1, s, [long] + [1 + 37 * i % 301 for i in range(b - 1)])


@pytest.mark.parametrize("d", [64, 128])
def test_decode_keys_of_later_tokens_may_hold_anything(d):
    """Infinities and NaN in the key of a drafted token: the tokens before it do not see it."""
    from flashback_cute import flashback_attn_relpos_decode

    q, k, v, table = _mk((2, 4, 8, d), BF16, 0), _mk((2, 300, 2, d), BF16, 1), _mk((2, 300, 2, d), BF16, 2), _mk((32, 8), BF16, 3)
    lens = [300, 77]
    want, tol = _decode_ref(q, k, v, lens, table, 128, False, d ** -0.5)
    for bad in (float("nan"), float("inf"), -float("inf")):
        broken = k.clone()
        for i, n in enumerate(lens):
            broken[i, n - 2:n] = bad  # the keys of tokens 2 and 3
        got = flashback_attn_relpos_decode(q, broken, v, torch.tensor(lens, dtype=torch.int32, device=DEV), table)
        _within("out", got[:, :2], want[:, :2], tol[:, :2])


# ---------------------------------------------------------------------------------------------
# very large entries
# ---------------------------------------------------------------------------------------------
LARGE = {BF16: (1e3, 1e5, -1e9, -1.2e30, 3e38), F16: (3e3, -6e4, 65504.0), F32: (1e5 + 0.3, -1e9, -1.2e30, 3.3e38)}


def _results(dtype, d, hq, hkv, causal, sq, sk, table, two, packed=None):
    if packed:
        q, k, v, do = (_mk((sum(n), h, d), dtype, i) for i, (n, h) in enumerate(zip((packed, packed, packed, packed), (hq, hkv, hkv, hq))))
        cu = torch.tensor([0, *itertools.accumulate(packed)], dtype=torch.int32, device=DEV)
        call = lambda *a: flashback_attn_relpos_varlen_func(*a, cu, cu, max(packed), max(packed), causal=causal, bidirectional=two)  # noqa: E731
    else:
        q, k, v, do = (_mk((2, s, h, d), dtype, i) for i, (s, h) in enumerate(((sq, hq), (sk, hkv), (sk, hkv), (sq, hq))))
        call = lambda *a: flashback_attn_relpos_func(*a, causal=causal, bidirectional=two)  # noqa: E731
    leaves = [t.requires_grad_() for t in (q, k, v, table.clone())]
    out = call(*leaves)
    return (q, k, v, do), (out.detach(), *torch.autograd.grad(out, leaves, do))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_a_constant_table_is_no_bias(dtype, d):
    """Softmax does not see a constant: the same bits as without a bias, however large the constant."""
    for causal, two, sq, sk, packed in ((True, False, 150, 211, None), (False, True, 211, 150, None), (False, False, 90, 300, None), (True, False, 0, 0, [70, 1, 130])):
        zero = torch.zeros(32, 4, dtype=dtype, device=DEV)
        want = _results(dtype, d, 4, 2, causal, sq, sk, zero, two, packed)[1]
        for c in LARGE[dtype]:
            got = _results(dtype, d, 4, 2, causal, sq, sk, zero + torch.tensor(c, dtype=dtype), two, packed)[1]
            assert all(torch.equal(a, b) for a, b in zip(got, want)), c


def large_tables(dtype, num, heads):
    """Entries that hide softly, that only some rows' keys have, that no key has, and a mixture of all sizes."""
    big = 6e4 if dtype == F16 else 1e6
    first, near, last, mixed = (_mk((num, heads), dtype, 20 + i) for i in range(4))
    first[0] = -big                       # the query's own position: the first causal row sees nothing else
    near[num // 2 + 1] = big              # r = 1: rows far ahead of the first key do not see it
    near[num - 1] = -big
    last[num // 2 - 1], last[num - 1] = big, -0.5 * big
    sizes = torch.tensor([0.0, 1.0, -1.0, big, -big, 0.1 * big, -0.1 * big, 0.01 * big], device=DEV)
    mixed = (mixed.float() + sizes[torch.randint(8, mixed.shape, generator=torch.Generator(device=DEV).manual_seed(5), device=DEV)]).clamp(-65504, 65504 if dtype == F16 else 1e7).to(dtype)
    return [first, near, last, mixed]


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_large_entries(dtype, d):
    """Rows whose keys all have entries of about the same size, whatever it is: bounds that do not grow with it."""
    for which in range(4):
        for causal, two, sq, sk in ((True, False, 150, 150), (True, True, 70, 200), (False, True, 200, 70), (False, True, 130, 260), (False, False, 120, 90)):
            table = large_tables(dtype, 32, 4)[which]
            (q, k, v, do), got = _results(dtype, d, 4, 2, causal, sq, sk, table, two)
            ref = orc.attention(q, k, v, table, 128, two, d ** -0.5, causal, do, apart=True)
            for name, a, b, tol in zip(("out", "dq", "dk", "dv", "dtable"), got, ref[:5], ref.tol):
                _within(f"{name} table {which} causal {causal} two {two} {sq} x {sk}", a, b, tol)


def test_the_first_row_under_a_large_own_entry():
    """It sees one key: P = 1, O = V, and dV has all of dO."""
    for dtype in (BF16, F16, F32):
        for c in LARGE[dtype]:
            table = torch.zeros(32, 4, dtype=dtype, device=DEV)
            table[0] = c
            (q, k, v, do), (out, dq, dk, dv, dt) = _results(dtype, 64, 4, 4, True, 1, 1, table, False)
            assert torch.equal(out, v.detach()) and torch.equal(dv, do)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_decode_large_entries(dtype):
    from flashback_cute import flashback_attn_relpos_decode

    q, k, v, lens = _mk((3, 3, 8, 64), dtype, 0), _mk((3, 9000, 2, 64), dtype, 1), _mk((3, 9000, 2, 64), dtype, 2), [9000, 2, 140]
    on = torch.tensor(lens, dtype=torch.int32, device=DEV)
    want = flashback_attn_relpos_decode(q, k, v, on, torch.zeros(32, 8, dtype=dtype, device=DEV))
    for c in LARGE[dtype]:
        assert torch.equal(flashback_attn_relpos_decode(q, k, v, on, torch.full((32, 8), c, dtype=dtype, device=DEV)), want), c
    for table in large_tables(dtype, 32, 8):
        got = flashback_attn_relpos_decode(q[1:], k[1:], v[1:], on[1:], table)
        for i, n in enumerate(lens[1:]):
            r = orc.attention(q[1 + i:2 + i], k[1 + i:2 + i, :n], v[1 + i:2 + i, :n], table, 128, False, 0.125, True, apart=True)
            _within("out", got[i:i + 1], r.out, r.tol[0])


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_rows_of_no_sequence_get_zeros(dtype):
    """Packed tensors with rows before the first sequence and behind the last: results and gradients there are zeros, whatever the memory held."""
    def poison():
        torch.cuda.synchronize()
        hold = [torch.full((n,), float("nan"), device=DEV) for n in (1 << 24, 1 << 20, 1 << 18, 1 << 16, 1 << 14) for _ in range(6)]
        del hold

    for lead, lens, rest, causal in ((0, [70, 1, 130], 41, True), (37, [20], 3000, False), (5, [0, 129, 0], 300, True), (9, [0, 0], 20, False)):
        total = lead + sum(lens) + rest
        cu = torch.tensor([lead, *(lead + n for n in itertools.accumulate(lens))], dtype=torch.int32, device=DEV)
        full = [_mk((total, h, 64), dtype, i) for i, h in enumerate((4, 2, 2, 4))]
        inside = slice(lead, lead + sum(lens))
        for t in full:
            t[:lead], t[inside.stop:] = float("nan"), float("nan")
        leaves = [t.requires_grad_() for t in (*full[:3], _mk((32, 4), dtype, 9))]
        poison()
        out = flashback_attn_relpos_varlen_func(*leaves, cu, cu, max(lens), max(lens), causal=causal)
        poison()
        grads = torch.autograd.grad(out, leaves, full[3])
        for t in (out, *grads[:3]):
            assert (t[:lead] == 0).all() and (t[inside.stop:] == 0).all()
        q, k, v, do = (t.detach()[inside] for t in full)
        ref = orc.attention(q, k, v, leaves[3].detach(), 128, not causal, 0.125, causal, do, lens, lens)
        for name, got, want, tol in zip(("out", "dq", "dk", "dv", "dtable"), (out.detach(), *grads), ref[:5], ref.tol):
            _within(name, got if name == "dtable" else got[inside], want, tol)


# ---------------------------------------------------------------------------------------------
# the bias tensor at sizes whose tiles are the largest ones
# ---------------------------------------------------------------------------------------------
def _which(sq, sk, num, far, two):
    """(sq, sk) buckets on the GPU, from the oracle's bucket function by distance."""
    side = num // 2 if two else num
    dist = torch.tensor([orc.bucket(min(n, far), side, far) for n in range(max(sq, sk) + abs(sk - sq) + 1)], device=DEV)
    r = torch.arange(sk, device=DEV)[None, :] - (torch.arange(sq, device=DEV)[:, None] + sk - sq)
    return torch.where(r <= 0, dist[r.abs()], side + dist[r.abs()] if two else dist[0])


@pytest.mark.parametrize("heads,sq,sk", [(8, 1537, 2051), (16, 2047, 4099), (12, 3001, 1030)])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_bias_tensor_full_tiles(dtype, heads, sq, sk):
    """CTAs of up to 256 rows (gradient) and 128 rows (fill): every element of the bias, every entry of the table's gradient."""
    for num, far, two in ((32, 128, True), (64, 1500, False)):
        table, which = _mk((num, heads), dtype, 0).requires_grad_(), _which(sq, sk, num, far, two)
        bias = flashback_relpos_bias(table, sq, sk, max_distance=far, bidirectional=two)
        grad = _mk(bias.shape, dtype, 1)
        got = torch.autograd.grad(bias, table, grad)[0]
        want, size = (torch.zeros(num, heads, dtype=torch.float64, device=DEV) for _ in range(2))
        for h in range(heads):
            assert torch.equal(bias[h].detach(), table.detach()[:, h][which])
            want[:, h].index_add_(0, which.flatten(), grad[h].double().flatten())
            size[:, h].index_add_(0, which.flatten(), grad[h].double().abs().flatten())
        # float32 sums: 256 rows by 8 warps along a diagonal and a cut row at each end, 8 warps, a run of up to 32 neighbours (5 steps), 8 warps; then 64 bits; one rounding
        u = torch.finfo(dtype).eps / 2
        _within("dtable", got, want, (256 / 8 + 2 + 8 + 5 + 8) * 2.0 ** -24 * size * (1 + u) + u * want.abs())


@pytest.mark.parametrize("sq,sk", [(70000, 1), (20011, 3), (4099, 17), (1, 70000), (5, 30001)])
def test_bias_tensor_tall_and_wide(sq, sk):
    for dtype, two in ((BF16, True), (F32, False)):
        table, which = _mk((32, 3), dtype, 0).requires_grad_(), _which(sq, sk, 32, 128, two)
        bias = flashback_relpos_bias(table, sq, sk, bidirectional=two)
        grad = _mk(bias.shape, dtype, 1)
        got = torch.autograd.grad(bias, table, grad)[0]
        want, size = (torch.zeros(32, 3, dtype=torch.float64, device=DEV) for _ in range(2))
        for h in range(3):
            assert torch.equal(bias[h].detach(), table.detach()[:, h][which])
            want[:, h].index_add_(0, which.flatten(), grad[h].double().flatten())
            size[:, h].index_add_(0, which.flatten(), grad[h].double().abs().flatten())
        u = torch.finfo(dtype).eps / 2
        _within("dtable", got, want, (256 / 8 + 2 + 8 + 5 + 8) * 2.0 ** -24 * size * (1 + u) + u * want.abs())
