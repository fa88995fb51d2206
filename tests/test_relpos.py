"""CPU tests of the relative position bias: the bucket function, refusals (host checks and C status codes), and the oracle itself."""

import ctypes
import math

import pytest
import torch

from flashback_cute import _lib, relpos
from oracle import relpos_oracle as orc


@pytest.mark.parametrize("side,far", [(2, 2), (3, 2), (4, 3), (16, 9), (16, 128), (32, 128), (32, 1000), (128, 65), (128, 2 ** 29)])
def test_bucket_starts_match_the_definition(side, far):
    starts = relpos.bucket_starts(side, far)
    assert len(starts) == side - 1 and list(starts) == sorted(starts) and starts[0] >= 0
    some = sorted({n for n in range(0, 300)} | {max(0, s + d) for s in starts for d in (-1, 0, 1)})
    for n in some:
        assert sum(s <= n for s in starts) == orc.bucket(min(n, far), side, far), n


def test_a_distance_on_a_border_belongs_to_the_upper_bucket():
    # 16 buckets a side, e = 8, max_distance 128: log(16/8)/log(128/8)*8 = 2 exactly, so 16 is the first of bucket 10
    assert orc.bucket(15, 16, 128) == 9 and orc.bucket(16, 16, 128) == 10
    assert sum(s <= 16 for s in relpos.bucket_starts(16, 128)) == 10


def test_buckets_agree_with_logarithms_off_the_borders():
    for n in range(1, 2000):
        x = math.log(max(n, 16) / 16) / math.log(128 / 16) * 16
        if n >= 16 and abs(x - round(x)) > 1e-9:
            assert orc.bucket(min(n, 128), 32, 128) == min(31, 16 + int(x))


@pytest.mark.parametrize("num,two,far", [(1, False, 128), (129, False, 128), (2, True, 128), (7, True, 128), (32, False, 16), (32, True, 8), (32, False, 2 ** 30)])
def test_refused_tables(num, two, far):
    with pytest.raises(ValueError):
        relpos._check_buckets(num, two, far)


def test_refused_shapes():
    t = lambda *s, **kw: torch.zeros(*s, dtype=torch.bfloat16, **kw)  # noqa: E731
    with pytest.raises(ValueError):
        relpos._check_shapes(t(2, 3, 4, 64), t(2, 3, 4, 64), t(2, 5, 4, 64), rows=False)  # k and v differ
    with pytest.raises(ValueError):
        relpos._check_shapes(t(2, 3, 4, 64), t(1, 3, 4, 64), t(1, 3, 4, 64), rows=False)  # batch
    with pytest.raises(ValueError):
        relpos._check_shapes(t(3, 4, 64), t(3, 4, 64), t(3, 4, 64), rows=False)
    with pytest.raises(ValueError):
        relpos._check_shapes(t(3, 4, 64), t(3, 4, 64), t(3, 4, 64, device="meta"), rows=True)
    with pytest.raises(ValueError):
        relpos._check_table(t(32, 3), 4, t(1))
    with pytest.raises(ValueError):
        relpos._check_table(t(32), 4, t(1))
    with pytest.raises(TypeError):
        relpos._check_table(torch.zeros(32, 4), 4, t(1))
    with pytest.raises(ValueError):
        relpos._check_table(t(32, 4, device="meta"), 4, t(1))
    with pytest.raises(NotImplementedError):
        relpos.flashback_relpos_bias(t(32, 4), 3, 3)
    with pytest.raises(NotImplementedError):
        relpos.flashback_attn_relpos_func(t(2, 3, 4, 64), t(2, 3, 4, 64), t(2, 3, 4, 64), t(32, 4))


def test_layouts_the_kernels_cannot_take():
    ok = lambda t: relpos._strides_ok(t.shape, t.stride())  # noqa: E731
    assert ok(torch.zeros(1, 8, 1, 64)) and ok(torch.zeros(8, 1, 64))
    for bad in (torch.zeros(64).expand(2, 8, 3, 64), torch.zeros(2, 8, 64, 3).transpose(2, 3),
                torch.zeros(8, 2, 1, 64).transpose(0, 1), torch.zeros(64).as_strided((1, 1, 1, 64), (1, 1, 1, 1))):
        y = relpos._plain(bad)
        assert not ok(bad) and ok(y) and torch.equal(y, bad) and y.stride() == relpos._plain_strides(tuple(bad.shape))


def test_templates_put_pointers_where_the_structures_have_them():
    for struct, words in ((_lib.FbRelposFwdArgs, relpos._FW), (_lib.FbRelposBwdArgs, relpos._BW), (_lib.FbRelposDecodeArgs, relpos._DW)):
        w = _lib.template(struct())
        for n, (name, i) in enumerate(words.items()):
            w[i] = 4096 + n
        back = struct.from_buffer_copy(w.tobytes())
        where = dict(table=lambda a: a.bias.table, cu_q=lambda a: a.prob.cu_seqlens_q, cu_k=lambda a: a.prob.cu_seqlens_k, work=lambda a: a.workspace)
        for n, name in enumerate(words):
            x = where.get(name, lambda a: getattr(a, name))(back)
            assert getattr(x, "ptr", x) == 4096 + n, name


def _prob(**kw):
    base = dict(dtype=0, batch=1, heads_q=2, heads_kv=2, head_dim=64, seqlen_q=8, seqlen_k=8, causal=0, total_q=8, total_k=8,
                softmax_scale=0.125)
    base.update(kw)
    return _lib.FbProblem(**base)


def _bias(num=4, two=0, starts=(1, 2, 5), table=0x1000):
    arr = (ctypes.c_int32 * len(starts))(*starts)
    b = _lib.FbRelpos(table, 2, 1, num, two, ctypes.addressof(arr))
    b.keep = arr
    return b


def test_status_codes():
    lib = _lib.load()
    t = _lib.FbTensor(0x1000, 128, 64)
    fwd = lambda prob=_prob(), bias=None, **kw: lib.fb_relpos_fwd(  # noqa: E731
        ctypes.byref(_lib.FbRelposFwdArgs(prob=prob, bias=bias or _bias(), **{**dict(q=t, k=t, v=t, out=t, lse=0x1000), **kw})), None)
    assert lib.fb_relpos_fwd(None, None) == -1 and lib.fb_relpos_bwd(None, None) == -1
    assert lib.fb_relpos_bias(None, None) == -1 and lib.fb_relpos_bias_grad(None, None) == -1
    assert fwd(_prob(dtype=5)) == -2
    assert fwd(_prob(head_dim=96)) == -3
    assert fwd(_prob(flags=_lib.FB_FLAG_KV_OUT_F32)) == -9
    seg = _prob(causal=1, seqlen_q=256, seqlen_k=512, total_q=256, total_k=512)
    seg.seg_rows[0], seg.seg_shift[0] = 128, 64
    assert fwd(seg) == -9
    for bias in (_bias(num=1), _bias(num=129), _bias(num=2, two=1), _bias(num=7, two=1), _bias(two=2), _bias(starts=(1, 5, 2)), _bias(starts=(-1, 1, 2))):
        assert fwd(bias=bias) == -12
    assert fwd(bias=_bias(table=None)) == -1
    assert fwd(q=_lib.FbTensor(0x1008, 128, 64)) == -6
    assert fwd(out=_lib.FbTensor(None, 0, 0)) == -1
    bwd = _lib.FbRelposBwdArgs(prob=_prob(), bias=_bias(), q=t, k=t, v=t, out=t, dout=t, lse=0x1000, dtable=0x1000)
    assert lib.fb_relpos_bwd(ctypes.byref(bwd), None) == -1  # no workspace
    assert fwd(_prob(seqlen_k=0, total_k=0)) == -5
    bwd.workspace, bwd.prob = 0x1000, _prob(seqlen_k=0, total_k=0)
    assert lib.fb_relpos_bwd(ctypes.byref(bwd), None) == -5
    bwd.workspace = 0x1008
    assert lib.fb_relpos_bwd(ctypes.byref(bwd), None) == -6
    b = _lib.FbRelposBiasArgs(0, 2, 3, 4, _bias(), 0x1004)
    assert lib.fb_relpos_bias(ctypes.byref(b), None) == -6
    b = _lib.FbRelposBiasArgs(0, 2, 3, (1 << 30) + 1, _bias(), 0x1000)
    assert lib.fb_relpos_bias(ctypes.byref(b), None) == -10
    g = _lib.FbRelposBiasGradArgs(0, 2, 0, 4, _bias(table=None), 0x1000, 0x1000, 2, 1, 0x1000)
    assert lib.fb_relpos_bias_grad(ctypes.byref(g), None) == -5
    assert b"buckets" in lib.fb_status_string(-12)
    with pytest.raises(ValueError):
        _lib.raise_for_status(-12)


def test_decode_status_codes():
    lib = _lib.load()
    c = _lib.FbCache(0x1000, 1024, 128, 64)

    def args(**kw):
        base = dict(dtype=0, batch=2, heads_q=4, heads_kv=2, head_dim=64, seqlen_q=1, seqlen_k=500, softmax_scale=0.125, bias=_bias(), q=c, k=c, v=c, out=0x1000)
        base.update(kw)
        return _lib.FbRelposDecodeArgs(**base)

    code = lambda **kw: lib.fb_relpos_decode(ctypes.byref(args(**kw)), None)  # noqa: E731
    assert lib.fb_relpos_decode(None, None) == -1
    assert code(dtype=2) == -2 and code(head_dim=96) == -3 and code(heads_q=3) == -4 and code(seqlen_q=-1) == -5
    assert code(batch=70000) == -10 and code(seqlen_q=1 << 20) == -10
    assert code(heads_q=256, heads_kv=2, bias=_bias(num=100, starts=tuple(range(1, 100)))) == -10  # 128 x 100 table entries per kv head
    assert code(heads_q=40000, heads_kv=40000, seqlen_q=20) == -10
    assert code(bias=_bias(num=1)) == -12
    assert code(k=_lib.FbCache(0x1008, 1024, 128, 64)) == -6 and code(v=_lib.FbCache(0x1000, 1024, 100, 64)) == -6
    assert code(out=None) == -1 and code(out=0x1004) == -6
    assert code(seqlen_k=50000, batch=1) == -1  # more slices than a cluster holds, without a workspace
    assert lib.fb_relpos_decode_workspace_bytes(ctypes.byref(args(seqlen_k=50000, batch=1))) > 0
    assert lib.fb_relpos_decode_workspace_bytes(ctypes.byref(args(seqlen_k=40))) == 0 == lib.fb_relpos_decode_workspace_bytes(None)


def test_struct_layouts():
    lib = _lib.load()
    structs = (_lib.FbRelpos, _lib.FbRelposFwdArgs, _lib.FbRelposBwdArgs, _lib.FbRelposBiasArgs, _lib.FbRelposBiasGradArgs,
               _lib.FbCache, _lib.FbRelposDecodeArgs)
    for i, s in enumerate(structs):
        assert lib.fb_abi_sizeof(8 + i) == ctypes.sizeof(s), s.__name__


def test_workspace_bytes():
    lib = _lib.load()
    big = _prob(batch=2, heads_q=16, heads_kv=4, seqlen_q=4096, seqlen_k=4096, total_q=8192, total_k=8192)
    assert lib.fb_relpos_workspace_bytes(ctypes.byref(big), 32) == (16 * 8192 + 2 * 16 * 32 * 32) * 4
    assert lib.fb_relpos_workspace_bytes(ctypes.byref(_prob(dtype=2, seqlen_q=17, total_q=17)), 4) == (2 * 17 + 2 + 2 * 2 * 4) * 4
    assert lib.fb_relpos_workspace_bytes(None, 32) == 0 and lib.fb_relpos_workspace_bytes(ctypes.byref(big), 500) == 0
    assert lib.fb_relpos_bias_workspace_bytes(0, 2, 5, 7, 4) > 0 and lib.fb_relpos_bias_workspace_bytes(0, 2, 0, 7, 4) == 0


def test_oracle_gradients_are_the_formulas():
    """The oracle's closed form against automatic differentiation of the definition in 64 bits."""
    torch.manual_seed(0)
    q, k, v, do = torch.randn(2, 9, 4, 64), torch.randn(2, 13, 2, 64), torch.randn(2, 13, 2, 64), torch.randn(2, 9, 4, 64)
    table = torch.randn(8, 4)
    ref = orc.attention(q, k, v, table, 5, True, 0.125, True, do)
    a, b, c, t = (x.double().requires_grad_() for x in (q, k, v, table))
    which = orc.buckets(9, 13, 8, 5, True)
    s = torch.einsum("bihd,bjhd->bhij", a, b.repeat_interleave(2, 2)) * 0.125 + t[which].permute(2, 0, 1)
    s = s.masked_fill(torch.arange(13)[None, :] - torch.arange(9)[:, None] > 4, -math.inf)
    out = torch.einsum("bhij,bjhd->bihd", s.softmax(-1), c.repeat_interleave(2, 2))
    want = (out, *torch.autograd.grad(out, (a, b, c, t), do.double()))
    for x, y in zip(ref[:5], want):
        assert torch.allclose(x, y, rtol=1e-11, atol=1e-11)


def test_decode_long_caches_join_through_the_workspace():
    """Beyond 8192 cache rows the slices are joined by a second launch, never by a cluster (whose sizes are 2, 4 and 8)."""
    lib = _lib.load()
    c = _lib.FbCache(0x1000, 1024, 128, 64)

    def floats(batch, hkv, sk, d=64):
        a = _lib.FbRelposDecodeArgs(dtype=0, batch=batch, heads_q=2 * hkv, heads_kv=hkv, head_dim=d, seqlen_q=1, seqlen_k=sk, softmax_scale=0.125,
                                    bias=_bias(), q=c, k=c, v=c, out=0x1000)
        return lib.fb_relpos_decode_workspace_bytes(ctypes.byref(a)) // 4 / (batch * 2 * hkv * (d + 2))

    for batch, hkv in ((1, 1), (24, 8), (37, 4), (32, 8), (200, 1), (295, 1), (296, 1)):
        base = batch * hkv
        for sk in (8193, 16384, 32768, 1 << 20):
            assert floats(batch, hkv, sk) == min(128, -(-148 * 8 // base), -(-sk // 64)), (base, sk)  # the slices of a sequence
        for sk in (40, 1000, 8192):
            if base < 296:
                assert floats(batch, hkv, sk) == 0


def test_the_backward_wants_the_shifts():
    lib = _lib.load()
    t = _lib.FbTensor(0x1000, 128, 64)
    bwd = _lib.FbRelposBwdArgs(prob=_prob(), bias=_bias(), q=t, k=t, v=t, out=t, dout=t, lse=0x1000, dtable=0x1000, workspace=0x1000)
    assert lib.fb_relpos_bwd(ctypes.byref(bwd), None) == -1


def test_bounds_apart_from_the_entries_size():
    """The oracle's bounds for scores less the row's largest entry: those of a table without the common part, where the others grow with it."""
    torch.manual_seed(1)
    q, k, v, do = torch.randn(1, 9, 2, 64), torch.randn(1, 13, 2, 64), torch.randn(1, 13, 2, 64), torch.randn(1, 9, 2, 64)
    table = torch.randn(8, 2).bfloat16().float()
    far = lambda c, apart: orc.attention(q, k, v, table.double() + c, 5, True, 0.125, False, do, apart=apart).tol  # noqa: E731
    small, large = far(0.0, True), far(2.0 ** 24, True)
    for a, b, loose in zip(small, large, far(2.0 ** 24, False)):
        assert torch.allclose(a, b, rtol=1e-6) and (loose >= 10 * b).all()  # (buckets without a pair: 0)


def test_workspace_of_the_bias_gradient_follows_the_tensor():
    """Partial sums only for diagonals that a block of rows has: no more than a few bytes per element, however tall the tensor."""
    lib = _lib.load()
    for dtype, size in ((0, 2), (2, 4)):
        for heads in (1, 16):
            for sq, sk in ((1 << 20, 1), (1 << 20, 64), (1 << 18, 1000), (70000, 1), (4095, 4099), (1 << 15, 1 << 15)):
                n = lib.fb_relpos_bias_workspace_bytes(dtype, heads, sq, sk, 32)
                # one part of 32 float32 per 256 rows and 128 or 256 diagonals, of which 256 + sk - 1 at most; small tensors: down to 32 rows
                parts = lambda rows: -(-sq // rows) * -(-(rows + sk - 1) // (64 * 8 // size))  # noqa: E731
                assert 0 < n <= heads * parts(32) * 32 * 4, (heads, sq, sk, n)
                assert heads * sq * sk < 1 << 26 or n == heads * parts(256) * 32 * 4, (heads, sq, sk, n)
