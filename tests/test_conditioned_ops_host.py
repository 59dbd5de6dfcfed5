"""Refusals of the conditioned-block operators that need no GPU: CPU tensors,
and the C entry points' checks of sizes, strides, alignment and workspaces,
which come before any CUDA call."""
import ctypes

import pytest
import torch

D = ctypes.c_void_p(1 << 20)  # 16-byte aligned stand-in pointers, never dereferenced
ODD = ctypes.c_void_p((1 << 20) + 4)
F = ctypes.c_float


def lib():
    from xgen_b200 import _lib

    return _lib.lib(), _lib.i64_array, _lib.f64_array


def test_cpu_tensors_are_refused():
    from xgen_b200.attention import cross_attention
    from xgen_b200.int8_linear import H3Int8Linear, int8_linear
    from xgen_b200.ops import quantize_per_token_int8, rope_axes, sandwich_norm

    x = torch.zeros(1, 4, 64, dtype=torch.bfloat16)
    q = torch.zeros(1, 2, 4, 64, dtype=torch.bfloat16)
    w = torch.zeros(64, 64, dtype=torch.int8)
    for call in (lambda: sandwich_norm(x, x), lambda: rope_axes(q, q, torch.zeros(2, 1), axes=(64,)), lambda: cross_attention(q, q, q),
                 lambda: int8_linear(x, w, torch.ones(64)), lambda: quantize_per_token_int8(x[0]),
                 lambda: H3Int8Linear(torch.zeros(64, 64))(x)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_rope_axes_arguments():
    h, i64, f64 = lib()
    st = i64([256, 128, 64])

    def call(q=D, dtype=0, batch=1, seq=2, heads=2, kh=2, width=64, kind=0, axes=2, channels=(32, 32), thetas=(1e4, 1e4), k=D, ko=D,
             qw=None, eps=0.0):
        return h.xgb_rope_axes(q, st, k, st, dtype, batch, seq, heads, kh, width, D, kind, 0, 2, axes, i64(channels), f64(thetas), 0,
                               qw, None, F(eps), F(0), D, ko, None)

    assert call(q=None) == -1 and call(ko=None) == -1 and call(dtype=3) == -1 and call(kind=4) == -1
    assert call(width=513) == -2 and call(heads=0) == -2 and call(axes=9) == -2 and call(axes=0) == -2
    assert call(channels=(32, 31)) == -2 and call(channels=(32, 34)) == -2 and call(channels=(0, 32)) == -2
    assert call(thetas=(1e4, -1.0)) == -1 and call(thetas=(float("nan"), 1e4)) == -1
    assert call(qw=D, eps=-1.0) == -1
    assert call(batch=0) == 0 and call(seq=0) == 0  # nothing to do


def test_sandwich_norm_arguments():
    h, i64, _ = lib()
    st = i64([256, 64])

    def call(y=D, dtype=0, batch=1, seq=2, width=64, post=1, pre=2, eps=1e-6, gate=None, ldg=0, scale=None, shift=None, ld=64, idx=None,
             rows=0, quant=0, codes=None, cs=None):
        return h.xgb_sandwich_norm(y, st, D, st, dtype, batch, seq, width, post, None, pre, None, F(eps), gate, ldg, F(1), scale, ld,
                                   shift, ld, idx, 0, rows, D, D, quant, codes, cs, None)

    assert call(y=None) == -1 and call(dtype=3) == -1 and call(post=3) == -1 and call(pre=-1) == -1 and call(eps=-1.0) == -1
    assert call(quant=1) == -1 and call(codes=D, cs=D) == -1 and call(quant=2, codes=D) == -1
    assert call(scale=D, idx=D, rows=2) == -1 and call(gate=D, ldg=64) == -1 and call(idx=D, rows=2) == -1
    assert call(gate=D, ldg=64, idx=D, rows=0) == -1
    assert call(width=16385) == -2 and call(width=0) == -2
    assert call(gate=D, ldg=63, idx=D, rows=2) == -3
    assert call(batch=0) == 0


def test_int8_arguments():
    h, _, _ = lib()

    def gemm(a=D, m=2, n=32, k=32, dtype=0, act=0, out=D, ldo=32, gate=None, ldg=32, idx=None, irows=1, rows=2, res=None, ldr=32):
        return h.xgb_int8_gemm(a, D, m, n, k, D, D, dtype, None, act, out, ldo, gate, ldg, idx, irows, rows, res, ldr, None, None)

    assert gemm(a=None) == -1 and gemm(dtype=2) == -1 and gemm(act=4) == -1
    assert gemm(k=131072) == -2 and gemm(k=24) == -2 and gemm(n=24) == -2 and gemm(m=0) == -2
    assert gemm(gate=D) == -1 and gemm(gate=D, idx=D, res=D, act=1) == -1 and gemm(gate=D, idx=D, res=D, m=3, irows=2) == -1
    assert gemm(ldo=31) == -3 and gemm(gate=D, idx=D, res=D, ldg=16) == -3
    assert gemm(a=ODD) == -4 and gemm(out=ODD) == -4
    assert h.xgb_int8_linear_workspace(D, 32, 3, 32) == 0  # one launch
    assert h.xgb_int8_linear_workspace(ODD, 32, 3, 32) == 96 + 12
    need = h.xgb_int8_linear_workspace(D, 32, 300, 32)
    assert need == 9600 + 1200

    def linear(x=D, ldx=32, m=300, k=32, ws=D, bytes_=need):
        return h.xgb_int8_linear(x, ldx, D, m, 32, k, D, 0, None, 0, D, 32, None, 0, None, 1, 0, None, 0, ws, bytes_, None, None)

    assert linear(x=None) == -1 and linear(ldx=31) == -3 and linear(k=24) == -2
    assert linear(ws=None) == -7 and linear(bytes_=need - 1) == -7 and linear(ws=ODD) == -4
    assert h.xgb_int8_quantize_per_token(None, 0, 1, 16, 16, D, D, None) == -1
    assert h.xgb_int8_quantize_per_token(D, 2, 1, 16, 16, D, D, None) == -1
    assert h.xgb_int8_quantize_per_token(D, 0, 2, 16, 8, D, D, None) == -3
    assert h.xgb_int8_quantize_per_token(D, 0, 0, 16, 16, D, D, None) == 0


def test_cross_attention_arguments():
    h, i64, _ = lib()
    qs, ks = i64([4 * 64 * 2, 64, 2 * 64, 1]), i64([8 * 64 * 2, 64, 2 * 64, 1])

    def call(q=D, qst=qs, kst=ks, dtype=0, b=2, heads=2, kvh=2, sq=4, skv=8, d=64, scale=0.1, ost=qs, ws=None, wsb=0, mask=None):
        return h.xgb_cross_attention(q, qst, D, kst, D, ks, dtype, b, heads, kvh, sq, skv, d, None, mask, 0, 1, F(scale), D, ost, ws, wsb, None,
                                     None)

    assert call(q=None) == -1 and call(dtype=2) == -1 and call(scale=0.0) == -1 and call(scale=float("nan")) == -1
    assert call(d=96) == -2 and call(heads=3) == -2 and call(sq=0) == -2 and call(skv=0) == -2 and call(b=1 << 17) == -2
    assert call(qst=i64([512, 64, 128, 2])) == -3 and call(qst=i64([512, 64, 132, 1])) == -3
    assert call(kst=i64([1024, 64, 0, 1])) == -3 and call(ost=i64([0, 64, 128, 1])) == -3 and call(qst=i64([512, 64, -128, 1])) == -3
    assert call(q=ODD) == -4
    takes = h.xgb_cross_attention_takes_mask
    assert call(sq=9, mask=D) == -2 and takes(2, 2, 8, 8) and not takes(2, 2, 9, 4096)
    assert takes(4, 2, 12, 1024) and not takes(4, 2, 12, 1023) and not takes(4, 2, 13, 1024) and not takes(3, 2, 1, 8)
    need = h.xgb_cross_attention_workspace(1, 2, 2, 1, 4096, 64)  # few rows, many keys: split
    assert need > 0
    assert call(b=1, sq=1, skv=4096) == -7 and call(b=1, sq=1, skv=4096, ws=D, wsb=need - 1) == -7
    assert h.xgb_cross_attention_workspace(1, 2, 2, 1, 64, 64) == 0 and h.xgb_cross_attention_workspace(4, 24, 24, 4096, 512, 64) == 0
    assert h.xgb_pack_keys(None, 0, 1, D, ks, D, ks, 1, 2, 8, 64, D, D, D, None) == -1
    assert h.xgb_pack_keys(D, 0, 1, D, ks, D, ks, 1, 2, 8, 96, D, D, D, None) == -2
    assert h.xgb_pack_keys(D, 0, 1, D, i64([1024, 64, 12, 1]), D, ks, 1, 2, 8, 64, D, D, D, None) == -3
    assert h.xgb_pack_keys(D, 0, 1, ODD, ks, D, ks, 1, 2, 8, 64, D, D, D, None) == -4


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_eps_of_a_norm_that_names_none(dtype):
    """torch.nn.RMSNorm(d) has eps None, for which the module takes the epsilon
    of the type that it computes in. At a deviation of 0.02 a wrong one shows."""
    from xgen_b200.ops import _norm_of

    norm = torch.nn.RMSNorm(128, dtype=dtype)
    x = (0.02 * torch.randn(64, 128, generator=torch.Generator().manual_seed(0))).to(dtype)
    _, eps = _norm_of(norm)
    ref = norm(x).double()
    y = x.double() * torch.rsqrt(x.double().pow(2).mean(-1, keepdim=True) + eps)
    # the module's result is rounded at most twice (the type, then the weight of one)
    assert ((y - ref).abs() <= (torch.finfo(dtype).eps + 2.0 ** -20) * y.abs()).all()


def test_shapes_of_a_gate_index():
    """An index is one for each token (in the tokens' shape or flat) or one for
    the trailing dimensions, repeated before them; others would be read as
    something else than they say."""
    from xgen_b200.int8_linear import _plan

    def form(shape, dtype=torch.bfloat16):
        return torch.Size(shape), torch.empty(shape, device="meta").stride(), dtype, 0

    def plan(lead, index):
        return _plan(form((*lead, 64)), torch.Size(lead), torch.bfloat16, None, form((64, 64), torch.int8), form((64,), torch.float32), None, None,
                     form((4, 64)), form(index, torch.int64), form((*lead, 64)))

    for lead, index, rows in (((3, 37), (3, 37), 111), ((3, 37), (37,), 37), ((3, 37), (1, 37), 37), ((3, 37), (111,), 111), ((5,), (5,), 5),
                              ((2, 3, 7), (3, 7), 21), ((2, 3, 7), (7,), 7), ((2, 3, 7), (1, 1, 7), 7), ((1, 9), (9,), 9), ((3, 1), (3,), 3),
                              ((3, 37), (1,), 1), ((), (), 1), ((), (1,), 1), ((3, 0), (0,), 0)):
        assert plan(lead, index)[5][1] == rows, (lead, index)
    for lead, index in (((3, 37), (3,)), ((3, 37), (3, 1)), ((3, 37), (37, 3)), ((4,), (2,)), ((2, 3, 7), (2,)), ((2, 3, 7), (2, 3)), ((2, 3, 7), (2, 3, 1)),
                        ((6, 6), (12,)), ((6, 6), (3,)), ((2, 3, 7), (2, 1, 7)), ((4,), (3,)), ((4,), (0,)), ((3, 37), (1, 1, 37, 1))):
        with pytest.raises(ValueError, match="index"):
            plan(lead, index)


def test_forward_mode_tangents_are_refused():
    """A tangent would be lost: the operators carry no derivative of either mode."""
    import torch.autograd.forward_ad as forward_ad
    from xgen_b200.attention import cross_attention
    from xgen_b200.int8_linear import int8_linear
    from xgen_b200.ops import rope_axes, sandwich_norm

    x, q = torch.zeros(1, 4, 64, dtype=torch.bfloat16), torch.zeros(1, 2, 4, 64, dtype=torch.bfloat16)
    w, pos = torch.zeros(64, 64, dtype=torch.int8), torch.zeros(2, 1)
    with forward_ad.dual_level():
        xd, qd = forward_ad.make_dual(x, x), forward_ad.make_dual(q, q)
        for call in (lambda: sandwich_norm(x, xd), lambda: rope_axes(qd, q, pos, axes=(64,)), lambda: cross_attention(q, qd, q),
                     lambda: int8_linear(xd, w, torch.ones(64))):
            with pytest.raises(ValueError, match="autograd"):
                call()
            with torch.no_grad(), pytest.raises(ValueError, match="autograd"):
                call()  # forward mode goes on under no_grad
        with pytest.raises(ValueError, match="CUDA"):
            sandwich_norm(x, x)


def test_positions_that_need_a_gradient_are_refused():
    from xgen_b200.ops import rope_axes

    q, pos = torch.zeros(1, 2, 4, 64, dtype=torch.bfloat16), torch.zeros(2, 1, requires_grad=True)
    with pytest.raises(ValueError, match="autograd"):
        rope_axes(q, q, pos, axes=(64,))
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
        rope_axes(q, q, pos, axes=(64,))
