"""int8_linear / H3Int8Linear against the exact integer product.

The codes have to equal torch's rounding of the correctly rounded quotient.
With those codes the sum is an exact integer; it and the scales' product are
rounded to 32 bits, then one fused step adds the bias: 4 * 2^-24 of
|sum s| + |bias|. GELU and SiLU have slopes below 1.2 and are evaluated within
2^-20 of their argument; the result is rounded once (half a step)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_timeouts(cuda_device):
    yield
    from xgen_b200.attention import kernel_errors

    assert kernel_errors(cuda_device) == 0


def problem(m, n, k, dtype, dev, seed=0, bias=True):
    g = torch.Generator(device=dev).manual_seed(seed)
    x = (torch.randn(m, k, generator=g, device=dev) * (0.1 + 2 * torch.rand(m, 1, generator=g, device=dev))).to(dtype)
    w = torch.randint(-127, 128, (n, k), generator=g, device=dev, dtype=torch.int8)
    ws = 1e-4 * (0.5 + torch.rand(n, generator=g, device=dev))
    return x, w, ws, (torch.randn(n, generator=g, device=dev).to(dtype) if bias else None)


def codes_of(x):
    top = x.float().abs().amax(-1)
    s = (top / torch.full_like(top, 127.0)).clamp_min(torch.finfo(torch.float32).tiny)
    return (x.float() / s[:, None]).round().clamp(-127, 127).to(torch.int8), s


def reference(q, s, w, ws, bias, activation, gated):
    """(result, bound on its error before rounding) in 64 bits."""
    acc = (q.double() @ w.double().t()) * s.double()[:, None] * ws.double()
    y = acc if bias is None else acc + bias.double()
    dy = 4 * 2.0 ** -24 * (acc.abs() + (bias.double().abs() if bias is not None else 0))
    if activation == "gelu":
        return y * torch.special.ndtr(y), 1.2 * dy + 2.0 ** -20 * y.abs()
    if activation == "gelu_tanh":
        return y / 2 * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3))), 1.2 * dy + 2.0 ** -20 * y.abs()
    if activation == "swiglu":
        g, v = y.chunk(2, -1)
        dg, dv = dy.chunk(2, -1)
        act = g * torch.sigmoid(g)
        return act * v, (1.2 * dg + 2.0 ** -20 * g.abs()) * v.abs() + dv * act.abs()
    if gated is not None:
        gate, idx, res = gated
        rows = gate.double()[idx.repeat(q.shape[0] // idx.numel())]
        return res.double() + rows * y, dy * rows.abs() + 2.0 ** -23 * (rows * y).abs() + 2.0 ** -23 * res.double().abs()
    return y, dy


def within(got, ref, slack):
    info = torch.finfo(got.dtype)
    bound = info.eps / 2 * (ref.abs() + slack) + slack + info.smallest_normal * info.eps / 2
    worst = ((got.double() - ref).abs() / bound).max().item()
    assert worst <= 1.0, worst


@pytest.mark.parametrize("rows,cols", [(1, 16), (3, 1536), (130, 5120), (5, 17), (2, 40000), (1, 131056), (300, 64), (9, 1030)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_codes_are_the_rounded_quotients(cuda_device, rows, cols, dtype):
    from xgen_b200.ops import quantize_per_token_int8

    g = torch.Generator(device=cuda_device).manual_seed(rows)
    wide = (torch.randn(rows, cols + 3, generator=g, device=cuda_device) * 3).to(dtype)
    for x in (wide[:, :cols], wide[:, :cols].contiguous(), wide[:, 1:cols + 1]):
        q, s = quantize_per_token_int8(x)
        rq, rs = codes_of(x)
        assert torch.equal(s, rs) and torch.equal(q, rq)


def test_codes_of_ties_zeros_tiny_and_not_finite(cuda_device):
    from xgen_b200.ops import quantize_per_token_int8

    x = torch.zeros(6, 256, device=cuda_device, dtype=torch.bfloat16)
    x[0, :128] = torch.arange(128, device=cuda_device) * 0.5  # ties: k + 0.5 over a scale of one
    x[0, 200] = 127.0
    x[2, 3] = 1e-38
    x[3, :4] = torch.tensor([1e-39, -1e-39, 5e-40, 0.0])
    x[4, 5] = float("nan")
    x[5, 5], x[5, 6] = float("inf"), 1.0
    q, s = quantize_per_token_int8(x)
    rq, rs = codes_of(x[:4])
    assert torch.equal(s[:4], rs) and torch.equal(q[:4], rq)
    assert torch.isnan(s[4]) and torch.isinf(s[5])


@pytest.mark.parametrize("m,n,k", [(1, 16, 16), (1, 4608, 1536), (7, 144, 96), (16, 512, 2064), (33, 1536, 1536), (128, 256, 128),
                                   (129, 272, 1040), (300, 1024, 5120), (1000, 2064, 80), (65, 16, 4096), (513, 768, 656),
                                   (4, 64, 1536), (13, 48, 1888), (32, 160, 768), (3, 96, 8192), (2, 80, 208), (24, 272, 1024), (5, 32, 4912)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("activation", [None, "gelu", "gelu_tanh", "swiglu", "gated"])
def test_matches_exact_product(cuda_device, m, n, k, dtype, activation):
    from xgen_b200.int8_linear import int8_linear

    if activation == "swiglu":
        n = 2 * n
    x, w, ws, bias = problem(m, n, k, dtype, cuda_device, seed=m + n, bias=(m + n) % 3 != 0)
    gated = None
    if activation == "gated":
        gated = (torch.randn(5, n, device=cuda_device).to(dtype), torch.randint(0, 5, (m,), device=cuda_device),
                 torch.randn(m, n, device=cuda_device).to(dtype))
    kind = None if activation == "gated" else activation
    got = int8_linear(x, w, ws, bias, activation=kind, **({} if gated is None else dict(gate=gated[0], gate_index=gated[1],
                                                                                        residual=gated[2])))
    ref, slack = reference(*codes_of(x), w, ws, bias, kind, gated)
    assert got.dtype == dtype and got.shape == ref.shape
    within(got, ref, slack)


def test_largest_sums(cuda_device):
    """131056 products of 127 * 127 and of -128 * -128 stay within the integers."""
    from xgen_b200.int8_linear import int8_linear_quantized

    k = 131056
    q = torch.full((2, k), 127, dtype=torch.int8, device=cuda_device)
    q[1] = -128
    w = torch.full((16, k), 127, dtype=torch.int8, device=cuda_device)
    w[3] = -128
    s, ws = torch.full((2,), 2.0 ** -20, device=cuda_device), torch.full((16,), 2.0 ** -10, device=cuda_device)
    got = int8_linear_quantized(q, s, w, ws)
    ref, slack = reference(q, s, w, ws, None, None, None)
    within(got, ref, slack)


def test_batched_views_and_one_index_for_the_batch(cuda_device):
    from xgen_b200.int8_linear import int8_linear

    b, s, k, n = 3, 37, 208, 160
    x, w, ws, bias = problem(b * s, n, k, torch.bfloat16, cuda_device)
    wide = torch.randn(b, s, 2 * k, device=cuda_device).bfloat16()
    idx = torch.randint(0, 4, (s,), device=cuda_device)
    table = torch.randn(4, 3 * n, device=cuda_device).bfloat16()
    gate = table[:, n:2 * n]
    res = torch.randn(b, s, 2 * n, device=cuda_device).bfloat16()[..., :n]
    for v in (wide[..., k:], wide[..., 3:3 + k], x.view(b, s, k), wide[:, :, :k].transpose(0, 1).contiguous().transpose(0, 1)):
        got = int8_linear(v, w, ws, bias, gate=gate, gate_index=idx, residual=res)
        ref, slack = reference(*codes_of(v.reshape(b * s, k)), w, ws, bias, None, (gate, idx, res.reshape(b * s, n)))
        within(got.view(b * s, n), ref, slack)
    odd = torch.randn(4, n + 3, device=cuda_device).bfloat16()[:, 1:n + 1]  # gate rows off 16 bytes
    got = int8_linear(x.view(b, s, k), w, ws, bias, gate=odd, gate_index=idx, residual=res[:1].expand(b, s, n))
    ref, slack = reference(*codes_of(x), w, ws, bias, None, (odd, idx, res[:1].expand(b, s, n).reshape(b * s, n)))
    within(got.view(b * s, n), ref, slack)


def test_index_outside_the_table(cuda_device):
    from xgen_b200.int8_linear import int8_linear

    x, w, ws, bias = problem(5, 64, 64, torch.bfloat16, cuda_device)
    gate, res = torch.randn(2, 64, device=cuda_device).bfloat16(), torch.randn(5, 64, device=cuda_device).bfloat16()
    idx = torch.tensor([0, 2, 1, -1, 1 << 40], device=cuda_device)
    got = int8_linear(x, w, ws, bias, gate=gate, gate_index=idx, residual=res)
    assert torch.isnan(got[[1, 3, 4]]).all() and torch.isfinite(got[[0, 2]]).all()


def test_rows_do_not_touch_each_other(cuda_device):
    """A token with a NaN gives a row of NaN, and no other row."""
    from xgen_b200.int8_linear import int8_linear

    x, w, ws, bias = problem(200, 320, 256, torch.float16, cuda_device)
    clean = int8_linear(x, w, ws, bias)
    x[77, 3] = float("nan")
    got = int8_linear(x, w, ws, bias)
    assert torch.isnan(got[77]).all()
    keep = torch.arange(200, device=cuda_device) != 77
    assert torch.equal(got[keep], clean[keep])
    assert torch.equal(clean[40:41], int8_linear(x[40:41], w, ws, bias))  # one token alone: the same bits


def test_module(cuda_device):
    from xgen_b200.int8_linear import H3Int8Linear
    from xgen_b200.ops import quantize_per_token_int8

    g = torch.Generator().manual_seed(3)
    weight, bias = torch.randn(256, 128, generator=g) * 0.1, torch.randn(256, generator=g)
    layer = H3Int8Linear(weight, bias, activation="swiglu").to(cuda_device)
    x = torch.randn(2, 19, 128, generator=g).to(cuda_device, torch.bfloat16)
    with torch.no_grad():
        got = layer(x)
        q, s = quantize_per_token_int8(x.view(38, 128))
        assert torch.equal(got, layer.forward_quantized(q.view(2, 19, 128), s.view(2, 19)))
        again = H3Int8Linear.from_packed(layer.weight, layer.weight_scale, layer.bias, "swiglu")
        assert torch.equal(got, again(x)) and layer.calls == 2
    assert got.shape == (2, 19, 128)
    # against the unquantised layer: both roundings are uniform within half a
    # code; of N(0,1) rows the code is max/127 ~ 3/127, rms error 3/127/sqrt(12)
    plain = torch.nn.functional.linear(x.float(), weight.to(cuda_device), bias.to(cuda_device))
    codes = H3Int8Linear.from_packed(layer.weight, layer.weight_scale, layer.bias).forward(x).float()
    rel = (codes - plain).norm() / (plain - bias.to(cuda_device)).norm()
    assert rel < 2 * math.sqrt(2) * 3.5 / 127 / math.sqrt(12)


def test_graph_replay(cuda_device):
    from xgen_b200.int8_linear import int8_linear

    x, w, ws, bias = problem(33, 320, 256, torch.bfloat16, cuda_device)
    int8_linear(x, w, ws, bias)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = int8_linear(x, w, ws, bias)
    x.copy_(torch.randn_like(x))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, int8_linear(x, w, ws, bias))


def test_refusals(cuda_device):
    from xgen_b200.int8_linear import H3Int8Linear, int8_linear, int8_linear_quantized
    from xgen_b200.ops import quantize_per_token_int8

    x, w, ws, bias = problem(4, 64, 64, torch.bfloat16, cuda_device)
    gate, idx, res = torch.ones(2, 64, device=cuda_device).bfloat16(), torch.zeros(4, dtype=torch.long, device=cuda_device), torch.ones(4, 64, device=cuda_device).bfloat16()
    for bad in (dict(activation="relu"), dict(gate=gate), dict(gate=gate, gate_index=idx, residual=res, activation="gelu"),
                dict(gate=gate, gate_index=idx[:3], residual=res), dict(gate=gate, gate_index=idx.int(), residual=res),
                dict(gate=gate.half(), gate_index=idx, residual=res), dict(gate=gate, gate_index=idx, residual=res[:2])):
        with pytest.raises(ValueError):
            int8_linear(x, w, ws, bias, **bad)
    for bad in ((x.float(), w, ws), (x[:, :48], w, ws), (x, w.float(), ws), (x, w, ws.half()), (x, w, ws[:8]), (x, w[:, :40], ws),
                (x, w[:20], ws[:20]), (x, w, ws, bias[:8]), (x, w, ws, bias.half()), (x.cpu(), w, ws)):
        with pytest.raises(ValueError):
            int8_linear(*bad)
    with pytest.raises(ValueError):
        int8_linear_quantized(x, ws[:4], w, ws)
    with pytest.raises(ValueError):
        quantize_per_token_int8(x.float())
    with pytest.raises(ValueError):
        quantize_per_token_int8(x.t())
    with pytest.raises(ValueError, match="divisible by 16"):
        H3Int8Linear(torch.randn(17, 32))
    with pytest.raises(ValueError, match="autograd"):
        int8_linear(x.clone().requires_grad_(), w, ws)
    assert int8_linear(x[:0], w, ws, bias).shape == (0, 64)


@pytest.mark.parametrize("m", [2, 130])
def test_shapes_of_the_index(cuda_device, m):
    """Every form that is taken names the same rows; one for each sample is not
    taken for one for each token."""
    from xgen_b200.int8_linear import int8_linear, int8_linear_quantized
    from xgen_b200.ops import quantize_per_token_int8

    b, s, n = 3, m, 64
    x, w, ws, bias = problem(b * s, n, 64, torch.bfloat16, cuda_device)
    gate, res = torch.randn(4, n, device=cuda_device).bfloat16(), torch.randn(b, s, n, device=cuda_device).bfloat16()
    one = torch.randint(0, 4, (s,), device=cuda_device)
    every = torch.randint(0, 4, (b, s), device=cuda_device)
    codes, scales = quantize_per_token_int8(x)

    def call(at):
        got = int8_linear(x.view(b, s, 64), w, ws, bias, gate=gate, gate_index=at, residual=res)
        again = int8_linear_quantized(codes.view(b, s, 64), scales.view(b, s), w, ws, bias, gate=gate, gate_index=at, residual=res)
        assert torch.equal(got, again)
        return got

    for forms in ((one, one[None], one.expand(b, s), one.repeat(b)), (every, every.flatten(), every.t().contiguous().t()),
                  (one[:1], one[:1, None], one[:1].expand(s), one[0])):
        first = call(forms[0])
        at = forms[0].expand(b, s).reshape(-1)
        ref, slack = reference(*codes_of(x), w, ws, bias, None, (gate, at, res.view(b * s, n)))
        within(first.view(b * s, n), ref, slack)
        assert all(torch.equal(first, call(f)) for f in forms[1:])
    for bad in (torch.arange(b, device=cuda_device), torch.arange(b, device=cuda_device)[:, None], every.t(), every[:, :, None], every[:2]):
        with pytest.raises(ValueError, match="index"):
            call(bad)
    with pytest.raises(ValueError, match="index"):
        int8_linear(x[:4], w, ws, bias, gate=gate, gate_index=one[:2], residual=res.view(b * s, n)[:4])
