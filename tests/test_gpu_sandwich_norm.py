"""sandwich_norm against its formula in 64 bits.

Tolerance: x is a rounding (half a step) of a 32-bit value that is off by a few
2^-24 of its terms; a norm multiplies by a reciprocal deviation whose relative
error, and that of the mean, is below 32 * 2^-24 (sums of at most 16384 values
in chains of at most 64, then a tree), so 2^-18 of the largest value of the
row behind it, times weight and modulation, holds a normed value."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def norm64(x, kind, weight, eps):
    """(normed, bound on its 32-bit error relative to nothing) of x [.., W]."""
    if kind is None:
        return x, x.abs() * 2.0 ** -22
    d = x - x.mean(-1, keepdim=True) if kind == "layernorm" else x
    rstd = torch.rsqrt(d.pow(2).mean(-1, keepdim=True) + eps)
    w = 1.0 if weight is None else weight.double().cpu()
    slack = 2.0 ** -18 * x.abs().amax(-1, keepdim=True) * rstd * (w.abs() if weight is not None else 1.0)
    return d * rstd * w, slack.expand_as(x)


def reference(branch, residual, a):
    at = a["indices"].cpu() if a.get("indices") is not None else None
    table = lambda name: a[name].double().cpu()[at] if a.get(name) is not None else None  # noqa: E731
    eps, rs = a.get("eps", 1e-6), a.get("residual_scale", 1.0)
    y, dy = norm64(branch.double().cpu(), a["post_norm"], a.get("post_weight"), eps)
    gate = table("gate")
    if gate is not None:
        y, dy = y * gate, dy * gate.abs()
    x = residual.double().cpu() + rs * y
    dx = abs(rs) * (dy + 2.0 ** -22 * y.abs()) + 2.0 ** -23 * residual.double().cpu().abs()
    if a["pre_norm"] is None:
        return x, dx, None, None
    h, dh = norm64(x, a["pre_norm"], a.get("pre_weight"), eps)
    # the error of x itself, through the norm: relative to the deviation
    d = x - x.mean(-1, keepdim=True) if a["pre_norm"] == "layernorm" else x
    rstd = torch.rsqrt(d.pow(2).mean(-1, keepdim=True) + eps)
    w = a["pre_weight"].double().cpu().abs() if a.get("pre_weight") is not None else 1.0
    dh = dh + 4 * dx.amax(-1, keepdim=True) * rstd * w * (1 + (d * rstd).abs())
    scale = table("scale")
    if scale is not None:
        h, dh = h * (1 + scale) + table("shift"), dh * (1 + scale).abs() + 2.0 ** -21 * (h.abs() * (1 + scale.abs()) + table("shift").abs())
    return x, dx, h, dh


def within(got, ref, slack):
    info = torch.finfo(got.dtype)
    bound = info.eps / 2 * (ref.abs() + slack) + slack + info.smallest_normal * info.eps / 2
    worst = ((got.double().cpu() - ref).abs() / bound).max().item()
    assert worst <= 1.0, worst


def arguments(w, rows, dtype, dev, g, post, pre, seq, *, weights=True, gate=True, modulate=True, batched=None):
    table = (0.4 * torch.randn(rows, 3 * w, generator=g)).to(dev, dtype)
    a = {"post_norm": post, "pre_norm": pre, "residual_scale": 0.7}
    if weights and post:
        a["post_weight"] = (1 + 0.2 * torch.randn(w, generator=g)).to(dev, dtype)
    if weights and pre:
        a["pre_weight"] = (1 + 0.2 * torch.randn(w, generator=g)).to(dev, dtype)
    if gate:
        a["gate"] = table[:, :w]
    if modulate and pre:
        a["scale"], a["shift"] = table[:, w:2 * w], table[:, 2 * w:]
    if gate or (modulate and pre):
        a["indices"] = torch.randint(0, rows, (seq,) if batched is None else (batched, seq), generator=g).to(dev)
    return a


@pytest.mark.parametrize("b,s,w", [(1, 1, 1), (1, 3, 8), (2, 5, 33), (1, 7, 1536), (2, 33, 257), (1, 4, 5120), (3, 2, 2048),
                                   (1, 2, 16384), (1, 3, 9999), (1, 130, 64), (1, 5, 8192), (2, 3, 776),
                                   (1, 300, 1536), (3, 101, 2040), (1, 297, 5120), (2, 150, 512), (1, 9, 400), (1, 299, 8184)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("post,pre", [("rmsnorm", "layernorm"), ("layernorm", "rmsnorm"), (None, "rmsnorm"), ("rmsnorm", None)])
def test_matches_formula(cuda_device, b, s, w, dtype, post, pre):
    from xgen_b200.ops import sandwich_norm

    g = torch.Generator().manual_seed(w + s)
    y = (0.8 * torch.randn(b, s, w, generator=g) + 0.3).to(cuda_device, dtype)
    x = (2 * torch.randn(b, s, w, generator=g) - 0.5).to(cuda_device, dtype)
    for plain in (False, True):
        a = arguments(w, 5, dtype, cuda_device, g, post, pre, s, weights=not plain, gate=not plain, modulate=not plain,
                      batched=b if s % 2 else None)
        got = sandwich_norm(y, x, **a)
        rx, dx, rh, dh = reference(y, x, a)
        if pre is None:
            within(got, rx, dx)
        else:
            within(got[0], rx, dx)
            within(got[1], rh, dh)


@pytest.mark.parametrize("w", [16, 129, 1536, 5120, 10000])
@pytest.mark.parametrize("quant", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_codes(cuda_device, w, quant, dtype):
    """Scales are the row's largest magnitude over 127 or 448; a code is the
    nearest one to h / s: off by half a step (int8 1/2, e4m3 2^-4 relative or
    2^-10 below its normal range), and the error of h."""
    from xgen_b200.ops import sandwich_norm

    g = torch.Generator().manual_seed(w)
    y = torch.randn(2, 9, w, generator=g).to(cuda_device, dtype)
    x = (2 * torch.randn(2, 9, w, generator=g)).to(cuda_device, dtype)
    a = arguments(w, 3, dtype, cuda_device, g, "rmsnorm", "rmsnorm", 9)
    got_x, codes, scales = sandwich_norm(y, x, quant=quant, **a)
    assert codes.dtype == (torch.int8 if quant == "int8" else torch.float8_e4m3fn) and codes.shape == x.shape
    rx, dx, h, dh = reference(y, x, a)
    within(got_x, rx, dx)
    s = scales.double().cpu()[..., None]
    top = h.abs().amax(-1, keepdim=True)
    most = 127.0 if quant == "int8" else 448.0
    assert ((s * most - top).abs() <= dh.amax(-1, keepdim=True) + 2.0 ** -22 * top).all()
    value = codes.double().cpu() if quant == "int8" else codes.float().double().cpu()
    step = 0.5 * s if quant == "int8" else torch.maximum(2.0 ** -4 * h.abs(), 2.0 ** -10 * s)
    assert ((value * s - h).abs() <= step * (1 + 2.0 ** -20) + 2 * dh + 2.0 ** -22 * top).all()
    assert value.abs().max() <= most


def test_strides_and_alignment(cuda_device):
    from xgen_b200.ops import sandwich_norm

    g = torch.Generator().manual_seed(2)
    base = torch.randn(2, 6, 140, generator=g).to(cuda_device, torch.bfloat16)
    for w, lo in ((128, 0), (128, 1), (128, 8), (100, 3)):
        y, x = base[..., lo:lo + w], base.flip(0)[:, :, lo:lo + w]
        a = arguments(w, 4, torch.bfloat16, cuda_device, g, "rmsnorm", "rmsnorm", 6)
        got = sandwich_norm(y, x, **a)
        rx, dx, rh, dh = reference(y, x, a)
        within(got[0], rx, dx)
        within(got[1], rh, dh)
    # tokens before samples, one branch shared by the batch
    y, x = base[:1, :, :128].expand(3, 6, 128), torch.randn(6, 3, 128, generator=g).to(cuda_device, torch.bfloat16).transpose(0, 1)
    a = arguments(128, 1, torch.bfloat16, cuda_device, g, "layernorm", "rmsnorm", 6)
    got = sandwich_norm(y, x, **a)
    rx, dx, rh, dh = reference(y, x, a)
    within(got[0], rx, dx)
    within(got[1], rh, dh)


def test_far_mean_and_constant_rows(cuda_device):
    """A mean of 1000 deviations keeps its digits; a constant row has none."""
    from xgen_b200.ops import sandwich_norm

    g = torch.Generator().manual_seed(4)
    x = (1000 + torch.randn(1, 4, 1024, generator=g)).to(cuda_device)
    x[0, 3] = 7.0
    y = torch.zeros_like(x)
    _, h = sandwich_norm(y, x, post_norm=None, pre_norm="layernorm")
    ref = torch.nn.functional.layer_norm(x.double(), (1024,), eps=1e-6)
    # the mean is a sum of 1024 values near 1000: at most 32 roundings lie on one
    # value's way (chain, then tree), each 2^-24 of it; the deviation is one
    assert (h.double() - ref).abs()[0, :3].max() <= 32 * 2.0 ** -24 * 1010
    assert h[0, 3].abs().max() == 0


def test_index_outside_the_table(cuda_device):
    from xgen_b200.ops import sandwich_norm

    x = torch.randn(1, 5, 64, device=cuda_device).bfloat16()
    gate = torch.randn(2, 64, device=cuda_device).bfloat16()
    idx = torch.tensor([0, 2, 1, -1, 1 << 40], device=cuda_device)
    got, h = sandwich_norm(x, x, gate=gate, indices=idx)
    assert torch.isnan(got[0, [1, 3, 4]]).all() and torch.isnan(h[0, [1, 3, 4]]).all()
    assert torch.isfinite(got[0, [0, 2]]).all() and torch.isfinite(h[0, [0, 2]]).all()
    _, codes, scales = sandwich_norm(x, x, gate=gate, indices=idx, quant="int8")
    assert torch.isnan(scales[0, [1, 3, 4]]).all() and torch.isfinite(scales[0, [0, 2]]).all()


def test_zero_rows_and_empty(cuda_device):
    from xgen_b200.ops import sandwich_norm

    z = torch.zeros(2, 3, 256, device=cuda_device).bfloat16()
    x, codes, scales = sandwich_norm(z, z, quant="int8")
    assert not x.any() and not codes.any() and (scales > 0).all()
    x, h = sandwich_norm(z[:, :0], z[:, :0])
    assert x.shape == (2, 0, 256) and h.shape == (2, 0, 256)


def test_refusals(cuda_device):
    from xgen_b200.ops import sandwich_norm

    x = torch.randn(2, 4, 64, device=cuda_device).bfloat16()
    t = torch.randn(3, 64, device=cuda_device).bfloat16()
    i = torch.zeros(4, dtype=torch.long, device=cuda_device)
    for bad in (dict(scale=t, indices=i), dict(gate=t), dict(indices=i), dict(gate=t, indices=i.int()), dict(gate=t, indices=i[:3]),
                dict(gate=t.float(), indices=i), dict(gate=t[:, :32], indices=i), dict(pre_norm=None, quant="int8"),
                dict(post_norm="batchnorm"), dict(quant="int4"), dict(post_norm=None, post_weight=t[0]), dict(pre_weight=t[0, :8])):
        with pytest.raises(ValueError):
            sandwich_norm(x, x, **bad)
    with pytest.raises(ValueError):
        sandwich_norm(x, x.float())
    with pytest.raises(ValueError):
        sandwich_norm(x, x[:, :3])
    with pytest.raises(ValueError):
        sandwich_norm(torch.zeros(1, 1, 16385, device=cuda_device), torch.zeros(1, 1, 16385, device=cuda_device))
    with pytest.raises(ValueError, match="autograd"):
        sandwich_norm(x.clone().requires_grad_(), x)


def codes_in_64_bits(y, x, a, quant):
    """(x, codes' values, scales, where the quotient is off a code's border by more than 2^-30 of itself) from the definition."""
    norm = lambda t, kind, w: (lambda d: d / (d.pow(2).mean(-1, keepdim=True) + a["eps"]).sqrt() * (1.0 if w is None else w.double()))(  # noqa: E731
        t - t.mean(-1, keepdim=True) if kind == "layernorm" else t) if kind else t
    at = a.get("indices")
    v = norm(y.double(), a["post_norm"], a.get("post_weight"))
    if a.get("gate") is not None:
        v = v * a["gate"].double()[at]
    new = x.double() + a["residual_scale"] * v
    h = norm(new, a["pre_norm"], a.get("pre_weight"))
    if a.get("scale") is not None:
        h = h * (1 + a["scale"].double()[at]) + a["shift"].double()[at]
    s = (h.abs().amax(-1, keepdim=True) / (127 if quant == "int8" else 448)).clamp_min(torch.finfo(torch.float32).tiny)
    code = (lambda q: q.round()) if quant == "int8" else (lambda q: q.float().to(torch.float8_e4m3fn).double())
    low, high = (code(h / s * (1 + d)) for d in (-2.0 ** -30, 2.0 ** -30))
    return new, code(h / s), s[..., 0], low == high


@pytest.mark.parametrize("b,s,w", [(1, 16384, 336), (3, 1, 1), (2, 300, 33), (1, 700, 1001), (1, 200, 2001), (2, 60, 4100), (1, 9, 8200),
                                   (1, 5, 16384), (2, 801, 1536)])
@pytest.mark.parametrize("quant", ["int8", "e4m3"])
@pytest.mark.parametrize("post,pre", [("rmsnorm", "layernorm"), ("layernorm", "rmsnorm"), (None, "rmsnorm")])
def test_codes_of_32_bit_rows_are_the_definitions(cuda_device, b, s, w, quant, post, pre):
    """Next to a code's border a last bit decides, and the decoded value moves by
    a whole code: 32-bit rows are computed in 64 bits, and every code but those
    within 2^-30 of a border, relative, is that of the definition (64-bit errors
    are a few thousand times smaller). x and the scales are rounded once: half a
    step, 2^-24, and a 2^-20 part of it for the 64-bit errors."""
    from xgen_b200.ops import sandwich_norm

    g = torch.Generator().manual_seed(w)
    base = torch.randn(b, s, w + 1, generator=g).to(cuda_device)
    y, x = 0.7 * base[..., 1:] + 0.1, 2 * torch.randn(b, s, w, generator=g).to(cuda_device)
    a = {**arguments(w, 6, torch.float32, cuda_device, g, post, pre, s, modulate=s % 2 == 0), "residual_scale": 0.5, "eps": 2.0 ** -20}
    got, codes, scales = sandwich_norm(y, x, quant=quant, **a)
    rx, value, rs, sure = codes_in_64_bits(y, x, a, quant)
    assert sure.double().mean() > 1 - 1e-5
    off = (codes.float().double() != value) & sure
    assert not off.any(), (int(off.sum()), off.numel())
    assert ((scales.double() - rs).abs() <= 2.0 ** -24 * (1 + 2.0 ** -20) * rs).all()
    assert ((got.double() - rx).abs() <= 2.0 ** -24 * (1 + 2.0 ** -20) * rx.abs() + 2.0 ** -45).all()  # a sum that cancels: 64-bit errors
    again = sandwich_norm(base[..., 1:].mul(0.7).add(0.1), x, quant=quant, **a)  # the same rows, aligned
    assert all(torch.equal(p.view(torch.uint8) if p.dtype == torch.float8_e4m3fn else p, q.view(torch.uint8) if q.dtype == torch.float8_e4m3fn else q)
               for p, q in zip((got, codes, scales), again))


def test_codes_of_32_bit_rows_not_finite_and_tiny(cuda_device):
    from xgen_b200.ops import sandwich_norm

    x = torch.randn(1, 6, 200, device=cuda_device)
    x[0, 1, 3], x[0, 2, 4], x[0, 3] = float("nan"), float("inf"), 0.0
    x[0, 4] *= 1e-30
    gate, at = torch.ones(2, 200, device=cuda_device), torch.tensor([0, 0, 0, 0, 0, 2], device=cuda_device)
    got, codes, scales = sandwich_norm(torch.zeros_like(x), x, quant="int8", post_norm=None, pre_norm="rmsnorm", gate=gate, indices=at)
    assert torch.isnan(scales[0, 1]) and torch.isnan(scales[0, 2]) and torch.isnan(scales[0, 5]) and torch.isnan(got[0, 5]).all()
    assert not codes[0, 3].any() and scales[0, 3] == torch.finfo(torch.float32).tiny
    # far below eps the norm is x * 1000
    assert scales[0, 4] > 0 and codes[0, 4].abs().max() == 127
    assert torch.isfinite(scales[0, [0, 3, 4]]).all() and torch.equal(got[0, :5].nan_to_num(), x[0, :5].nan_to_num())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("w", [33, 64, 1536, 9999])
@pytest.mark.parametrize("quant", [1, 2])
def test_values_and_codes_of_one_call(cuda_device, dtype, w, quant):
    """The C entry may be given h_out and codes together: each is what a call
    for it alone gives (the codes of 32-bit rows are taken from h in 64 bits,
    which h_out rounds once)."""
    from xgen_b200 import _lib
    from xgen_b200.ops import _DTYPE_CODE_F32

    y, x = (torch.randn(2, 7, w, generator=torch.Generator().manual_seed(w + n)).to(cuda_device, dtype) for n in range(2))
    strides = (_lib.c_i64 * 3)(*x.stride())

    def call(values, codes):
        out = [torch.empty_like(x), torch.empty_like(x) if values else None, torch.empty(2, 7, w, dtype=torch.uint8, device=cuda_device) if codes else None,
               torch.empty(2, 7, device=cuda_device) if codes else None]
        p = [t.data_ptr() if t is not None else None for t in out]
        _lib.call("xgb_sandwich_norm", y.data_ptr(), strides, x.data_ptr(), strides, _DTYPE_CODE_F32[dtype], 2, 7, w, 2, None, 1, None, 1e-6, None, 0,
                  1.0, None, 0, None, 0, None, 0, 0, p[0], p[1], quant if codes else 0, p[2], p[3], torch.cuda.current_stream().cuda_stream)
        return out

    both, values, codes = call(True, True), call(True, False), call(False, True)
    assert torch.equal(both[2], codes[2]) and torch.equal(both[3], codes[3])
    if dtype == torch.float32:
        torch.testing.assert_close(both[1], values[1], rtol=2.0 ** -18, atol=2.0 ** -18 * values[1].abs().max().item())
    else:
        assert torch.equal(both[0], values[0]) and torch.equal(both[1], values[1])


@pytest.mark.parametrize("w", [100, 129, 1000, 1536, 5120, 10000])
def test_layernorm_far_from_zero(cuda_device, w):
    """The mean is taken off before anything is multiplied, and its own rounding
    error e is summed with the squares and taken off too.

    A constant row c: e is at most 32 roundings, 2^-19 |c|; the difference from
    the mean is exactly e everywhere, its mean is known to 2^-19 of it, so what
    is left is 2^-38 |c|, times 1/sqrt(eps).
    A mean of 1000 deviations: differences are exact (within a factor of two of
    the mean), their mean is known to 2^-19 of their mean magnitude (one
    deviation at most), 1/deviation to 2^-19: 2^-19 (1 + |h|) and the last
    roundings, 2^-22 (1 + |h|)."""
    from xgen_b200.ops import sandwich_norm

    eps, consts = 1e-5, torch.tensor([3.1415, 1000.3, 30.3, -7e4, 0.1], device=cuda_device)
    x = consts[None, :, None].expand(1, 5, w).contiguous()
    zero = torch.zeros_like(x)
    bound = 2.0 ** -38 * consts.abs() / eps ** 0.5
    for h in (sandwich_norm(zero, x, post_norm=None, pre_norm="layernorm", eps=eps)[1],
              sandwich_norm(x, zero, post_norm="layernorm", pre_norm=None, eps=eps)):
        assert (h[0].abs().amax(-1) <= bound).all(), h[0].abs().amax(-1) / bound
    x = (1000 + torch.randn(1, 50, w, generator=torch.Generator().manual_seed(w))).to(cuda_device)
    ref = torch.nn.functional.layer_norm(x.double(), (w,), eps=eps)
    bound = (2.0 ** -19 + 2.0 ** -22) * (1 + ref.abs())
    zero = torch.zeros_like(x)
    for h in (sandwich_norm(zero, x, post_norm=None, pre_norm="layernorm", eps=eps)[1],
              sandwich_norm(x, zero, post_norm="layernorm", pre_norm=None, eps=eps)):
        assert ((h.double() - ref).abs() <= bound).all(), ((h.double() - ref).abs() / bound).max()
