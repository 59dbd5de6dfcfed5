"""rope_axes against its formula in 64 bits.

Tolerance: the result is a rounding of a 32-bit value, half a step of the type
relative to it, and that value is off by what 32-bit arithmetic does to
a cos - b sin: a few 2^-24 of |a| + |b| for the products, the sum and cos/sin
(whose argument is rounded to 2^-25 of a turn, 2 pi 2^-25 radians), and with
the norm as much again for the mean of up to 512 squares, the reciprocal root
and the weight. 64 * 2^-24 of |a| + |b| holds both."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def rope64(x, positions, axes, thetas, interleaved, norm):
    """(rotated, magnitude |a| + |b| behind each value) of x [B, S, H, D]."""
    x = x.double().cpu()
    if norm is not None:
        x = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + norm.eps) * norm.weight.detach().double().cpu()
    out, size = x.clone(), x.abs()
    half, at = sum(axes) // 2, 0
    for n, d in enumerate(axes):
        for i in range(d // 2):
            angle = (positions[..., n].double().cpu() * thetas[n] ** (-2.0 * i / d))[..., None]
            c, s = torch.cos(angle), torch.sin(angle)
            l, r = (2 * at, 2 * at + 1) if interleaved else (at, at + half)
            a, b = x[..., l], x[..., r]
            out[..., l], out[..., r] = a * c - b * s, b * c + a * s
            size[..., l] = size[..., r] = a.abs() + b.abs()
            at += 1
    return out, size


def check(got, x, positions, axes, interleaved=False, norm=None, theta=10000.0):
    thetas = theta if isinstance(theta, tuple) else (theta,) * len(axes)
    ref, size = rope64(x, positions, axes, thetas, interleaved, norm)
    slack = 64 * 2.0 ** -24 * size
    info = torch.finfo(x.dtype)
    bound = info.eps / 2 * (ref.abs() + slack) + slack + info.smallest_normal * info.eps / 2
    assert got.shape == x.shape and got.dtype == x.dtype and got.is_contiguous()
    worst = ((got.double().cpu() - ref).abs() / bound).max().item()
    assert worst <= 1.0, worst


def make_norm(d, dtype, dev, g):
    norm = torch.nn.RMSNorm(d, eps=1e-5, device=dev, dtype=dtype)
    norm.weight = torch.nn.Parameter((1 + 0.2 * torch.randn(d, generator=g)).to(dev, dtype), requires_grad=False)
    return norm


@pytest.mark.parametrize("b,s,h,hk,d,axes", [
    (1, 1, 1, 1, 64, (16, 24, 24)), (1, 300, 24, 24, 128, (32, 48, 48)), (2, 77, 12, 4, 128, (32, 32, 32)),
    (3, 5, 2, 1, 96, (48, 48)), (1, 33, 3, 3, 80, (16, 30, 34)), (2, 19, 2, 2, 7, (2, 4)), (1, 9, 1, 1, 512, (512,)),
    (1, 41, 5, 2, 72, (8, 16, 16)), (1, 257, 2, 2, 256, (64, 64, 64, 64)), (1, 13, 48, 48, 64, (64,))])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("normed", [False, True])
def test_matches_formula(cuda_device, b, s, h, hk, d, axes, interleaved, dtype, normed):
    from xgen_b200.ops import rope_axes

    g = torch.Generator().manual_seed(s + d)
    fused = torch.randn(b, s, (h + 2 * hk) * d, generator=g).to(cuda_device, dtype)
    q, k = fused[..., :h * d].unflatten(-1, (h, d)), fused[..., h * d:(h + hk) * d].unflatten(-1, (hk, d))
    positions = torch.randint(0, 200, (b, s, len(axes)), generator=g).to(cuda_device)
    nq, nk = (make_norm(d, dtype, cuda_device, g) for _ in range(2)) if normed else (None, None)
    qo, ko = rope_axes(q, k, positions, axes=axes, interleaved=interleaved, norm_q=nq, norm_k=nk)
    check(qo, q, positions, axes, interleaved, nq)
    check(ko, k, positions, axes, interleaved, nk)


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64, torch.float32, torch.float64])
def test_position_types_and_far_positions(cuda_device, dtype):
    """Angles of 1e5 and 1e6 radians, negative ones, fractions."""
    from xgen_b200.ops import rope_axes

    g = torch.Generator().manual_seed(3)
    q = torch.randn(1, 64, 2, 64, generator=g).to(cuda_device)
    positions = torch.randint(-1000000, 1000000, (64, 3), generator=g).to(cuda_device, dtype)
    if dtype.is_floating_point:
        positions = positions / 7
    qo, none = rope_axes(q, None, positions, axes=(16, 24, 24), theta=(10000.0, 500.0, 1e6))
    assert none is None
    check(qo, q, positions, (16, 24, 24), theta=(10000.0, 500.0, 1e6))


def test_equals_the_tables_of_the_grid(cuda_device):
    """Positions of a grid give the rotation of rope_3d's tables."""
    from xgen_b200.h3.rope import rope_3d
    from xgen_b200.ops import rope_axes

    grid, extra = (3, 4, 5), 6
    cos, sin = rope_3d(grid, extra)
    t, h, w = torch.meshgrid(*(torch.arange(n) for n in grid), indexing="ij")
    pos = torch.stack([t.reshape(-1), h.reshape(-1), w.reshape(-1)], -1)
    tail = torch.stack([grid[0] + torch.arange(extra), torch.zeros(extra).long(), torch.zeros(extra).long()], -1)
    pos = torch.cat([pos, tail]).to(cuda_device)
    q = torch.randn(2, pos.shape[0], 3, 128, generator=torch.Generator().manual_seed(1)).to(cuda_device)
    got, _ = rope_axes(q, None, pos, axes=(32, 48, 48))
    c, s = cos.to(cuda_device)[None, :, None], sin.to(cuda_device)[None, :, None]
    ref = q * c + torch.cat([-q[..., 64:], q[..., :64]], -1) * s
    torch.testing.assert_close(got, ref, rtol=0, atol=2e-5)


def test_strides_alignment_and_broadcast(cuda_device):
    """Views at odd element offsets, heads before tokens, broadcast heads and batch."""
    from xgen_b200.ops import rope_axes

    g = torch.Generator().manual_seed(5)
    positions = torch.rand(21, 2, generator=g).to(cuda_device) * 50
    base = torch.randn(2, 4, 21, 67, generator=g).to(cuda_device, torch.bfloat16)
    for view in (base[..., 1:65].transpose(1, 2), base[..., 3:67].transpose(1, 2)[:, :, ::2],
                 base[:1, :1, :, :64].transpose(1, 2).expand(3, 21, 5, 64)):
        qo, ko = rope_axes(view, view, positions, axes=(32, 32))
        check(qo, view, positions, (32, 32))
        assert torch.equal(qo, ko)
    wide = torch.rand(2, 21, 5, generator=g).to(cuda_device)[:, :, ::2][..., :2]  # strided positions
    qo, _ = rope_axes(base[..., :64].transpose(1, 2), None, wide, axes=(32, 32))
    check(qo, base[..., :64].transpose(1, 2), wide, (32, 32))


def test_empty_sequences(cuda_device):
    from xgen_b200.ops import rope_axes

    q = torch.empty(2, 0, 3, 64, device=cuda_device)
    qo, ko = rope_axes(q, q, torch.empty(0, 1, device=cuda_device), axes=(64,))
    assert qo.shape == q.shape and ko.shape == q.shape


def test_not_a_number_stays_in_its_head(cuda_device):
    from xgen_b200.ops import rope_axes

    q = torch.randn(1, 6, 4, 64, device=cuda_device).bfloat16()
    clean, _ = rope_axes(q, None, torch.arange(6, device=cuda_device)[:, None], axes=(64,),
                         norm_q=torch.nn.RMSNorm(64, eps=1e-6, device=cuda_device, dtype=torch.bfloat16).requires_grad_(False))
    q[0, 2, 1, 5] = float("nan")
    got, _ = rope_axes(q, None, torch.arange(6, device=cuda_device)[:, None], axes=(64,),
                       norm_q=torch.nn.RMSNorm(64, eps=1e-6, device=cuda_device, dtype=torch.bfloat16).requires_grad_(False))
    bad = torch.zeros(1, 6, 4, 64, dtype=torch.bool, device=cuda_device)
    bad[0, 2, 1] = True
    assert torch.isnan(got[bad]).all() and torch.equal(got[~bad], clean[~bad])


def test_refusals(cuda_device):
    from xgen_b200.ops import rope_axes

    q = torch.randn(1, 4, 2, 64, device=cuda_device)
    pos = torch.zeros(4, 2, device=cuda_device)
    for bad in (dict(axes=(32, 31)), dict(axes=(32, 34)), dict(axes=(64,)), dict(axes=(32, 32), theta=-1.0),
                dict(axes=(32, 32), theta=(1.0,)), dict(axes=(32, 32), norm_q=torch.nn.LayerNorm(64))):
        with pytest.raises(ValueError):
            rope_axes(q, None, pos, **bad)
    with pytest.raises(ValueError):
        rope_axes(q, q[:, :3], pos, axes=(32, 32))
    with pytest.raises(ValueError):
        rope_axes(q, None, pos.half(), axes=(32, 32))
    with pytest.raises(ValueError):
        rope_axes(q.double(), None, pos, axes=(32, 32))
    with pytest.raises(ValueError, match="autograd"):
        rope_axes(q.clone().requires_grad_(), None, pos, axes=(32, 32))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("std", [1.0, 0.02, 1e-4])
def test_norm_without_an_eps(cuda_device, dtype, std):
    """torch.nn.RMSNorm's default: the module itself is the definition. At
    positions of zero nothing turns; the module may round in between, so a step
    of the type."""
    from xgen_b200.ops import rope_axes

    g = torch.Generator().manual_seed(7)
    norm = torch.nn.RMSNorm(64, device=cuda_device, dtype=dtype).requires_grad_(False)
    q = (std * torch.randn(1, 30, 2, 64, generator=g)).to(cuda_device, dtype)
    got, _ = rope_axes(q, None, torch.zeros(30, 1, device=cuda_device, dtype=torch.int64), axes=(64,), norm_q=norm)
    ref = norm(q).double()
    step = torch.finfo(dtype).eps
    assert ((got.double() - ref).abs() <= 2 * step * ref.abs() + step * torch.finfo(dtype).smallest_normal).all()


@pytest.mark.parametrize("d,axes", [(128, (32, 32, 32)), (128, (16,)), (72, (8, 16, 16)), (96, (30, 20))])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_channels_that_are_not_rotated_are_copied(cuda_device, d, axes, interleaved, dtype):
    """Bit for bit, infinities, NaN and zeros of either sign among them, in the
    vector form (d and the axes' sum multiples of 16) and the scalar one."""
    from xgen_b200.ops import rope_axes

    r = sum(axes)
    q = torch.randn(1, 40, 3, d, generator=torch.Generator().manual_seed(d)).to(cuda_device, dtype)
    for n, value in enumerate((float("inf"), -float("inf"), float("nan"), -0.0, 0.0)):
        q[0, n::7, :, r + n] = value
        q[0, n::9, :, d - 1 - n] = value
    positions = torch.arange(40 * len(axes), device=cuda_device).view(40, -1)
    got, key = rope_axes(q, q, positions, axes=axes, interleaved=interleaved)
    bits = torch.int32 if dtype == torch.float32 else torch.int16
    nan = torch.isnan(q[..., r:])
    assert torch.equal(torch.isnan(got[..., r:]), nan)
    assert torch.equal(got[..., r:].contiguous().view(bits)[~nan], q[..., r:].contiguous().view(bits)[~nan])
    check(got[..., :r].contiguous(), q[..., :r], positions, axes, interleaved)
    assert torch.equal(key.view(bits), got.view(bits))


def test_bases_are_read_at_every_call(cuda_device):
    """Bases and axes that float() and int() take count with their values of the
    time of the call."""
    from xgen_b200.ops import rope_axes

    q = torch.randn(1, 9, 2, 64, device=cuda_device)
    positions = torch.arange(18, device=cuda_device).view(9, 2)
    theta = torch.tensor(100.0)
    for wrap in (lambda t: t, lambda t: (t, t), lambda t: [t, t]):
        for value in (100.0, 5000.0):
            theta.fill_(value)
            got, _ = rope_axes(q, None, positions, axes=(32, 32), theta=wrap(theta))
            assert torch.equal(got, rope_axes(q, None, positions, axes=(32, 32), theta=value)[0])
    axes = torch.tensor([32, 32])
    rope_axes(q, None, positions, axes=axes)
    axes.copy_(torch.tensor([16, 48]))
    assert torch.equal(rope_axes(q, None, positions, axes=axes)[0], rope_axes(q, None, positions, axes=(16, 48))[0])
    pair = tuple(axes)  # two views of it
    rope_axes(q, None, positions, axes=pair)
    axes.copy_(torch.tensor([48, 16]))
    assert torch.equal(rope_axes(q, None, positions, axes=pair)[0], rope_axes(q, None, positions, axes=(48, 16))[0])
