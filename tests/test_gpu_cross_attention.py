"""cross_attention against softmax attention in 64 bits over the keys that are
there.

Tolerance, with P rounded to the inputs' type (half a step e = eps/2 relative):
  the output's rounding                        e |o|
  P's rounding                                 e A,  A = sum p |v| / sum p
  a score's 32-bit error, which p carries as its own relative error: a sum of
  D products, each step within 2^-23 (the tensor core may truncate) of the sum
  of magnitudes, in numerator and denominator  2 scale D 2^-23 max sum |q k| / 8
  the two products' accumulation and exp2      2^-16 A
and for fp16 the p below its smallest number: 2^-25 for each key (sum p >= 1).
D/8: the tensor core adds at least 16 products in one step, D/16 steps, doubled."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def reference(q, k, v, valid, scale):
    """(o, A, largest sum |q k|) in 64 bits; valid bool [B, Skv]."""
    b, h, sq, d = q.shape
    group = h // k.shape[1]
    q, k, v = (t.double().cpu() for t in (q, k, v))
    o, a, top = torch.zeros(b, h, sq, d).double(), torch.zeros(b, h, sq, d).double(), 0.0
    for n in range(b):
        at = valid[n].nonzero()[:, 0]
        if not len(at):
            continue
        for j in range(h):
            kk, vv = k[n, j // group, at], v[n, j // group, at]
            p = torch.softmax(q[n, j] @ kk.t() * scale, -1)
            o[n, j], a[n, j] = p @ vv, p @ vv.abs()
            top = max(top, (q[n, j].abs() @ kk.abs().t()).max().item())
    return o, a, top


def check(got, q, k, v, valid, scale=None):
    scale = scale or 1 / math.sqrt(q.shape[-1])
    o, a, top = reference(q, k, v, valid, scale)
    info = torch.finfo(q.dtype)
    e = info.eps / 2
    slack = (e + 2 * scale * (q.shape[-1] / 8) * 2.0 ** -23 * top + 2.0 ** -16) * a
    if q.dtype == torch.float16:
        slack = slack + 2.0 ** -25 * k.shape[2] * torch.nan_to_num(v.double().cpu()).abs().max() * (a > 0)
    bound = e * (o.abs() + slack) + slack + info.smallest_normal * e
    assert got.shape == q.shape and got.dtype == q.dtype
    worst = ((got.double().cpu() - o).abs() / bound).max().item()
    assert worst <= 1.0, worst


def inputs(b, h, hk, sq, skv, d, dtype, dev, seed=0):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(b, sq, h, d, generator=g).to(dev, dtype).transpose(1, 2)
    kv = torch.randn(b, skv, 2, hk, d, generator=g)
    kv[:, :, 0] += torch.randn(hk, d, generator=g)
    kv = kv.to(dev, dtype)
    return q, kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)


@pytest.fixture(autouse=True)
def no_timeouts(cuda_device):
    yield
    from xgen_b200.attention import kernel_errors

    assert kernel_errors(cuda_device) == 0


@pytest.mark.parametrize("b,h,hk,sq,skv", [
    (1, 1, 1, 1, 1), (1, 2, 2, 128, 64), (1, 2, 1, 129, 65), (2, 3, 3, 300, 77), (1, 4, 2, 257, 512), (2, 2, 2, 1000, 333),
    (1, 1, 1, 5, 1000), (3, 2, 1, 64, 63), (1, 24, 24, 700, 226), (1, 6, 2, 1, 4099), (1, 1, 1, 3000, 2), (5, 8, 8, 17, 129),
    (2, 6, 2, 8, 1030), (1, 2, 2, 8, 600), (1, 1, 1, 1, 9000), (1, 2, 2, 9, 2000), (40, 4, 1, 2, 300)])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_matches_softmax(cuda_device, b, h, hk, sq, skv, d, dtype):
    from xgen_b200.attention import cross_attention

    q, k, v = inputs(b, h, hk, sq, skv, d, dtype, cuda_device, seed=sq + skv)
    got = cross_attention(q, k, v)
    check(got, q, k, v, torch.ones(b, skv, dtype=torch.bool))


@pytest.mark.parametrize("sq", [1, 40, 300])
@pytest.mark.parametrize("skv", [1, 64, 200, 1025])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_lengths(cuda_device, sq, skv, d, kind):
    """Every sample its own count: none, one, ends inside, at and over a tile's
    and the states' end; NaN and infinities behind it."""
    from xgen_b200.attention import cross_attention

    lens = [0, 1, min(63, skv), min(64, skv), min(65, skv), skv - 1, skv, skv + 100, -3]
    q, k, v = inputs(len(lens), 4, 2, sq, skv, d, torch.bfloat16, cuda_device, seed=skv)
    n = torch.tensor(lens, device=cuda_device, dtype=kind)
    valid = torch.arange(skv, device=cuda_device)[None] < n[:, None]
    for fill in (float("nan"), float("inf"), -3e38):
        k = k.masked_fill(~valid[:, None, :, None], fill)
        v = v.masked_fill(~valid[:, None, :, None], fill)
        got = cross_attention(q, k, v, kv_lens=n)
        check(got, q, k, v, valid.cpu())
    assert not got[0].any() and not got[-1].any()


@pytest.mark.parametrize("sq", [1, 300])
@pytest.mark.parametrize("skv", [1, 65, 333, 1500])
@pytest.mark.parametrize("d", [64, 128])
def test_masks(cuda_device, sq, skv, d):
    from xgen_b200.attention import cross_attention

    g = torch.Generator().manual_seed(skv)
    valid = torch.rand(5, skv, generator=g) < 0.6
    valid[0] = False
    valid[1] = True
    valid[2] = False
    valid[2, -1] = True  # the last key alone
    q, k, v = inputs(5, 4, 2, sq, skv, d, torch.float16, cuda_device, seed=skv)
    mask = valid.to(cuda_device)
    k, v = (t.masked_fill(~mask[:, None, :, None], float("nan")) for t in (k, v))
    got = cross_attention(q, k, v, key_mask=mask)
    check(got, q, k, v, valid)
    assert not got[0].any()
    assert torch.equal(got, cross_attention(q, k, v, key_mask=mask[:, None, None]))
    one = mask[3:4]
    kk, vv = (t[3:4].expand(5, -1, -1, -1) for t in (k, v))
    got = cross_attention(q, kk, vv, key_mask=one)
    check(got, q, kk, vv, valid[3:4].expand(5, -1))


@pytest.mark.parametrize("d,dtype", [(64, torch.float16), (128, torch.bfloat16)])
@pytest.mark.parametrize("skv", [1, 60, 64, 200, 520])
def test_many_units_for_each_cta(cuda_device, d, dtype, skv):
    """Long query sequences: every CTA walks several units, of one key tile and
    of many, and of samples without keys in between."""
    from xgen_b200.attention import cross_attention

    b, h, sq = 4, 6, 10000  # 960 units
    q, k, v = inputs(b, h, 3, sq, skv, d, dtype, cuda_device, seed=skv)
    lens = torch.tensor([skv, 0, max(1, skv // 3), skv], dtype=torch.int32)
    for n in (None, lens):
        got = cross_attention(q, k, v, kv_lens=n.to(cuda_device) if n is not None else None)
        valid = torch.ones(b, skv, dtype=torch.bool) if n is None else torch.arange(skv)[None] < n[:, None]
        at = torch.cat([torch.arange(0, sq, 97), torch.arange(sq - 20, sq)])  # rows of all units
        check(got[:, :, at], q[:, :, at], k, v, valid)
        if n is not None:
            assert not got[1].any()


def test_later_tiles_far_above_the_first(cuda_device):
    """The first 64 keys set a row's reference value; later scores exceed it by
    2^20 to 2^400, in some rows only, once or again and again."""
    from xgen_b200.attention import cross_attention

    for dtype, steps in ((torch.bfloat16, (0, 60, 70, 300, 310, 50)), (torch.float16, (0, 12, 30, 60, 61, 3))):
        skv = 64 * len(steps) + 5
        q, k, v = inputs(1, 2, 2, 150, skv, 64, dtype, cuda_device, seed=3)
        q, k = q * 0.25, k * 0.25
        q[..., 0] = torch.where(torch.arange(150, device=cuda_device) % 3 == 0, 1.0, 0.0).to(dtype)
        raise_by = torch.tensor(steps, device=cuda_device).repeat_interleave(64)
        k[..., 0] = torch.cat([raise_by, raise_by[:5]]).to(dtype) / 4
        got = cross_attention(q, k, v, sm_scale=math.log(2) * 4)  # scores in log2 units: steps
        check(got, q, k, v, torch.ones(1, skv, dtype=torch.bool), math.log(2) * 4)


def test_large_scores_and_infinities(cuda_device):
    """Scores far apart (the running maximum rises many times), rows of -inf
    scores, and a value of infinity where it is attended to."""
    from xgen_b200.attention import cross_attention

    q, k, v = inputs(1, 2, 2, 200, 700, 128, torch.bfloat16, cuda_device, seed=9)
    ramp = torch.linspace(0.02, 6, 700, device=cuda_device).to(torch.bfloat16)[:, None]
    got = cross_attention(q, k * ramp, v)
    check(got, q, k * ramp, v, torch.ones(1, 700, dtype=torch.bool))
    got = cross_attention(q, k, v, sm_scale=1e-4)
    check(got, q, k, v, torch.ones(1, 700, dtype=torch.bool), 1e-4)
    q2 = torch.full_like(q, 1.0)
    k2 = k.clone()
    k2[:, :, 100:] = float("-inf")  # scores of -inf: as if the keys were not there
    got = cross_attention(q2, k2, v)
    check(got, q2, k[:, :, :100], v[:, :, :100], torch.ones(1, 100, dtype=torch.bool))
    assert not cross_attention(q2, torch.full_like(k, float("-inf")), v).any()
    v2 = v.clone()
    v2[0, 0, 3, 7] = float("inf")
    got = cross_attention(q, k, v2)
    assert torch.isinf(got[0, 0, :, 7]).all() and torch.isfinite(got[0, 1]).all()
    q3 = q.clone()
    q3[0, 1, 5] = float("nan")
    got, clean = cross_attention(q3, k, v), cross_attention(q, k, v)
    bad = torch.zeros(1, 2, 200, dtype=torch.bool, device=cuda_device)
    bad[0, 1, 5] = True
    assert torch.isnan(got[bad]).all() and torch.equal(got[~bad], clean[~bad])


def test_strides_broadcast_and_output(cuda_device):
    from xgen_b200.attention import cross_attention

    b, h, sq, skv, d = 3, 4, 150, 130, 64
    q, k, v = inputs(b, h, h, sq, skv, d, torch.bfloat16, cuda_device, seed=1)
    every = torch.ones(b, skv, dtype=torch.bool)
    hnd = [t.contiguous() for t in (q, k, v)]
    base = cross_attention(*hnd)
    check(base, q, k, v, every)
    assert torch.equal(base, cross_attention(q, k, v))
    # rows of a wider projection; every second token
    wide = torch.randn(b, sq, h, 2 * d, device=cuda_device).bfloat16()[..., d:].transpose(1, 2)
    check(cross_attention(wide, k, v), wide, k, v, every)
    half = cross_attention(q, k[:, :, ::2], v[:, :, 1::2])
    check(half, q, k[:, :, ::2], v[:, :, 1::2], every[:, :65])
    # states shared by the batch, and by the heads
    kb, vb = k[:1].expand(b, -1, -1, -1), v[:, :1].expand(-1, h, -1, -1)
    check(cross_attention(q, kb, vb), q, kb, vb, every)
    # into the layout of the next projection; what lies beside the view stays
    frame = torch.full((b, sq + 2, h, d), 5.0, device=cuda_device).bfloat16()
    out = frame[:, 1:-1].transpose(1, 2)
    assert cross_attention(q, k, v, out=out) is out
    assert torch.equal(out, base) and (frame[:, 0] == 5).all() and (frame[:, -1] == 5).all()


def test_empty(cuda_device):
    from xgen_b200.attention import cross_attention

    q, k, v = inputs(2, 2, 2, 10, 20, 64, torch.bfloat16, cuda_device)
    assert cross_attention(q[:, :, :0], k, v).shape == (2, 2, 0, 64)
    assert not cross_attention(q, k[:, :, :0], v[:, :, :0]).any()
    assert cross_attention(q[:0], k[:0], v[:0]).shape == (0, 2, 10, 64)


@pytest.mark.parametrize("sq,skv", [(1, 2000), (700, 200)])
def test_two_streams_and_graphs(cuda_device, sq, skv):
    """Calls on two streams at once, and two captured graphs replayed in turn
    and at once, give what single calls give: nothing is shared."""
    from xgen_b200.attention import cross_attention

    sets = [inputs(2, 4, 2, sq, skv, 128, torch.bfloat16, cuda_device, seed=n) for n in range(2)]
    lens = [torch.tensor([skv, skv // 3], device=cuda_device, dtype=torch.int32),
            torch.tensor([7, skv], device=cuda_device, dtype=torch.int32)]
    single = [cross_attention(*s, kv_lens=n) for s, n in zip(sets, lens)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        outs = []
        for st, s, n in zip(streams, sets, lens):
            with torch.cuda.stream(st):
                outs.append(cross_attention(*s, kv_lens=n))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, single))
    graphs, results = [], []
    for s, n in zip(sets, lens):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results.append(cross_attention(*s, kv_lens=n))
        graphs.append(graph)
    for _ in range(3):
        for r in results:
            r.zero_()
        torch.cuda.synchronize()
        for st, graph in zip(streams, graphs):
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(results, single))
    lens[0].copy_(torch.tensor([3, 0]))  # a replay reads the lengths of its time
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(results[0], cross_attention(*sets[0], kv_lens=lens[0]))


def test_same_call_gives_the_same_bits(cuda_device):
    from xgen_b200.attention import cross_attention

    for sq, skv in ((1, 4099), (3000, 300)):
        q, k, v = inputs(1, 4, 4, sq, skv, 128, torch.bfloat16, cuda_device)
        first = cross_attention(q, k, v)
        assert all(torch.equal(first, cross_attention(q, k, v)) for _ in range(5))


def test_long_caches(cuda_device):
    """Element offsets beyond 32 bits: 2^31 elements of K before the last head."""
    from xgen_b200.attention import cross_attention

    skv, h, d = 70000, 160, 128
    assert h * skv * d > 2 ** 30 and 2 * h * skv * d > 2 ** 31
    kv = torch.zeros(2, h, skv, d, device=cuda_device, dtype=torch.bfloat16)  # rows of one tensor: K, V
    g = torch.Generator().manual_seed(0)
    last = torch.randn(2, 1, 200, d, generator=g).to(cuda_device, torch.bfloat16)
    wide = kv.view(1, 2 * h, skv, d)
    wide[0, 2 * h - 1, -200:], wide[0, 2 * h - 2, -200:] = last[1, 0], last[0, 0]
    q = torch.randn(1, 1, 30, d, generator=g).to(cuda_device, torch.bfloat16)
    k, v = wide[:, 2 * h - 2:2 * h - 1, -200:], wide[:, 2 * h - 1:, -200:]
    check(cross_attention(q, k, v), q, k, v, torch.ones(1, 200, dtype=torch.bool))
    q2 = q.expand(1, 2 * h, 30, d)
    got = cross_attention(q2, wide[:, :, -200:], wide[:, :, -200:])
    check(got[:, -1:], q, wide[:, -1:, -200:], wide[:, -1:, -200:], torch.ones(1, 200, dtype=torch.bool))


def test_refusals(cuda_device):
    from xgen_b200.attention import cross_attention

    q, k, v = inputs(2, 4, 2, 10, 20, 64, torch.bfloat16, cuda_device)
    lens = torch.ones(2, dtype=torch.int32, device=cuda_device)
    mask = torch.ones(2, 20, dtype=torch.bool, device=cuda_device)
    for bad in (dict(kv_lens=lens, key_mask=mask), dict(kv_lens=lens[:1]), dict(kv_lens=lens.float()), dict(key_mask=mask.int()),
                dict(key_mask=mask[:, :10]), dict(sm_scale=0.0), dict(sm_scale=float("nan")), dict(out=q[:, :, :5]),
                dict(out=torch.empty_like(q).float()), dict(key_mask=mask[:, None].expand(2, 4, 20)[:, :, None])):
        with pytest.raises(ValueError):
            cross_attention(q, k, v, **bad)
    for bad in ((q.float(), k.float(), v.float()), (q, k.half(), v), (q[..., :32], k[..., :32], v[..., :32]), (q, k, v[:, :, :10]),
                (q[:, :3], k, v), (q[:1], k, v), (q, k[:, :, :, ::1].transpose(2, 3), v), (q.cpu(), k, v)):
        with pytest.raises(ValueError):
            cross_attention(*bad)
    odd = torch.zeros(2, 10, 4, 68, device=cuda_device, dtype=torch.bfloat16)[..., :64].transpose(1, 2)  # rows of 136 bytes
    with pytest.raises(ValueError):
        cross_attention(odd, k, v)
    with pytest.raises(ValueError):
        cross_attention(q, k[:, :, :1].expand(-1, -1, 20, -1), v)  # one key for all places
    with pytest.raises(ValueError, match="autograd"):
        cross_attention(q.clone().requires_grad_(), k, v)


@pytest.mark.parametrize("sq", [1, 3400])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rise", [7, 9, 20, 39, 60])
def test_large_values_behind_a_late_high_score(cuda_device, sq, d, rise):
    """Scores of later tiles that exceed the first's by 2^7 to 2^60, and values
    up to 2^116: below 2^126 / 330, so the result is finite. One token, and 84
    units, which are more than half the SMs and so keep all their keys."""
    from xgen_b200.attention import cross_attention

    q, k, v = inputs(2, 3, 3, sq, 330, d, torch.bfloat16, cuda_device, seed=rise)
    q, k = 0.05 * q, 0.05 * k
    q[..., 0] = 1.0
    k[..., 0] = torch.where(torch.arange(330, device=cuda_device) >= 100, float(rise), 0.0).to(torch.bfloat16)
    v = (v.float().clamp(-4, 4) * 2.0 ** 114).to(torch.bfloat16)
    got = cross_attention(q, k, v, sm_scale=math.log(2))
    assert torch.isfinite(got).all()
    at = torch.cat([torch.arange(0, sq, 61), torch.arange(max(0, sq - 20), sq)])
    check(got[:, :, at], q[:, :, at], k, v, torch.ones(2, 330, dtype=torch.bool), math.log(2))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens", [False, True])
def test_scores_that_rise_within_whole_units(cuda_device, d, dtype, lens):
    """The row's reference value is raised at some tiles, in some rows, of units
    that keep all their keys, again and again and by 2^3 to 2^300; the samples
    differ in their number of tiles."""
    from xgen_b200.attention import cross_attention

    steps = (0, 3, 60, 61, 70, 300, 310, 50) if dtype == torch.bfloat16 else (0, 3, 12, 30, 60, 61, 75, 3)
    skv = 64 * len(steps) - 9
    b, h, sq = 3, 3, 2600  # 99 units
    q, k, v = inputs(b, h, 3, sq, skv, d, dtype, cuda_device, seed=d)
    q, k = q * 0.25, k * 0.25
    q[..., 0] = ((torch.arange(sq, device=cuda_device) // 5) % 3 == 0).to(dtype)
    k[..., 0] = (torch.tensor(steps, device=cuda_device).repeat_interleave(64)[:skv] / 4).to(dtype)
    n = torch.tensor([skv, 150, 321], dtype=torch.int32) if lens else None
    got = cross_attention(q, k, v, sm_scale=math.log(2) * 4, kv_lens=n.to(cuda_device) if lens else None)
    valid = torch.arange(skv)[None] < n[:, None] if lens else torch.ones(b, skv, dtype=torch.bool)
    at = torch.cat([torch.arange(0, sq, 37), torch.arange(sq - 20, sq)])
    check(got[:, :, at], q[:, :, at], k, v, valid, math.log(2) * 4)


@pytest.mark.parametrize("sq", [1, 40, 3400])
def test_small_values(cuda_device, sq):
    """Magnitudes of 2^-80 keep their digits: the same result as at 1, scaled."""
    from xgen_b200.attention import cross_attention

    q, k, v = inputs(2, 3, 3, sq, 330, 128, torch.bfloat16, cuda_device, seed=4)
    v = (v.float().sign() * (1 + v.float().abs())).to(torch.bfloat16)
    got, small = cross_attention(q, k, v), cross_attention(q, k, (v.float() * 2.0 ** -80).to(torch.bfloat16))
    # what is lost of a sum where products below 2^-126 are: 330 of them against
    # a p of at least 2^-24 times 2^-80, 2^-13 of the mean magnitude
    a = cross_attention(q, k, v.abs()).double()
    assert ((small.double() * 2.0 ** 80 - got.double()).abs() <= 2.0 ** -8 * got.double().abs() + 2.0 ** -13 * a).all()


def test_scale_is_read_at_every_call(cuda_device):
    """A scale that float() takes, a tensor of one value among them, counts with
    its value of the time of the call."""
    from xgen_b200.attention import cross_attention

    q, k, v = inputs(1, 2, 2, 40, 90, 64, torch.bfloat16, cuda_device)
    scale = torch.tensor(0.25)
    first = cross_attention(q, k, v, sm_scale=scale)
    scale.fill_(0.03125)
    second = cross_attention(q, k, v, sm_scale=scale)
    assert torch.equal(first, cross_attention(q, k, v, sm_scale=0.25))
    assert torch.equal(second, cross_attention(q, k, v, sm_scale=0.03125)) and not torch.equal(first, second)
