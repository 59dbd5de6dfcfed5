"""The operators of a conditioned block one after another, as a model runs them.

    x, codes = sandwich_norm(branch, residual)         the norm before the block, as int8 codes
    q = Wq codes;  k, v = Wkv states                   int8 projections
    q = rope_axes(rms(q))                              positions of the queries
    o = cross_attention(q, k, v, keys that are there)
    x = x + gate * Wo o                                int8 with its gated residual
    x, h = sandwich_norm(Wd swiglu(Wu h'), x)          the feed-forward between two norms

Each step is held to its 64-bit definition of the tensors that it was given,
within the tolerance that its own tests derive; and the captured block replayed
on another stream repeats every bit."""
import pytest
import torch
import test_gpu_cross_attention as cross
import test_gpu_int8_linear as int8
import test_gpu_rope_axes as rope
import test_gpu_sandwich_norm as norms

pytestmark = pytest.mark.gpu


class Block:
    def __init__(self, heads, kv_heads, d, states, dtype, dev, seed):
        from xgen_b200.int8_linear import H3Int8Linear

        g = torch.Generator().manual_seed(seed)
        self.w, self.heads, self.kv_heads, self.d = heads * d, heads, kv_heads, d
        w = self.w

        def linear(n, k, activation=None):
            weight, bias = torch.randn(n, k, generator=g) / k ** 0.5, 0.1 * torch.randn(n, generator=g)
            return H3Int8Linear(weight.to(dev), bias.to(dev, dtype), activation)

        self.q, self.kv, self.o = linear(w, w), linear(2 * kv_heads * d, states), linear(w, w)
        self.up, self.down = linear(4 * w, w, "swiglu"), linear(w, 2 * w)
        self.norm = rope.make_norm(d, dtype, dev, g)
        self.table = (0.4 * torch.randn(7, 6 * w, generator=g)).to(dev, dtype)
        self.axes = (d // 4, 3 * d // 8, 3 * d // 8)

    def before(self, at):
        w = self.w
        return {"post_norm": "rmsnorm", "pre_norm": "layernorm", "gate": self.table[:, :w], "scale": self.table[:, w:2 * w],
                "shift": self.table[:, 2 * w:3 * w], "indices": at}

    def after(self, at):
        w = self.w
        return {"post_norm": "rmsnorm", "pre_norm": "rmsnorm", "gate": self.table[:, 3 * w:4 * w],
                "scale": self.table[:, 4 * w:5 * w], "shift": self.table[:, 5 * w:], "indices": at, "residual_scale": 0.7}

    def run(self, branch, residual, states, at, positions, **keys):
        """Every tensor between the steps, in their order."""
        from xgen_b200.attention import cross_attention
        from xgen_b200.ops import rope_axes, sandwich_norm

        b, s, w = residual.shape
        x, codes, scales = sandwich_norm(branch, residual, quant="int8", **self.before(at))
        q = self.q.forward_quantized(codes, scales, dtype=residual.dtype)
        kv = self.kv(states).unflatten(-1, (2, self.kv_heads, self.d))
        turned, _ = rope_axes(q.unflatten(-1, (self.heads, self.d)), None, positions, axes=self.axes, norm_q=self.norm)
        o = residual.new_empty(b, s, self.heads, self.d)
        cross_attention(turned.transpose(1, 2), kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2),
                        out=o.transpose(1, 2), **keys)
        x1 = self.o.forward_gated(o.flatten(2), self.table[:, :w], at, x)
        up = self.up(x1)
        x2, h = sandwich_norm(self.down(up), x1, **self.after(at))
        return x, codes, scales, q, kv, turned, o, x1, up, x2, h


@pytest.mark.parametrize("b,s,heads,kv_heads,d,skv,states,dtype,kind", [
    (2, 333, 12, 12, 128, 77, 1024, torch.bfloat16, "lens"), (1, 1, 12, 4, 64, 512, 768, torch.bfloat16, None),
    (3, 130, 4, 2, 64, 226, 256, torch.float16, "mask"), (4, 17, 6, 6, 128, 300, 512, torch.float16, "lens")])
def test_block(cuda_device, b, s, heads, kv_heads, d, skv, states, dtype, kind):
    block = Block(heads, kv_heads, d, states, dtype, cuda_device, seed=s)
    g = torch.Generator().manual_seed(skv)
    w = block.w
    branch, residual = (torch.randn(b, s, w, generator=g).to(cuda_device, dtype) for _ in range(2))
    enc = torch.randn(b, skv, states, generator=g).to(cuda_device, dtype)
    at = torch.randint(0, 7, (s,), generator=g).to(cuda_device)
    positions = torch.randint(0, 60, (s, 3), generator=g).to(cuda_device)
    keys, valid = {}, torch.ones(b, skv, dtype=torch.bool)
    if kind == "lens":  # the last sample has no keys
        lens = torch.tensor([skv, skv // 2, 1, 0][:b - 1] + [0])
        keys, valid = {"kv_lens": lens.to(cuda_device)}, torch.arange(skv) < lens[:, None]
    elif kind == "mask":
        valid = torch.rand(b, skv, generator=g) < 0.6
        keys = {"key_mask": valid.to(cuda_device)}
    inputs = (branch, residual, enc, at, positions)
    x, codes, scales, q, kv, turned, o, x1, up, x2, h = block.run(*inputs, **keys)

    rx, dx, rh, dh = norms.reference(branch, residual, block.before(at))
    norms.within(x, rx, dx)
    step = scales.double().cpu()[..., None]
    # half a code, the error of h, and that of the scale (2^-22 of its 127 codes)
    assert ((codes.double().cpu() * step - rh).abs() <= step / 2 + dh.amax(-1, keepdim=True) * 2 + step * 127 * 2.0 ** -22).all()

    def linear(got, module, codes, scales, gated=None):
        n = codes.shape[-1]
        ref, slack = int8.reference(codes.reshape(-1, n), scales.reshape(-1), module.weight, module.weight_scale,
                                    module.bias, module.activation, gated)
        int8.within(got.reshape(ref.shape), ref, slack)

    def codes_of(t):
        return int8.codes_of(t.reshape(-1, t.shape[-1]))

    linear(q, block.q, codes, scales)
    linear(kv.flatten(2), block.kv, *codes_of(enc))
    rope.check(turned, q.unflatten(-1, (heads, d)), positions[None], block.axes, False, block.norm)
    cross.check(o.transpose(1, 2), turned.transpose(1, 2), kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2), valid)
    linear(x1, block.o, *codes_of(o.flatten(2)), gated=(block.table[:, :w], at, x.reshape(-1, w)))
    linear(up, block.up, *codes_of(x1))
    down = block.down(up)
    linear(down, block.down, *codes_of(up))
    rx, dx, rh, dh = norms.reference(down, x1, block.after(at))
    norms.within(x2, rx, dx)
    norms.within(h, rh, dh)

    side = torch.cuda.Stream(cuda_device)
    side.wait_stream(torch.cuda.current_stream(cuda_device))
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            again = block.run(*inputs, **keys)
        for t in again:
            t.zero_()
        graph.replay()
        graph.replay()
    side.synchronize()
    for n, (a, c) in enumerate(zip((x, codes, scales, q, kv, turned, o, x1, up, x2, h), again)):
        assert torch.equal(a, c), n
    from xgen_b200.attention import kernel_errors

    assert kernel_errors(cuda_device) == 0
