"""The operators of a conditioned DiT block, their plain forms and the sizes they are measured at.

  rope      rotary positions with several axes (time, height, width), with the Q/K RMSNorm where a model has one
  cross     cross attention to an encoder's states: another length, padded or masked keys, shared heads
  int8      linear layer in 8-bit integers, scales for each token and output channel, with its epilogues
  norms     the norm after a block, its gate and residual, and the norm before the next block

`run` computes the plain form with elementary torch operations in 32 bits (angles in 64), or, where `own` is true, calls the
package's operators. `exact` computes the definitions in 64 bits.
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_TINY = 1.1754943508222875e-38  # the smallest normal 32-bit float: lower bound of a quantisation scale


# ------------------------------------------------------------------ cases
def listed():
    return [
        # Q and K of the whole 768P-5s sequence (31 x 48 x 84 video, 512 text, 1,250 audio tokens), 24 heads: the largest call.
        {"name": "rope_video", "op": "rope", "batch": 1, "seq": 126754, "heads": 24, "kv_heads": 24, "dim": 128, "axes": "32,48,48",
         "dtype": "bf16", "interleaved": False, "norm": False, "fractional": False, "per_sample": False},
        # A batch of two images with their text (odd length), fused QKV projection, Q/K norms, neighbouring channels paired.
        {"name": "rope_image_norm", "op": "rope", "batch": 2, "seq": 4173, "heads": 12, "kv_heads": 12, "dim": 128, "axes": "32,48,48",
         "dtype": "fp16", "interleaved": True, "norm": True, "fractional": True, "per_sample": True},
        # A few tokens of a small model, shared key heads: latency.
        {"name": "rope_tokens", "op": "rope", "batch": 1, "seq": 17, "heads": 12, "kv_heads": 4, "dim": 64, "axes": "16,16,16",
         "dtype": "bf16", "interleaved": False, "norm": True, "fractional": False, "per_sample": False},
        # All video tokens of 768P-5s attend to 512 text states: the largest call.
        {"name": "cross_video", "op": "cross", "batch": 1, "heads": 24, "kv_heads": 24, "seq_q": 124992, "seq_kv": 512, "dim": 128,
         "dtype": "bf16", "mask": "none"},
        # A padded batch: every sample has its own text length, one has none (an unconditional sample).
        {"name": "cross_ragged", "op": "cross", "batch": 4, "heads": 12, "kv_heads": 12, "seq_q": 4096, "seq_kv": 512, "dim": 64,
         "dtype": "fp16", "mask": "lens"},
        # One rank's eighth of the sequence, keys left out by a mask (several prompts in one row of states).
        {"name": "cross_masked", "op": "cross", "batch": 2, "heads": 24, "kv_heads": 24, "seq_q": 15845, "seq_kv": 333, "dim": 128,
         "dtype": "bf16", "mask": "keys"},
        # One query token for each of 4 samples against long encoder states, shared key heads.
        {"name": "cross_token", "op": "cross", "batch": 4, "heads": 24, "kv_heads": 8, "seq_q": 1, "seq_kv": 4099, "dim": 128,
         "dtype": "bf16", "mask": "lens"},
        # FFN up projection with its gate, a long sequence: the largest call, bound by the product.
        {"name": "int8_ffn_swiglu", "op": "int8", "rows": 32769, "in": 4096, "out": 16384, "dtype": "bf16", "epilogue": "swiglu",
         "bias": False},
        # Output projection of the 1536-wide block on 4,352 tokens, with the gated residual that follows it.
        {"name": "int8_out_gated", "op": "int8", "rows": 4352, "in": 1536, "out": 1536, "dtype": "bf16", "epilogue": "gated",
         "bias": True},
        # One token's QKV projection: latency and the weights' bytes.
        {"name": "int8_token", "op": "int8", "rows": 1, "in": 1536, "out": 4608, "dtype": "bf16", "epilogue": "none", "bias": True},
        # A quarter of the 768P-5s sequence at width 5120: the largest call, bound by memory.
        {"name": "norms_video", "op": "norms", "batch": 1, "seq": 31689, "width": 5120, "dtype": "bf16", "post": "rmsnorm",
         "pre": "layernorm", "gate": True, "modulate": True, "quant": "none", "rows": 6},
        # The 1536-wide block on 4,352 tokens for two samples, the second norm straight to 8-bit codes for the next projection.
        {"name": "norms_quant", "op": "norms", "batch": 2, "seq": 4352, "width": 1536, "dtype": "bf16", "post": "rmsnorm",
         "pre": "rmsnorm", "gate": True, "modulate": True, "quant": "int8", "rows": 12},
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over the logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))


def draw(rng):
    op = rng.choice(["rope", "cross", "int8", "norms"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op == "rope":
        dim, axes = rng.choice([(128, "32,48,48"), (128, "32,32,32"), (128, "128"), (64, "16,24,24"), (64, "16,16,16"), (96, "48,48")])
        kv = rng.choice([1, 2, 4, 8, 12])
        heads = kv * rng.choice([1, 1, 2, 3])
        batch = rng.choice([1, 1, 2, 3])
        most = min(126754, 126754 * 48 * 128 // (batch * (heads + kv) * dim))
        dtype = rng.choice([dtype, dtype, "fp32"])
        return {"op": op, "batch": batch, "seq": _spread(rng, 1, most // 2 if dtype == "fp32" else most), "heads": heads, "kv_heads": kv,
                "dim": dim, "axes": axes, "dtype": dtype, "interleaved": rng.random() < 0.4,
                "norm": rng.random() < 0.5, "fractional": rng.random() < 0.3, "per_sample": rng.random() < 0.3}
    if op == "cross":
        kv = rng.choice([1, 2, 4, 8, 12])
        heads = kv * rng.choice([1, 1, 2, 3])
        batch = rng.choice([1, 1, 2, 3, 5])
        dim = rng.choice([64, 128])
        seq_kv = _spread(rng, 1, 8192)
        most = max(1, min(124992, 124992 * 24 * 512 // (batch * heads * max(seq_kv, 128))))
        return {"op": op, "batch": batch, "heads": heads, "kv_heads": kv, "seq_q": _spread(rng, 1, most), "seq_kv": seq_kv, "dim": dim,
                "dtype": dtype, "mask": rng.choice(["none", "lens", "keys"])}
    if op == "int8":
        epilogue = rng.choice(["none", "gelu", "gelu_tanh", "swiglu", "gated"])
        k, n = 16 * _spread(rng, 4, 512), 16 * _spread(rng, 4, 512)
        if epilogue == "swiglu":
            n = 2 * n
        return {"op": op, "rows": _spread(rng, 1, 32769), "in": k, "out": n, "dtype": dtype, "epilogue": epilogue,
                "bias": rng.random() < 0.5}
    width = rng.choice([8 * _spread(rng, 8, 1024), _spread(rng, 33, 2000)])
    batch = rng.choice([1, 1, 2, 3])
    dtype = rng.choice([dtype, dtype, dtype, "fp32"])
    most = min(31689, 31689 * 5120 // (batch * width)) // (2 if dtype == "fp32" else 1)
    return {"op": op, "batch": batch, "seq": _spread(rng, 1, most), "width": width, "dtype": dtype,
            "post": rng.choice(["rmsnorm", "layernorm", "none"]), "pre": rng.choice(["rmsnorm", "layernorm"]),
            "gate": rng.random() < 0.7, "modulate": rng.random() < 0.7, "quant": rng.choice(["none", "none", "int8", "e4m3"]),
            "rows": rng.choice([1, 2, 6, 50])}


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, mean=0.0, out=dtype):
        return (torch.randn(*shape, generator=g, device=dev) * std + mean).to(out)

    def whole(low, high, shape):
        return torch.randint(low, high, shape, generator=g, device=dev)

    state = {"case": case}
    if case["op"] == "rope":
        b, s, h, hk, d = case["batch"], case["seq"], case["heads"], case["kv_heads"], case["dim"]
        axes = tuple(int(a) for a in case["axes"].split(","))
        fused = normal(b, s, (h + 2 * hk) * d)  # the QKV projection's output: Q and K are views of it
        state["query"] = fused[..., :h * d].unflatten(-1, (h, d))
        state["key"] = fused[..., h * d:(h + hk) * d].unflatten(-1, (hk, d))
        shape = (b, s, len(axes)) if case["per_sample"] else (s, len(axes))
        # token positions of a grid walk: the first axis slowest; far positions for long sequences
        edge = max(2, int(round(s ** (1 / len(axes)))))
        at = torch.arange(s, device=dev)
        grid = torch.stack([at // edge ** (len(axes) - 1 - a) % (edge if a else s + 1) for a in range(len(axes))], -1)
        shift = whole(0, 100, shape[:-2] + (1, len(axes))) if len(shape) == 3 else whole(0, 100, (1, len(axes)))
        positions = grid + shift
        if case["fractional"]:
            positions = positions.float() * 0.75 + torch.rand(shape, generator=g, device=dev)
        state["positions"] = positions.contiguous()
        state["axes"] = axes
        state["norms"] = (None, None)
        if case["norm"]:
            norms = []
            for _ in range(2):
                norm = torch.nn.RMSNorm(d, eps=1e-6, device=dev, dtype=dtype)
                norm.weight = torch.nn.Parameter(normal(d, std=0.1, mean=1.0), requires_grad=False)
                norms.append(norm)
            state["norms"] = tuple(norms)
    elif case["op"] == "cross":
        b, h, hk, d = case["batch"], case["heads"], case["kv_heads"], case["dim"]
        state["query"] = normal(b, case["seq_q"], h, d).transpose(1, 2)  # projections give [B, S, H, D]
        kv = normal(b, case["seq_kv"], 2 * hk, d)
        key, value = kv[:, :, :hk], kv[:, :, hk:]
        key += normal(1, 1, hk, d)  # keys have a bias for each channel
        state["kv_lens"] = state["key_mask"] = None
        if case["mask"] != "none":
            lens = whole(0, case["seq_kv"] + 1, (b,))
            lens[0] = case["seq_kv"]
            if b > 1:
                lens[-1] = 0  # a sample without a condition
            valid = torch.arange(case["seq_kv"], device=dev)[None] < lens[:, None]
            if case["mask"] == "keys":
                valid = torch.rand(b, case["seq_kv"], generator=g, device=dev) < 0.7
                state["key_mask"] = valid
            else:
                state["kv_lens"] = lens.to(torch.int32)
            kv.masked_fill_(~valid[:, :, None, None], float("nan"))  # what stands in padded places is never read as a number
        state["key"], state["value"] = key.transpose(1, 2), value.transpose(1, 2)
    elif case["op"] == "int8":
        m, k, n = case["rows"], case["in"], case["out"]
        # activations with a different range for each token and a few large channels, as after an AdaLN prologue
        x = torch.randn(m, k, generator=g, device=dev) * (0.2 + 3 * torch.rand(m, 1, generator=g, device=dev))
        x *= 1 + 9 * (torch.rand(k, generator=g, device=dev) < 0.01)
        state["x"] = x.to(dtype)
        weight = torch.randn(n, k, generator=g, device=dev) * 0.02
        scale = (weight.abs().amax(1) / torch.full((n,), 127.0, device=dev)).clamp_min(_TINY)
        state["weight"] = (weight / scale[:, None]).round().clamp(-127, 127).to(torch.int8)
        state["weight_scale"] = scale
        state["bias"] = normal(n) if case["bias"] else None
        state["gate"] = state["gate_index"] = state["residual"] = None
        if case["epilogue"] == "gated":
            state["gate"] = normal(6, n, std=0.5)
            state["gate_index"] = whole(0, 6, (m,))
            state["residual"] = normal(m, n)
    else:
        b, s, w = case["batch"], case["seq"], case["width"]
        state["branch"], state["residual"] = normal(b, s, w, std=0.7, mean=0.1), normal(b, s, w, std=2.0)
        state["post_weight"] = normal(w, std=0.1, mean=1.0) if case["post"] == "rmsnorm" else None
        state["pre_weight"] = normal(w, std=0.1, mean=1.0) if case["pre"] == "rmsnorm" else None
        table = normal(case["rows"], 3 * w, std=0.3)  # AdaLN rows: gate, scale, shift
        state["gate"] = table[:, :w] if case["gate"] else None
        state["scale"], state["shift"] = (table[:, w:2 * w], table[:, 2 * w:]) if case["modulate"] else (None, None)
        state["indices"] = whole(0, case["rows"], (s,)) if case["gate"] or case["modulate"] else None
    return state


# ------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    with torch.no_grad():
        if case["op"] == "rope":
            return _rope_own(state) if own else _rope(state)
        if case["op"] == "cross":
            return _cross_own(state) if own else _cross(state)
        if case["op"] == "int8":
            return _int8_own(state) if own else _int8(state)
        return _norms_own(state) if own else _norms(state)


def _rope_own(state):
    from xgen_b200.ops import rope_axes

    query, key = rope_axes(state["query"], state["key"], state["positions"], axes=state["axes"],
                           interleaved=state["case"]["interleaved"], norm_q=state["norms"][0], norm_k=state["norms"][1])
    return {"query": query, "key": key}


def _cross_own(state):
    from xgen_b200.attention import cross_attention

    return cross_attention(state["query"], state["key"], state["value"], kv_lens=state["kv_lens"], key_mask=state["key_mask"])


def _int8_own(state):
    from xgen_b200.int8_linear import int8_linear

    epilogue = state["case"]["epilogue"]
    return int8_linear(state["x"], state["weight"], state["weight_scale"], state["bias"],
                       activation=epilogue if epilogue in ("gelu", "gelu_tanh", "swiglu") else None, gate=state["gate"],
                       gate_index=state["gate_index"], residual=state["residual"])


def _norms_own(state):
    from xgen_b200.ops import sandwich_norm

    case = state["case"]
    got = sandwich_norm(state["branch"], state["residual"], post_norm=None if case["post"] == "none" else case["post"],
                        pre_norm=case["pre"], post_weight=state["post_weight"], pre_weight=state["pre_weight"], gate=state["gate"],
                        residual_scale=0.5, scale=state["scale"], shift=state["shift"], indices=state["indices"],
                        quant=None if case["quant"] == "none" else case["quant"])
    if case["quant"] == "none":
        return {"residual": got[0], "normed": got[1]}
    codes, scales = got[1], got[2]
    return {"residual": got[0], "normed": (codes.float() * scales[..., None]).to(got[0].dtype), "scales": scales}


def _rope(state):
    case, axes = state["case"], state["axes"]
    dev, rotary = state["query"].device, sum(axes)
    axis = torch.repeat_interleave(torch.arange(len(axes), device=dev), torch.tensor([d // 2 for d in axes], device=dev))
    angles = state["positions"].double()[..., axis] * torch.pow(torch.tensor(10000.0, device=dev, dtype=torch.float64), -_exponents(axes, dev))
    cos, sin = angles.cos().float().unsqueeze(-2), angles.sin().float().unsqueeze(-2)

    def one(x, norm):
        x = x.float()
        if norm is not None:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + norm.eps) * norm.weight.float()
        turn, rest = x[..., :rotary], x[..., rotary:]
        if case["interleaved"]:
            a, b = turn[..., 0::2], turn[..., 1::2]
            turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
        else:
            a, b = turn[..., :rotary // 2], turn[..., rotary // 2:]
            turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
        return torch.cat((turned, rest), -1).to(state["query"].dtype)

    return {"query": one(state["query"], state["norms"][0]), "key": one(state["key"], state["norms"][1])}


def _exponents(axes, dev):
    """Exponent of theta for each pair: 2 i / d of its axis, in 64 bits."""
    return torch.cat([torch.arange(0, d, 2, device=dev, dtype=torch.float64) / d for d in axes])


def _valid(state):
    case, key = state["case"], state["key"]
    if state["key_mask"] is not None:
        return state["key_mask"]
    at = torch.arange(case["seq_kv"], device=key.device)[None]
    if state["kv_lens"] is not None:
        return at < state["kv_lens"][:, None]
    return (at >= 0).expand(case["batch"], -1)


def _cross(state):
    case, query = state["case"], state["query"]
    b, h, s, d = query.shape
    groups = h // case["kv_heads"]
    valid = _valid(state)
    key = state["key"].float()
    value = state["value"].float().masked_fill(~valid[:, None, :, None], 0.0)
    scores = query.float().unflatten(1, (case["kv_heads"], groups)).flatten(2, 3) @ key.transpose(-1, -2)
    scores = (scores * (1.0 / math.sqrt(d))).masked_fill_(~valid[:, None, None, :], float("-inf"))
    top = scores.amax(-1, keepdim=True)
    scores -= torch.where(top == float("-inf"), torch.zeros_like(top), top)
    scores.exp_()
    total = scores.sum(-1, keepdim=True)
    out = (scores @ value) / torch.where(total == 0, torch.ones_like(total), total)
    return out.view(b, h, s, d).to(query.dtype)


def _int8(state):
    epilogue = state["case"]["epilogue"]
    x = state["x"].float()
    top = x.abs().amax(-1, keepdim=True)
    scale = (top / torch.full_like(top, 127.0)).clamp_min(_TINY)
    codes = (x / scale).round().clamp(-127, 127)
    y = (codes @ state["weight"].float().t()) * (scale * state["weight_scale"])
    if state["bias"] is not None:
        y = y + state["bias"].float()
    if epilogue == "gelu":
        y = 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    elif epilogue == "gelu_tanh":
        y = 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
    elif epilogue == "swiglu":
        gate, value = y.chunk(2, -1)
        y = gate * torch.sigmoid(gate) * value
    elif epilogue == "gated":
        y = state["residual"].float() + state["gate"].float()[state["gate_index"]] * y
    return y.to(state["x"].dtype)


def _norm(x, kind, weight, eps=1e-6):
    if kind == "layernorm":
        x = x - x.mean(-1, keepdim=True)
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)
    return x if weight is None else x * weight.to(x.dtype)


def _norms(state):
    case, at = state["case"], state["indices"]
    y = state["branch"].float()
    if case["post"] != "none":
        y = _norm(y, case["post"], state["post_weight"])
    if state["gate"] is not None:
        y = y * state["gate"].float()[at]
    x = state["residual"].float() + 0.5 * y
    normed = _norm(x, case["pre"], state["pre_weight"])
    if state["scale"] is not None:
        normed = normed * (1 + state["scale"].float()[at]) + state["shift"].float()[at]
    dtype = state["residual"].dtype
    if case["quant"] == "none":
        return {"residual": x.to(dtype), "normed": normed.to(dtype)}
    most = 127.0 if case["quant"] == "int8" else 448.0
    top = normed.abs().amax(-1)
    scales = (top / torch.full_like(top, most)).clamp_min(_TINY)
    codes = (normed / scales[..., None]).clamp(-most, most)
    codes = codes.round() if case["quant"] == "int8" else codes.to(torch.float8_e4m3fn).float()
    return {"residual": x.to(dtype), "normed": (codes * scales[..., None]).to(dtype), "scales": scales}


# ------------------------------------------------------------------ definitions in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return {"rope": _rope64, "cross": _cross64, "int8": _int8_64, "norms": _norms64}[case["op"]](state)


def _rope64(state):
    case, axes = state["case"], state["axes"]
    half = sum(axes) // 2
    found = {}
    for name, norm in (("query", state["norms"][0]), ("key", state["norms"][1])):
        x = state[name].double().clone()
        if norm is not None:
            x /= (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + norm.eps).sqrt()
            x *= norm.weight.double()
        z, first = x.clone(), 0
        for n, d in enumerate(axes):
            for i in range(d // 2):
                angle = state["positions"][..., n].double()[..., None] / 10000.0 ** (2.0 * i / d)
                c, s = torch.cos(angle), torch.sin(angle)
                p = first + i
                left, right = (2 * p, 2 * p + 1) if case["interleaved"] else (p, half + p)
                z[..., left] = x[..., left] * c - x[..., right] * s
                z[..., right] = x[..., left] * s + x[..., right] * c
            first += d // 2
        found[name] = z
    return found


def _cross64(state):
    query, key, value = state["query"], state["key"], state["value"]
    b, h, s, d = query.shape
    group = h // key.shape[1]
    valid = _valid(state)
    out = torch.zeros(b, h, s, d, dtype=torch.float64, device=query.device)
    for n in range(b):
        at = valid[n].nonzero()[:, 0]
        if not len(at):
            continue
        for j in range(h):
            k, v = key[n, j // group, at].double(), value[n, j // group, at].double()
            out[n, j] = torch.softmax(query[n, j].double() @ k.t() / math.sqrt(d), -1) @ v
    return out


def _int8_64(state):
    epilogue, x = state["case"]["epilogue"], state["x"].double()
    scale = (x.abs().amax(-1, keepdim=True) / 127).float().clamp_min(_TINY).double()
    y = torch.round(x / scale) @ state["weight"].double().t() * scale * state["weight_scale"].double()
    if state["bias"] is not None:
        y += state["bias"].double()
    if epilogue == "gelu":
        y = y * torch.special.ndtr(y)
    elif epilogue == "gelu_tanh":
        y = y / 2 * (1 + torch.tanh((2 / math.pi) ** 0.5 * (y + 0.044715 * y ** 3)))
    elif epilogue == "swiglu":
        n = y.shape[-1] // 2
        y = y[:, :n] / (1 + torch.exp(-y[:, :n])) * y[:, n:]
    elif epilogue == "gated":
        y = state["residual"].double() + state["gate"].double().index_select(0, state["gate_index"]) * y
    return y


def _norms64(state):
    case, at = state["case"], state["indices"]

    def norm(x, kind, weight):
        if kind == "layernorm":
            x = x - x.sum(-1, keepdim=True) / x.shape[-1]
        x = x / ((x * x).sum(-1, keepdim=True) / x.shape[-1] + 1e-6).sqrt()
        return x if weight is None else x * weight.double()

    y = state["branch"].double()
    if case["post"] != "none":
        y = norm(y, case["post"], state["post_weight"])
    if state["gate"] is not None:
        y = y * state["gate"].double().index_select(0, at)
    x = state["residual"].double() + y / 2
    h = norm(x, case["pre"], state["pre_weight"])
    if state["scale"] is not None:
        h = h * (1 + state["scale"].double().index_select(0, at)) + state["shift"].double().index_select(0, at)
    if case["quant"] == "none":
        return {"residual": x, "normed": h}
    most = 127.0 if case["quant"] == "int8" else 448.0
    scales = (h.abs().amax(-1) / most).clamp_min(_TINY)
    codes = h / scales[..., None]
    codes = codes.round() if case["quant"] == "int8" else codes.float().to(torch.float8_e4m3fn).double()
    return {"residual": x, "normed": codes * scales[..., None], "scales": scales}


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "rope":
        values = case["batch"] * case["seq"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        positions = case["seq"] * (case["batch"] if case["per_sample"] else 1) * len(case["axes"].split(",")) * (4 if case["fractional"] else 8)
        return {"bytes": 2 * values * size + positions, "flops": values * (7 if case["norm"] else 3)}
    if case["op"] == "cross":
        # about half of the padded places and seven tenths of the masked ones hold a key
        share = {"none": 1.0, "lens": 0.5, "keys": 0.7}[case["mask"]]
        keys = max(1.0, case["batch"] * case["seq_kv"] * share)
        query = case["batch"] * case["heads"] * case["seq_q"] * case["dim"]
        return {"bytes": int(2 * query * size + 2 * keys * case["kv_heads"] * case["dim"] * size),
                "flops": int(4 * keys * case["heads"] * case["seq_q"] * case["dim"])}
    if case["op"] == "int8":
        m, k, n = case["rows"], case["in"], case["out"]
        out = n // 2 if case["epilogue"] == "swiglu" else n
        more = m * n * size + 6 * n * size + 8 * m if case["epilogue"] == "gated" else 0
        return {"bytes": m * k * size + n * k + 4 * n + (n * size if case["bias"] else 0) + m * out * size + more, "flops": 2 * m * n * k}
    values = case["batch"] * case["seq"] * case["width"]
    code = size if case["quant"] == "none" else 1
    return {"bytes": values * (3 * size + code) + 3 * case["rows"] * case["width"] * size, "flops": 20 * values}
