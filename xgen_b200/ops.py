"""torch-facing wrappers of the libxgb.so elementwise and FP8 operators.

Each function mirrors a reference operator (same name where the reference
exposes one, same argument meaning and error behaviour) and runs the
sm_100a kernel on the caller's current CUDA stream. There is no CPU path:
non-CUDA tensors raise ValueError (or return None where the reference's
`try_*` contract does so to select its own eager fallback).
"""
from __future__ import annotations

import functools

import torch
import torch.autograd.forward_ad as _forward_ad
from torch.nn import RMSNorm as _RMSNorm

from . import _lib
from ._lib import call, f64_array, i64_array

_DTYPE_CODE = {torch.bfloat16: _lib.XGB_BF16, torch.float16: _lib.XGB_F16}
_DTYPE_CODE_F32 = {**_DTYPE_CODE, torch.float32: _lib.XGB_F32}
_raw_stream = torch._C._cuda_getCurrentRawStream  # the current stream's handle, without a Stream object
_current_device = torch._C._cuda_getDevice
_I64x3, _I64x4 = _lib.c_i64 * 3, _lib.c_i64 * 4


def _stream(t: torch.Tensor) -> int:
    return torch.cuda.current_stream(t.device).cuda_stream


def _require_cuda(*tensors: torch.Tensor, what: str) -> None:
    for t in tensors:
        if not t.is_cuda:
            raise ValueError(f"{what} requires CUDA tensors")


def _refuse_autograd(what: str, *tensors) -> None:
    """Refuses tensors whose derivatives, of either mode, a call would lose."""
    backward, forward = torch.is_grad_enabled(), _forward_ad._current_level >= 0
    if not (backward or forward):
        return
    for t in tensors:
        if t is not None and backward and t.requires_grad:
            raise ValueError(f"{what} carries no autograd: call it under torch.no_grad()")
        if t is not None and forward and _forward_ad.unpack_dual(t).tangent is not None:
            raise ValueError(f"{what} carries no autograd: its tensors may not have tangents")


def _form(t):
    """Shape, strides, type and device: what the checks of a call go by. They
    are made once for each set of forms (lru_cache) and not again: a third of a
    small call's time on the host."""
    return None if t is None else (t.shape, t.stride(), t.dtype, t.get_device())


def _device_in(what: str, *forms) -> int:
    """Index of the one GPU that all tensors (None: not given) are on."""
    at = {f[3] for f in forms if f is not None}
    if min(at) < 0:
        raise ValueError(f"{what} requires CUDA tensors")
    if len(at) > 1:
        raise ValueError(f"{what} needs its tensors on one device")
    return at.pop()


def _like(t: torch.Tensor) -> torch.Tensor:
    """An empty contiguous tensor of t's shape, type and device."""
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _call_on(index: int, name: str, *args) -> None:
    """call(name, *args, stream) with device `index` current (launches go to
    the current device, whatever their stream) and on its current stream."""
    fn = getattr(_lib.lib(), name)
    if index == _current_device():
        status = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            status = fn(*args, _raw_stream(index))
    if status:
        _lib.check(name, status)


def try_h3_partial_rope(query: torch.Tensor, key: torch.Tensor, cos: torch.Tensor,
                        sin: torch.Tensor):
    """Rotate-half RoPE over the first cos.shape[-1] channels of contiguous
    bf16 Q/K [B, S, H, D]; returns None for inputs the fused kernel does not
    take (the caller then runs its eager RoPE), exactly as
    x_base/x_base/operator/h3_partial_rope.py:32-47."""
    if (torch.is_grad_enabled() or not query.is_cuda or query.dtype != torch.bfloat16
            or query.ndim != 4 or query.shape != key.shape or key.dtype != query.dtype
            or cos.ndim != 2 or cos.shape != sin.shape or cos.shape[0] != query.shape[1]
            or cos.shape[-1] <= 0 or cos.shape[-1] % 2 or cos.shape[-1] > query.shape[-1]
            or cos.dtype != torch.float32 or sin.dtype != torch.float32
            or any(t.device != query.device or not t.is_contiguous()
                   for t in (query, key, cos, sin))):
        return None
    b, s, h, w = query.shape
    q_out, k_out = torch.empty_like(query), torch.empty_like(key)
    call("xgb_partial_rope", query.data_ptr(), key.data_ptr(), cos.data_ptr(), sin.data_ptr(),
         q_out.data_ptr(), k_out.data_ptr(), b, s, h, w, cos.shape[-1], _stream(query))
    return q_out, k_out


def try_h3_qk_rms(query: torch.Tensor, key: torch.Tensor, norm_q, norm_k, rotary_emb=None):
    """Per-head RMSNorm (times weight) of strided bf16 Q/K views [B, S, H, D],
    optionally fused with the partial RoPE; None when unsupported, as
    x_base/x_base/operator/h3_qk_rms.py:48-84."""
    if (torch.is_grad_enabled() or not query.is_cuda or query.ndim != 4 or query.numel() == 0
            or query.shape != key.shape or query.dtype != torch.bfloat16
            or key.dtype != query.dtype or query.stride(-1) != 1 or key.stride(-1) != 1
            or query.device != key.device or type(norm_q) is not torch.nn.RMSNorm
            or type(norm_k) is not torch.nn.RMSNorm or norm_q.eps is None or norm_k.eps is None):
        return None
    b, s, h, w = query.shape
    if w > 256:
        return None
    rotary, cos, sin = 0, None, None
    if rotary_emb is not None:
        cos, sin = rotary_emb
        if (cos.ndim != 2 or cos.shape != sin.shape or cos.shape[0] != s
                or not 0 < cos.shape[-1] <= w or cos.shape[-1] % 2
                or cos.dtype != torch.float32 or sin.dtype != torch.float32
                or any(t.device != query.device or not t.is_contiguous() for t in (cos, sin))):
            return None
        rotary = cos.shape[-1]
    weights = (norm_q.weight, norm_k.weight)
    if any(wt is None or wt.shape != (w,) or wt.dtype != query.dtype
           or wt.device != query.device or not wt.is_contiguous() for wt in weights):
        return None
    q_out = torch.empty(query.shape, device=query.device, dtype=query.dtype)
    k_out = torch.empty_like(q_out)
    call("xgb_qk_rms", query.data_ptr(), i64_array(query.stride()[:3]), key.data_ptr(),
         i64_array(key.stride()[:3]), weights[0].data_ptr(), weights[1].data_ptr(),
         float(norm_q.eps), float(norm_k.eps), cos.data_ptr() if cos is not None else None,
         sin.data_ptr() if sin is not None else None, rotary, q_out.data_ptr(), k_out.data_ptr(),
         b, s, h, w, _stream(query))
    return q_out, k_out


def indexed_affine(x: torch.Tensor, table: torch.Tensor, addend: torch.Tensor,
                   indices: torch.Tensor, *, modulation: bool) -> torch.Tensor:
    """AdaLN modulate (`modulation=True`: x*(1+table[idx]) + addend[idx]) or
    gated residual (`modulation=False`: addend + table[idx]*x) with the
    reference's bf16 rounding after each op; the CUDA branch of `_apply`,
    x_base/x_base/operator/h3_indexed_affine.py:32-49. Raises ValueError for
    layouts that branch does not take."""
    _require_cuda(x, table, addend, indices, what="H3 indexed affine")
    if not (x.ndim == 3 and x.is_contiguous() and indices.is_contiguous() and indices.ndim == 1
            and indices.numel() == x.shape[1] and indices.dtype == torch.int64
            and x.dtype == table.dtype == addend.dtype == torch.bfloat16
            and table.ndim == 2 and table.stride(-1) == 1 and table.shape[-1] == x.shape[-1]
            and (addend.stride(-1) == 1 if modulation else
                 (addend.is_contiguous() and addend.shape == x.shape))):
        raise ValueError("H3 indexed affine requires contiguous bf16 [B,S,H] input, int64 "
                         "indices [S] and row-strided bf16 tables")
    out = torch.empty_like(x)
    b, s, w = x.shape
    call("xgb_indexed_affine", x.data_ptr(), table.data_ptr(), table.stride(0), addend.data_ptr(),
         addend.stride(0) if modulation else 0, indices.data_ptr(), out.data_ptr(), b, s, w,
         int(modulation), _stream(x))
    return out


def gate_first_swiglu(x: torch.Tensor, *, with_amax: bool = False):
    """silu(gate) * value over a packed [..., 2F] bf16 tensor with eager bf16
    rounding; x_base/x_base/operator/h3_swiglu.py:31-41."""
    _require_cuda(x, what="H3 SwiGLU")
    if x.dtype != torch.bfloat16 or x.shape[-1] % 2 or not x.is_contiguous():
        raise ValueError("H3 SwiGLU requires a contiguous bf16 [..., 2F] tensor")
    width = x.shape[-1] // 2
    out = torch.empty((*x.shape[:-1], width), device=x.device, dtype=x.dtype)
    rows = out.numel() // width if width else 0
    amax = torch.zeros((), device=x.device, dtype=torch.float32) if with_amax else None
    call("xgb_swiglu", x.data_ptr(), out.data_ptr(), rows, width,
         amax.data_ptr() if amax is not None else None, _stream(x))
    return (out, amax) if with_amax else out


def quantize_activation(x: torch.Tensor, group=None):
    """Per-tensor dynamic e4m3 (scale = max(amax/448, FLT_MIN)); bit-exact
    with quantize_activation / quantize_per_tensor of
    x_base/x_base/operator/h3_fp8_quant.py:18-25 and h3_fp8.py:9-12. With a
    process group the scale is all-reduced with MAX before packing, so every
    rank of a tensor-parallel group packs with the same scale."""
    _require_cuda(x, what="H3 FP8 quantization")
    if x.dtype not in _DTYPE_CODE:
        raise ValueError("H3 FP8 quantization requires a bf16/fp16 tensor")
    x = x.contiguous()
    out = torch.empty(x.shape, device=x.device, dtype=torch.float8_e4m3fn)
    scale = torch.empty((), device=x.device, dtype=torch.float32)
    n = x.numel()
    if n == 0:
        scale.fill_(torch.finfo(torch.float32).tiny)
        if group is not None:
            import torch.distributed as dist

            dist.all_reduce(scale, op=dist.ReduceOp.MAX, group=group)
        return out, scale
    ws_bytes = _lib.lib().xgb_fp8_quantize_per_tensor_workspace(n)
    ws = torch.empty(max(ws_bytes, 4), device=x.device, dtype=torch.uint8)
    if group is None:
        call("xgb_fp8_quantize_per_tensor", x.data_ptr(), _DTYPE_CODE[x.dtype], n, out.data_ptr(),
             scale.data_ptr(), ws.data_ptr(), ws_bytes, _stream(x))
        return out, scale
    import torch.distributed as dist

    call("xgb_fp8_abs_peak_scale", x.data_ptr(), _DTYPE_CODE[x.dtype], n, scale.data_ptr(),
         ws.data_ptr(), ws_bytes, _stream(x))
    dist.all_reduce(scale, op=dist.ReduceOp.MAX, group=group)
    call("xgb_fp8_quantize_with_scale", x.data_ptr(), _DTYPE_CODE[x.dtype], n, scale.data_ptr(),
         out.data_ptr(), _stream(x))
    return out, scale


def norm_modulate_quant(x: torch.Tensor, norm: str, weight, eps: float, scale: torch.Tensor,
                        shift: torch.Tensor, indices: torch.Tensor, *, return_bf16: bool = False):
    """Fused AdaLN prologue: per-token e4m3 of
    bf16(bf16(norm(x) * bf16(1 + scale[idx])) + shift[idx]) for x [B, S, H]
    (norm "layernorm" without affine or "rmsnorm" x weight); returns
    (codes [B*S, H], scales [B*S]) and, with return_bf16, the modulated bf16."""
    _require_cuda(x, scale, shift, indices, what="H3 norm/modulate")
    if (x.ndim != 3 or x.dtype != torch.bfloat16 or x.stride(-1) != 1 or x.stride(0) != x.shape[1] * x.stride(1)
            or scale.dtype != torch.bfloat16 or shift.dtype != torch.bfloat16
            or scale.stride(-1) != 1 or shift.stride(-1) != 1 or indices.dtype != torch.int64
            or indices.numel() != x.shape[1] or norm not in ("layernorm", "rmsnorm")):
        raise ValueError("norm_modulate_quant needs bf16 [B,S,H] rows, bf16 tables, int64 [S] indices")
    b, s, h = x.shape
    rows = b * s
    codes = torch.empty((rows, h), device=x.device, dtype=torch.float8_e4m3fn)
    scales = torch.empty((rows,), device=x.device, dtype=torch.float32)
    mod = torch.empty((b, s, h), device=x.device, dtype=torch.bfloat16) if return_bf16 else None
    call("xgb_norm_modulate_quant", x.data_ptr(), x.stride(1), rows, h, s,
         1 if norm == "rmsnorm" else 0, weight.data_ptr() if weight is not None else None,
         float(eps), scale.data_ptr(), scale.stride(0), shift.data_ptr(), shift.stride(0),
         indices.contiguous().data_ptr(), codes.data_ptr(), scales.data_ptr(),
         mod.data_ptr() if mod is not None else None, _stream(x))
    return (codes, scales, mod) if return_bf16 else (codes, scales)


def output_adaln(x: torch.Tensor, scale: torch.Tensor, shift: torch.Tensor,
                 indices: torch.Tensor, *, norm: str = "layernorm", weight=None,
                 eps: float = 1e-6, fused: bool = False) -> torch.Tensor:
    """Final-layer output AdaLN of the H3 transformer (`norm_out`,
    x_diffusers/x_diffusers/framework/transformer/minimax_h3.py:672-696):
    bf16(bf16(norm(x) * bf16(1 + scale[idx])) + shift[idx]); scale/shift are
    the [M, H] tables of lookup_final().

    Default: the reference's own LayerNorm followed by the bit-exact
    indexed-affine kernel, bitwise equal to the reference's fused output path
    (x_base/tests/test_h3_output_adaln.py:29-45). fused=True runs norm and
    modulation in one pass (xgb_norm_modulate_quant without the e4m3
    output), whose fp32 statistics can round a value one bf16 ulp apart."""
    _require_cuda(x, scale, shift, indices, what="H3 output AdaLN")
    if (x.ndim != 3 or x.dtype != torch.bfloat16 or x.stride(-1) != 1 or x.stride(0) != x.shape[1] * x.stride(1)
            or scale.dtype != torch.bfloat16 or shift.dtype != torch.bfloat16
            or scale.stride(-1) != 1 or shift.stride(-1) != 1 or indices.dtype != torch.int64
            or indices.numel() != x.shape[1] or norm not in ("layernorm", "rmsnorm")):
        raise ValueError("output_adaln needs bf16 [B,S,H] rows, bf16 tables, int64 [S] indices")
    b, s, h = x.shape
    if not fused:
        if norm == "layernorm":
            n = torch.nn.functional.layer_norm(x, (h,), eps=eps)
        else:
            n = torch.nn.functional.rms_norm(x, (h,), weight, eps=eps)
        return indexed_affine(n, scale, shift, indices, modulation=True)
    out = torch.empty((b, s, h), device=x.device, dtype=torch.bfloat16)
    call("xgb_norm_modulate_quant", x.data_ptr(), x.stride(1), b * s, h, s,
         1 if norm == "rmsnorm" else 0, weight.data_ptr() if weight is not None else None,
         float(eps), scale.data_ptr(), scale.stride(0), shift.data_ptr(), shift.stride(0),
         indices.contiguous().data_ptr(), None, None, out.data_ptr(), _stream(x))
    return out


def quantize_per_token(x: torch.Tensor):
    """Per-row dynamic e4m3 of a 2-D bf16/fp16 matrix: (codes, scales[rows])."""
    _require_cuda(x, what="H3 FP8 quantization")
    if x.dtype not in _DTYPE_CODE or x.ndim != 2 or x.stride(-1) != 1:
        raise ValueError("per-token FP8 quantization requires a row-major 2-D bf16/fp16 matrix")
    rows, cols = x.shape
    out = torch.empty((rows, cols), device=x.device, dtype=torch.float8_e4m3fn)
    scales = torch.empty((rows,), device=x.device, dtype=torch.float32)
    call("xgb_fp8_quantize_per_token", x.data_ptr(), _DTYPE_CODE[x.dtype], rows, cols,
         x.stride(0), out.data_ptr(), scales.data_ptr(), _stream(x))
    return out, scales


_POSITION_CODE = {torch.int32: 0, torch.int64: 1, torch.float32: 2, torch.float64: 3}


def rope_axes(query: torch.Tensor, key: torch.Tensor | None, positions: torch.Tensor, *, axes,
              theta=10000.0, interleaved: bool = False, norm_q=None, norm_k=None):
    """Rotary positions with several axes (time, height, width), taken from
    the positions themselves rather than from a table, and the per-head Q/K
    RMSNorm before them.

    query [B, S, H, D], key [B, S, H', D] (or None): bf16, fp16 or fp32 views
    with unit channel stride, D <= 512. positions [S, A] or [B, S, A]: int32,
    int64, float32 or float64 (grid indices, or fractions of them where a
    model rescales its grid). axes: even channel counts of the A axes, whose
    pairs follow one another; channels behind their sum R pass through.
    theta: one base, or one for each axis. Pair i turns by position *
    theta ** (-2 i / d) within its axis of d channels (angles in 64 bits) and
    is made of channels (i, i + R/2), the convention of the cos/sin tables of
    h3.rope, or of (2i, 2i + 1) with interleaved=True. norm_q / norm_k: the
    torch.nn.RMSNorm modules of a model with Q/K norms, applied first.

    32-bit arithmetic, one rounding at the end (the try_h3_* operators round
    after every step, as the reference does). Fast where D and R are multiples
    of 16 and rows begin on 16 bytes; other forms take about eight times as
    long. Returns contiguous (query, key)."""
    what = "rotary positions"
    w_q, eps_q = _norm_of(norm_q)
    w_k, eps_k = _norm_of(norm_k) if key is not None else (None, 0.0)
    _refuse_autograd(what, query, key, positions, w_q, w_k)
    # numbers, not what they are taken from: a plan goes by its arguments' values
    if type(axes) is not tuple or type(sum(axes)) is not int:
        axes = tuple(map(int, axes))
    theta = tuple(map(float, theta)) if isinstance(theta, (tuple, list)) else float(theta)
    plan = _rope_plan(_form(query), _form(key), _form(positions), axes, theta, _form(w_q), _form(w_k))
    index, q_strides, k_strides, sizes, copy_positions, position_args, rotation = plan
    if copy_positions:
        positions = positions.contiguous()
    q_out = _like(query)
    k_out = k_ptr = k_out_ptr = None
    if key is not None:
        k_out = _like(key)
        k_ptr, k_out_ptr = key.data_ptr(), k_out.data_ptr()
    if sizes is not None:
        _call_on(index, "xgb_rope_axes", query.data_ptr(), q_strides, k_ptr, k_strides, *sizes, positions.data_ptr(),
                 *position_args, *rotation, int(interleaved), w_q.data_ptr() if w_q is not None else None,
                 w_k.data_ptr() if w_k is not None else None, eps_q, eps_k, q_out.data_ptr(), k_out_ptr)
    return q_out, k_out


@functools.lru_cache(maxsize=1024)
def _rope_plan(query, key, positions, axes, theta, w_q, w_k):
    """Checks a rope_axes call by its tensors' forms; the arguments of the C
    call that follow from them (sizes None: nothing to do)."""
    what = "rotary positions"
    index = _device_in(what, query, key, positions, w_q, w_k)
    shape, strides, dtype, _ = query
    code = _DTYPE_CODE_F32.get(dtype)
    if code is None or len(shape) != 4:
        raise ValueError(f"{what} need bf16, fp16 or fp32 queries [B, S, H, D]")
    b, s, h, d = shape
    if strides[3] != 1 and d > 1:
        raise ValueError(f"{what} need views with unit channel stride")
    for w in (w_q, w_k):
        if w is not None and (w[0] != (d,) or w[2] != dtype or (w[1] != (1,) and d > 1)):
            raise ValueError(f"{what}: norms must be torch.nn.RMSNorm over the head dim with a weight of the query's type")
    thetas = theta if isinstance(theta, tuple) else (theta,) * len(axes)
    if not axes or any(a <= 0 or a % 2 for a in axes) or len(thetas) != len(axes) or not all(
            0 < t < float("inf") for t in thetas):
        raise ValueError(f"{what} need positive even axis channels and a positive theta for each axis")
    if sum(axes) > d:
        raise ValueError(f"{what} need axis channels within the head dim")
    p_shape, p_strides, p_type, _ = positions
    n = len(axes)
    at = _POSITION_CODE.get(p_type)
    if at is None or not (p_shape == (s, n) or p_shape == (b, s, n)):
        raise ValueError(f"{what}: positions must be integers or 32/64-bit floats of shape [S, A] or [B, S, A]")
    copy = n > 1 and p_strides[-1] != 1
    if copy:
        p_strides = (s * n, n, 1)[-len(p_shape):]
    kh, k_strides = 0, None
    if key is not None:
        if len(key[0]) != 4 or key[2] != dtype or (key[1][3] != 1 and d > 1):
            raise ValueError(f"{what} need [B, S, H, D] views of one type with unit channel stride")
        kb, ks, kh, kd = key[0]
        if kb != b or ks != s or kd != d:
            raise ValueError(f"{what}: query and key differ in batch, sequence or head dim")
        k_strides = _I64x4(*key[1])
    empty = not b * s * d or not h or (key is not None and not kh)
    if empty and b * s * d and (h or kh):
        raise ValueError(f"{what} need at least one head of query and key")
    return (index, _I64x4(*strides), k_strides, None if empty else (code, b, s, h, kh, d), copy,
            (at, p_strides[0] if len(p_shape) == 3 else 0, p_strides[-2]), (n, i64_array(axes), f64_array(thetas)))


def _norm_of(norm):
    """(weight, eps) of a Q/K norm module, (None, 0) without one. A module that
    names no eps takes the epsilon of the type it computes in, which for all
    three types is fp32."""
    if norm is None:
        return None, 0.0
    weight = norm.weight if type(norm) is _RMSNorm else None
    if weight is None:
        raise ValueError("rotary positions: norms must be torch.nn.RMSNorm with a weight")
    eps = norm.eps
    return weight, eps if eps is not None else torch.finfo(torch.float32).eps


_NORM_CODE = {None: 0, "layernorm": 1, "rmsnorm": 2}
_QUANT_CODE = {None: (0, None), "int8": (1, torch.int8), "e4m3": (2, torch.float8_e4m3fn)}


def sandwich_norm(branch: torch.Tensor, residual: torch.Tensor, *, post_norm: str | None = "rmsnorm",
                  pre_norm: str | None = "rmsnorm", post_weight=None, pre_weight=None, eps: float = 1e-6,
                  gate=None, residual_scale: float = 1.0, scale=None, shift=None, indices=None,
                  quant: str | None = None):
    """The norm after a block, its gate and residual, and the norm and
    modulation before the next block, in one pass:

        x = residual + residual_scale * gate[idx] * post(branch)
        h = pre(x) * (1 + scale[idx]) + shift[idx]

    branch, residual [B, S, W]: bf16, fp16 or fp32 views of one type with unit
    channel stride, W <= 16384. post_norm / pre_norm: "layernorm", "rmsnorm" or
    None, times an optional weight [W]; pre_norm=None returns x alone. gate,
    scale, shift: rows [M, W] of AdaLN tables (row-strided views; scale and
    shift come together); indices: int64 [S], shared by the batch, or [B, S];
    an index outside the tables makes its row NaN. Returns (x, h), or with
    quant="int8" / "e4m3" (x, codes, scales [B, S]): the per-token codes that
    int8_linear_quantized / H3FP8Linear.forward_quantized take.

    32-bit arithmetic; x and h are rounded once each, h from the x before its
    rounding. Codes of fp32 rows are taken in 64 bits, and so are the
    definition's: in 32 bits a few of a million would fall on the other side of
    a border between two codes, as they do for 16-bit rows, whose own rounding
    is larger. Fast where W is a multiple of 8 and rows, weights and table rows
    begin on 16 bytes; other forms take four times as long or more (fp32 rows
    with codes have one form)."""
    what = "sandwich norm"
    _refuse_autograd(what, branch, residual, post_weight, pre_weight, gate, scale, shift)
    plan = _sandwich_plan(_form(branch), _form(residual), post_norm, pre_norm, _form(post_weight), _form(pre_weight), _form(gate),
                          _form(scale), _form(shift), _form(indices), quant)
    index, y_strides, x_strides, sizes, norms, strides, index_batch, table_rows, quant_code, code_type = plan
    if indices is not None:
        indices = indices.contiguous()
    x_out = _like(branch)
    h_out = codes = scales = None
    if quant_code:
        codes = branch.new_empty(branch.shape, dtype=code_type)
        scales = branch.new_empty(branch.shape[:2], dtype=torch.float32)
    elif pre_norm is not None:
        h_out = _like(branch)
    if sizes is not None:
        _call_on(index, "xgb_sandwich_norm", branch.data_ptr(), y_strides, residual.data_ptr(), x_strides, *sizes, norms[0],
                 _ptr(post_weight), norms[1], _ptr(pre_weight), eps, _ptr(gate), strides[0], residual_scale, _ptr(scale),
                 strides[1], _ptr(shift), strides[2], _ptr(indices), index_batch, table_rows, x_out.data_ptr(), _ptr(h_out),
                 quant_code, _ptr(codes), _ptr(scales))
    if pre_norm is None:
        return x_out
    return (x_out, codes, scales) if quant_code else (x_out, h_out)


@functools.lru_cache(maxsize=1024)
def _sandwich_plan(branch, residual, post_norm, pre_norm, post_weight, pre_weight, gate, scale, shift, indices, quant):
    """Checks a sandwich_norm call by its tensors' forms; the arguments of the
    C call that follow from them (sizes None: nothing to do)."""
    what = "sandwich norm"
    index = _device_in(what, branch, residual, post_weight, pre_weight, gate, scale, shift, indices)
    shape, bs, dtype, _ = branch
    code = _DTYPE_CODE_F32.get(dtype)
    if code is None or len(shape) != 3 or shape != residual[0] or residual[2] != dtype:
        raise ValueError(f"{what} needs [B, S, W] branch and residual of one 16- or 32-bit float type")
    b, s, w = shape
    rs = residual[1]
    if (bs[2] != 1 or rs[2] != 1) and w > 1:
        raise ValueError(f"{what} needs views with unit channel stride")
    if w > 16384 or w == 0:
        raise ValueError(f"{what} takes rows of 1 to 16384 channels")
    if post_norm not in _NORM_CODE or pre_norm not in _NORM_CODE or quant not in _QUANT_CODE:
        raise ValueError(f"{what}: norms are 'layernorm', 'rmsnorm' or None, quant 'int8', 'e4m3' or None")
    if (scale is None) != (shift is None):
        raise ValueError(f"{what} needs scale and shift together")
    if pre_norm is None and (quant is not None or scale is not None or pre_weight is not None):
        raise ValueError(f"{what} without a norm before the next block has no modulation and no codes")
    if post_norm is None and post_weight is not None:
        raise ValueError(f"{what} without a norm after the block has no weight for it")
    for t in (post_weight, pre_weight):
        if t is not None and (t[0] != (w,) or t[2] != dtype or (t[1] != (1,) and w > 1)):
            raise ValueError(f"{what}: weights must be contiguous [W] of the branch's type")
    table_rows, strides = 0, []
    for t in (gate, scale, shift):
        if t is not None:
            table_rows = table_rows or (t[0][0] if len(t[0]) == 2 else 0)
            if t[0] != (table_rows, w) or t[2] != dtype or (t[1][1] != 1 and w > 1) or not table_rows:
                raise ValueError(f"{what}: gate, scale and shift must be [M, W] rows of the branch's type")
        # one row is never stepped over
        strides.append(0 if t is None else t[1][0] if table_rows > 1 else w)
    if (table_rows > 0) != (indices is not None):
        raise ValueError(f"{what}: indices come with gate or scale and shift")
    if indices is not None and (indices[2] != torch.int64 or not (indices[0] == (s,) or indices[0] == (b, s))):
        raise ValueError(f"{what}: indices must be int64 [S] or [B, S]")
    return (index, _I64x3(*bs), _I64x3(*rs), (code, b, s, w) if b * s else None, (_NORM_CODE[post_norm], _NORM_CODE[pre_norm]), strides,
            s if indices is not None and len(indices[0]) == 2 else 0, table_rows, *_QUANT_CODE[quant])


def _ptr(t):
    return t.data_ptr() if t is not None else None


def quantize_per_token_int8(x: torch.Tensor):
    """Per-row dynamic int8 of a bf16/fp16 matrix (rows may be strided):
    (codes, scales[rows]) with scale = max(amax/127, FLT_MIN) and codes the
    nearest integers to x / scale, ties to even."""
    what = "H3 INT8 quantization"
    index = _device_in(what, _form(x))
    _refuse_autograd(what, x)
    if x.dtype not in _DTYPE_CODE or x.ndim != 2 or (x.stride(-1) != 1 and x.shape[1] > 1) or x.shape[1] == 0 or (
            x.shape[0] > 1 and x.stride(0) < x.shape[1]):
        raise ValueError(f"{what} requires a row-major 2-D bf16/fp16 matrix")
    rows, cols = x.shape
    out = torch.empty((rows, cols), device=x.device, dtype=torch.int8)
    scales = torch.empty((rows,), device=x.device, dtype=torch.float32)
    if rows:
        _call_on(index, "xgb_int8_quantize_per_token", x.data_ptr(), _DTYPE_CODE[x.dtype], rows, cols, x.stride(0),
                 out.data_ptr(), scales.data_ptr())
    return out, scales
