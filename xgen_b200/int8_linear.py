"""Linear layers in 8-bit integers on the B200 tcgen05 GEMM.

`H3Int8Linear` is H3FP8Linear's counterpart for models whose weights are
stored as int8 with one scale for each output channel: activations get one
dynamic scale for each token, products are summed exactly in 32-bit integers,
and the epilogue (scales, bias, GELU, gate-first SwiGLU, or the AdaLN gate and
residual) runs in 32 bits with one rounding to the input's type. `int8_linear`
and `int8_linear_quantized` are the same on a caller's own tensors.
"""
from __future__ import annotations

import torch
from torch import nn

from ._lib import lib
from .attention import _err_ptr
from .ops import _DTYPE_CODE, _call_on, _device_of, _refuse_autograd, _row_stride

ACTIVATIONS = {None: 0, "gelu": 1, "gelu_tanh": 2, "swiglu": 3}
MAX_IN_FEATURES = 131056  # sums of 128 * 128 * K stay within 32-bit integers


def quantize_per_channel_int8(value: torch.Tensor):
    """Per-row (output channel) int8 of a [out, in] weight on its own device:
    (codes, fp32 scales), scale = max(amax/127, FLT_MIN)."""
    amax = value.float().abs().amax(dim=1)
    scale = (amax / torch.full_like(amax, 127.0)).clamp_min(torch.finfo(torch.float32).tiny)
    return (value.float() / scale[:, None]).round().clamp(-127, 127).to(torch.int8), scale


def _arguments(lead, dtype, weight, weight_scale, bias, activation, gate, gate_index, residual):
    """Checks what int8_linear and int8_linear_quantized share; `lead` is the
    input's shape without its channels. Returns (rows, weight, weight_scale,
    arguments of the epilogue, output)."""
    what = "H3 INT8 Linear"
    if weight.dtype != torch.int8 or weight.ndim != 2 or dtype not in _DTYPE_CODE:
        raise ValueError(f"{what} requires an int8 [out, in] weight and a bf16/fp16 result")
    n, k = weight.shape
    if n % 16 or k % 16 or not n or not k or k > MAX_IN_FEATURES:
        raise ValueError(f"{what} requires projection dimensions divisible by 16 (in <= {MAX_IN_FEATURES})")
    if weight_scale.dtype != torch.float32 or weight_scale.shape != (n,):
        raise ValueError(f"{what} requires an fp32 scale for each output channel")
    code = ACTIVATIONS.get(activation, -1)
    if code < 0:
        raise ValueError(f"Unknown {what} activation: {activation}")
    width = n // 2 if code == 3 else n
    if bias is not None:
        if bias.shape != (n,) or bias.dtype != dtype:
            raise ValueError(f"{what} requires a bias [out] of the result's type")
        bias = bias.contiguous()
    m = lead.numel()
    ldg = ldr = rows = index_rows = 0
    if gate is not None or gate_index is not None or residual is not None:
        if gate is None or gate_index is None or residual is None or code:
            raise ValueError(f"gated {what} needs gate rows, their index and a residual, and no activation")
        if (gate.ndim != 2 or gate.shape[1] != n or gate.shape[0] == 0 or gate.dtype != dtype or gate.stride(1) != 1
                or residual.dtype != dtype or residual.shape != (*lead, n) or residual.stride(-1) != 1):
            raise ValueError(f"gated {what} needs [M, out] gate rows and a residual of the result's shape and type")
        index_rows = gate_index.numel()
        if gate_index.dtype != torch.int64 or (m and (index_rows == 0 or m % index_rows)):
            raise ValueError(f"gated {what} needs an int64 index for each token, or one sequence's for every sample")
        gate_index = gate_index.contiguous()
        rows, residual = gate.shape[0], residual if residual.ndim == 2 else residual.reshape(m, n)
        if rows > 1 and gate.stride(0) < n:  # broadcast rows
            gate = gate.contiguous()
        if m > 1 and residual.stride(0) < n:
            residual = residual.contiguous()
        ldg, ldr = _row_stride(gate, n), residual.stride(0) if m > 1 else n
    out = weight.new_empty((*lead, width), dtype=dtype)
    epilogue = (_DTYPE_CODE[dtype], bias, code, out, width, gate, ldg, gate_index, index_rows, rows, residual, ldr)
    # (tensors that a view or copy above made live on in `epilogue`)
    return m, weight.contiguous(), weight_scale.contiguous(), epilogue, out


def _pointers(e):
    """The epilogue's arguments with its tensors as addresses."""
    dtype, bias, code, out, width, gate, ldg, index, index_rows, rows, residual, ldr = e
    return (dtype, bias.data_ptr() if bias is not None else None, code, out.data_ptr(), width,
            *((gate.data_ptr(), ldg, index.data_ptr(), index_rows, rows, residual.data_ptr(), ldr) if gate is not None else
              (None, 0, None, 0, 0, None, 0)))


def int8_linear_quantized(codes: torch.Tensor, scales: torch.Tensor, weight: torch.Tensor,
                          weight_scale: torch.Tensor, bias=None, *, activation: str | None = None, gate=None,
                          gate_index=None, residual=None, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """int8_linear on activations that are already int8: codes [..., in] and
    scales [...] (quantize_per_token_int8, or sandwich_norm with
    quant="int8"). dtype: bf16 or fp16, the type of the result and of bias,
    gate and residual."""
    what = "H3 INT8 Linear"
    index = _device_of(what, codes, scales, weight, weight_scale, bias, gate, gate_index, residual)
    _refuse_autograd(what, scales, weight_scale, bias, gate, residual)
    if codes.dtype != torch.int8 or codes.ndim < 1 or weight.ndim != 2 or codes.shape[-1] != weight.shape[1]:
        raise ValueError(f"{what} requires int8 codes of its weight's width")
    lead = codes.shape[:-1]
    if scales.dtype != torch.float32 or scales.shape != lead:
        raise ValueError(f"{what} requires an fp32 scale for each row of codes")
    m, weight, weight_scale, epilogue, out = _arguments(lead, dtype, weight, weight_scale, bias, activation, gate, gate_index,
                                                        residual)
    n, k = weight.shape
    if m:
        flat, scales = codes.reshape(m, k).contiguous(), scales.reshape(m).contiguous()
        _call_on(index, "xgb_int8_gemm", flat.data_ptr(), weight.data_ptr(), m, n, k, scales.data_ptr(), weight_scale.data_ptr(),
                 *_pointers(epilogue), _err_ptr(index))
    return out


def int8_linear(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, bias=None, *,
                activation: str | None = None, gate=None, gate_index=None, residual=None) -> torch.Tensor:
    """y = x W^T + bias in 8-bit integers for x [..., in] bf16/fp16, an int8
    weight [out, in] and its fp32 scales [out]; then, in the epilogue,

        activation "gelu" (erf), "gelu_tanh", or "swiglu": silu(first half of
        the output channels) * second half, out/2 columns; or
        residual + gate[gate_index] * y: gate [M, out] AdaLN rows, gate_index
        int64 for each token or for one sequence of a batch (an index outside
        the rows makes its token NaN), residual [..., out].

    Each token's largest magnitude becomes 127; sums are exact, one rounding."""
    what = "H3 INT8 Linear"
    index = _device_of(what, x, weight, weight_scale, bias, gate, gate_index, residual)
    _refuse_autograd(what, x, weight_scale, bias, gate, residual)
    if x.dtype not in _DTYPE_CODE or x.ndim < 1 or weight.ndim != 2 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"{what} requires BF16/FP16 input of its weight's width")
    lead = x.shape[:-1]
    m, weight, weight_scale, epilogue, out = _arguments(lead, x.dtype, weight, weight_scale, bias, activation, gate, gate_index,
                                                        residual)
    n, k = weight.shape
    if m:
        matrix = x if x.ndim == 2 else x.reshape(m, k)
        ldx, unit = matrix.stride()
        if unit != 1 or (m > 1 and ldx < k):
            matrix = matrix.contiguous()
            ldx = k
        ptr = matrix.data_ptr()
        ws_bytes = lib().xgb_int8_linear_workspace(ptr, ldx, m, k)
        ws = x.new_empty((ws_bytes,), dtype=torch.uint8) if ws_bytes else None
        _call_on(index, "xgb_int8_linear", ptr, ldx, weight.data_ptr(), m, n, k, weight_scale.data_ptr(), *_pointers(epilogue),
                 ws.data_ptr() if ws_bytes else None, ws_bytes, _err_ptr(index))
    return out


class H3Int8Linear(nn.Module):
    """Keep int8 weights; quantise activations to int8 on every call.

    activation: fused into every forward ("gelu", "gelu_tanh", or "swiglu" on
    a gate-first [gate | value] projection)."""

    def __init__(self, weight: torch.Tensor, bias: torch.Tensor | None = None, activation: str | None = None):
        super().__init__()
        if weight.ndim != 2 or weight.shape[0] % 16 or weight.shape[1] % 16:
            raise ValueError("H3 INT8 requires projection dimensions divisible by 16")
        codes, scale = quantize_per_channel_int8(weight.detach())
        self._attach(codes, scale, bias, activation)

    @classmethod
    def from_packed(cls, weight, scale, bias=None, activation: str | None = None):
        """Reuse int8 codes [out, in] and their fp32 scales [out]."""
        if weight.dtype != torch.int8 or weight.ndim != 2 or any(n % 16 for n in weight.shape):
            raise ValueError("Packed H3 INT8 projection requires an aligned int8 matrix")
        if scale.shape != (weight.shape[0],) or scale.dtype != torch.float32:
            raise ValueError("Packed H3 INT8 projection requires one FP32 scale for each output channel")
        result = cls.__new__(cls)
        nn.Module.__init__(result)
        result._attach(weight, scale.detach().clone(), bias, activation)
        return result

    def _attach(self, codes, scale, bias, activation):
        if activation not in ACTIVATIONS:
            raise ValueError(f"Unknown H3 INT8 Linear activation: {activation}")
        if activation == "swiglu" and codes.shape[0] % 2:
            raise ValueError("SwiGLU needs an even number of output channels")
        self.out_features, self.in_features = codes.shape
        self.activation = activation
        self.register_buffer("weight", codes.contiguous())
        self.register_buffer("weight_scale", scale)
        self.register_buffer("bias", bias.detach().clone() if bias is not None else None)
        self.calls = 0

    def _bias(self, dtype):
        return self.bias.to(dtype) if self.bias is not None else None

    def forward(self, x):
        out = int8_linear(x, self.weight, self.weight_scale, self._bias(x.dtype), activation=self.activation)
        self.calls += 1
        return out

    def forward_gated(self, x, gate_table, gate_index, residual):
        """residual + gate_table[gate_index] * self(x) in one GEMM."""
        out = int8_linear(x, self.weight, self.weight_scale, self._bias(x.dtype), activation=self.activation,
                          gate=gate_table, gate_index=gate_index, residual=residual)
        self.calls += 1
        return out

    def forward_quantized(self, codes, scales, gated=None, dtype: torch.dtype = torch.bfloat16):
        """The projection of activations that are already int8 codes [..., in]
        with scales [...]; gated: (gate_table, gate_index, residual)."""
        gate, index, residual = gated if gated is not None else (None, None, None)
        out = int8_linear_quantized(codes, scales, self.weight, self.weight_scale, self._bias(dtype),
                                    activation=self.activation, gate=gate, gate_index=index, residual=residual, dtype=dtype)
        self.calls += 1
        return out
