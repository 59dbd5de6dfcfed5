"""Linear layers in 8-bit integers on the B200 tcgen05 GEMM.

`H3Int8Linear` is H3FP8Linear's counterpart for models whose weights are
stored as int8 with one scale for each output channel: activations get one
dynamic scale for each token, products are summed exactly in 32-bit integers,
and the epilogue (scales, bias, GELU, gate-first SwiGLU, or the AdaLN gate and
residual) runs in 32 bits with one rounding to the input's type. `int8_linear`
and `int8_linear_quantized` are the same on a caller's own tensors.
"""
from __future__ import annotations

import functools
import math

import torch
from torch import nn

from ._lib import lib
from .attention import _err_ptr
from .ops import _DTYPE_CODE, _call_on, _device_in, _form, _refuse_autograd

ACTIVATIONS = {None: 0, "gelu": 1, "gelu_tanh": 2, "swiglu": 3}
MAX_IN_FEATURES = 131056  # sums of 128 * 128 * K stay within 32-bit integers


def quantize_per_channel_int8(value: torch.Tensor):
    """Per-row (output channel) int8 of a [out, in] weight on its own device:
    (codes, fp32 scales), scale = max(amax/127, FLT_MIN)."""
    amax = value.float().abs().amax(dim=1)
    scale = (amax / torch.full_like(amax, 127.0)).clamp_min(torch.finfo(torch.float32).tiny)
    return (value.float() / scale[:, None]).round().clamp(-127, 127).to(torch.int8), scale


def _one_for_each(index, lead) -> bool:
    """Whether an index of this shape names rows for tokens of shape `lead`: one
    for each token, in their shape or flat, or one for each place of their
    trailing dimensions, repeated before them (dimensions of one may lead)."""
    if index == (math.prod(lead),):
        return True
    while index and index[0] == 1:
        index = index[1:]
    return index == lead[len(lead) - len(index):]


@functools.lru_cache(maxsize=1024)
def _plan(x, lead, dtype, scales, weight, weight_scale, bias, activation, gate, gate_index, residual):
    """Checks what int8_linear and int8_linear_quantized share by the tensors'
    forms; `lead` is the input's shape without its channels. Returns the rows,
    channels, the C call's numbers and what has to be copied first, the device."""
    what = "H3 INT8 Linear"
    index = _device_in(what, x, scales, weight, weight_scale, bias, gate, gate_index, residual)
    if weight[2] != torch.int8 or len(weight[0]) != 2 or dtype not in _DTYPE_CODE:
        raise ValueError(f"{what} requires an int8 [out, in] weight and a bf16/fp16 result")
    n, k = weight[0]
    if n % 16 or k % 16 or not n or not k or k > MAX_IN_FEATURES:
        raise ValueError(f"{what} requires projection dimensions divisible by 16 (in <= {MAX_IN_FEATURES})")
    if weight_scale[2] != torch.float32 or weight_scale[0] != (n,):
        raise ValueError(f"{what} requires an fp32 scale for each output channel")
    code = ACTIVATIONS.get(activation, -1)
    if code < 0:
        raise ValueError(f"Unknown {what} activation: {activation}")
    width = n // 2 if code == 3 else n
    if bias is not None and (bias[0] != (n,) or bias[2] != dtype):
        raise ValueError(f"{what} requires a bias [out] of the result's type")
    m = math.prod(lead)
    ldg = ldr = rows = index_rows = 0
    copy_gate = copy_residual = False
    if gate is not None or gate_index is not None or residual is not None:
        if gate is None or gate_index is None or residual is None or code:
            raise ValueError(f"gated {what} needs gate rows, their index and a residual, and no activation")
        if (len(gate[0]) != 2 or gate[0][1] != n or gate[0][0] == 0 or gate[2] != dtype or gate[1][1] != 1
                or residual[2] != dtype or residual[0] != (*lead, n) or residual[1][-1] != 1):
            raise ValueError(f"gated {what} needs [M, out] gate rows and a residual of the result's shape and type")
        index_rows = math.prod(gate_index[0])
        if gate_index[2] != torch.int64 or not _one_for_each(tuple(gate_index[0]), tuple(lead)):
            raise ValueError(f"gated {what} needs an int64 index for each token, or one sequence's for every sample")
        rows = gate[0][0]
        copy_gate = rows > 1 and gate[1][0] < n  # broadcast rows
        ldg = gate[1][0] if rows > 1 and not copy_gate else n
        # rows of the residual a stride apart
        copy_residual = len(lead) != 1 or (m > 1 and residual[1][0] < n)
        ldr = residual[1][0] if m > 1 and not copy_residual else n
    return (m, n, k, (*lead, width), (_DTYPE_CODE[dtype], code, width), (ldg, index_rows, rows, ldr), copy_gate, copy_residual, index)


@functools.lru_cache(maxsize=1024)
def _workspace(offset, ldx, m, k):
    """Bytes for an input that starts `offset` bytes behind a 16-byte boundary."""
    return lib().xgb_int8_linear_workspace(16 + offset, ldx, m, k)


def _epilogue(plan, out, bias, gate, gate_index, residual):
    """The C call's arguments behind the scales, and the tensors that a copy
    made: they live until the call has been queued."""
    m, n, _, _, (dtype_code, code, width), (ldg, index_rows, rows, ldr), copy_gate, copy_residual, _ = plan
    if bias is not None:
        bias = bias.contiguous()
    head = (dtype_code, bias.data_ptr() if bias is not None else None, code, out.data_ptr(), width)
    if gate is None:
        return (*head, None, 0, None, 0, 0, None, 0), bias
    gate_index = gate_index.contiguous()
    if copy_gate:
        gate = gate.contiguous()
    if copy_residual:
        residual = residual.reshape(m, n)
        if m > 1 and (residual.stride(0) < n or residual.stride(1) != 1):
            residual = residual.contiguous()
        ldr = residual.stride(0) if m > 1 else n
    return ((*head, gate.data_ptr(), ldg, gate_index.data_ptr(), index_rows, rows, residual.data_ptr(), ldr),
            (bias, gate, gate_index, residual))


def int8_linear_quantized(codes: torch.Tensor, scales: torch.Tensor, weight: torch.Tensor,
                          weight_scale: torch.Tensor, bias=None, *, activation: str | None = None, gate=None,
                          gate_index=None, residual=None, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """int8_linear on activations that are already int8: codes [..., in] and
    scales [...] (quantize_per_token_int8, or sandwich_norm with
    quant="int8"). dtype: bf16 or fp16, the type of the result and of bias,
    gate and residual."""
    what = "H3 INT8 Linear"
    _refuse_autograd(what, scales, weight_scale, bias, gate, residual)
    if codes.dtype != torch.int8 or codes.ndim < 1 or weight.ndim != 2 or codes.shape[-1] != weight.shape[1]:
        raise ValueError(f"{what} requires int8 codes of its weight's width")
    lead = codes.shape[:-1]
    if scales.dtype != torch.float32 or scales.shape != lead:
        raise ValueError(f"{what} requires an fp32 scale for each row of codes")
    plan = _plan(_form(codes), lead, dtype, _form(scales), _form(weight), _form(weight_scale), _form(bias), activation, _form(gate), _form(gate_index),
                 _form(residual))
    m, n, k, index = *plan[:3], plan[-1]
    out = weight.new_empty(plan[3], dtype=dtype)
    epilogue, _held = _epilogue(plan, out, bias, gate, gate_index, residual)
    if m:
        weight, weight_scale = weight.contiguous(), weight_scale.contiguous()
        flat, scales = codes.reshape(m, k).contiguous(), scales.reshape(m).contiguous()
        _call_on(index, "xgb_int8_gemm", flat.data_ptr(), weight.data_ptr(), m, n, k, scales.data_ptr(), weight_scale.data_ptr(),
                 *epilogue, _err_ptr(index))
    return out


def int8_linear(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, bias=None, *,
                activation: str | None = None, gate=None, gate_index=None, residual=None) -> torch.Tensor:
    """y = x W^T + bias in 8-bit integers for x [..., in] bf16/fp16, an int8
    weight [out, in] and its fp32 scales [out]; then, in the epilogue,

        activation "gelu" (erf), "gelu_tanh", or "swiglu": silu(first half of
        the output channels) * second half, out/2 columns; or
        residual + gate[gate_index] * y: gate [M, out] AdaLN rows, gate_index
        int64 for each token (of x's shape without its channels, or flat) or for
        its trailing dimensions, [S] of [B, S, in] for one sequence of a batch
        (an index outside the rows makes its token NaN), residual [..., out].

    Each token's largest magnitude becomes 127; sums are exact, one rounding."""
    what = "H3 INT8 Linear"
    _refuse_autograd(what, x, weight_scale, bias, gate, residual)
    dtype, shape = x.dtype, x.shape
    if dtype not in _DTYPE_CODE or not shape or weight.ndim != 2 or shape[-1] != weight.shape[1]:
        raise ValueError(f"{what} requires BF16/FP16 input of its weight's width")
    plan = _plan(_form(x), shape[:-1], dtype, None, _form(weight), _form(weight_scale), _form(bias), activation, _form(gate), _form(gate_index),
                 _form(residual))
    m, n, k, index = *plan[:3], plan[-1]
    out = x.new_empty(plan[3])
    epilogue, _held = _epilogue(plan, out, bias, gate, gate_index, residual)
    if m:
        weight, weight_scale = weight.contiguous(), weight_scale.contiguous()
        matrix = x if len(shape) == 2 else x.reshape(m, k)
        ldx, unit = matrix.stride()
        if unit != 1 or (m > 1 and ldx < k):
            matrix = matrix.contiguous()
            ldx = k
        ptr = matrix.data_ptr()
        ws_bytes = _workspace(ptr % 16, ldx, m, k)
        ws = x.new_empty((ws_bytes,), dtype=torch.uint8) if ws_bytes else None
        _call_on(index, "xgb_int8_linear", ptr, ldx, weight.data_ptr(), m, n, k, weight_scale.data_ptr(), *epilogue,
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
