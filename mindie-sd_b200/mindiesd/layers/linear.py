"""`linear_forward`: the projections and feed-forward layers around an attention call, with what follows the
product done in its epilogue -- bias, activation, the per-sample gate of a modulated block and the residual
addition.  Operands are bf16 or fp16, or e4m3 with their scales (`token_quant_preprocess`,
`add_rms_norm_quant`); the reference leaves the first to torch.nn.Linear and the second to the quantised
layers of mindiesd/quantization/layer.py of MindIE-SD.

Inference only: there is no backward pass and no forward-mode derivative, so tensors that require gradients are
refused while gradients are recorded, and so are tensors that carry a tangent.
"""
import torch

from . import _custom_ops  # noqa: F401  (registers the fake implementations)
from .norm import refuse_gradients
from .._cabi import ACTIVATIONS
from ..utils.exception import ParametersInvalid
from ..utils.status import checked

_op = torch.ops.mindiesd.linear_fwd.default
_FLOATS = (torch.bfloat16, torch.float16, torch.float32)


def _want(ok, message):
    if not ok:
        raise ParametersInvalid(message)


def _check_optional(name, t, x):
    _want(isinstance(t, torch.Tensor), f"The data type of input {name} must be torch.Tensor, but got {type(t)}.")
    _want(t.device == x.device, f"The input {name} must be on {x.device}, but it is on {t.device}.")


def _explain(x, weight, bias, activation, residual, gate, x_scale, weight_scale, out_dtype):
    """Raises ParametersInvalid for arguments the operator does not take.  The operator makes the same checks on
    the way to the kernel; this says what was wrong, and costs a valid call nothing."""
    for name, t in (("x", x), ("weight", weight)):
        _want(isinstance(t, torch.Tensor), f"The data type of input {name} must be torch.Tensor, but got {type(t)}.")
    _want(weight.dim() == 2 and x.dim() >= 1 and x.shape[-1] == weight.shape[1] and weight.shape[0] > 0 and weight.shape[1] > 0,
          f"x must be [..., K] and weight [N, K], but got {tuple(x.shape)} and {tuple(weight.shape)}.")
    fp8 = x.dtype == torch.float8_e4m3fn
    _want(fp8 or x.dtype in (torch.bfloat16, torch.float16), f"x must be bfloat16, float16 or float8_e4m3fn, but got {x.dtype}.")
    _want(weight.dtype == x.dtype, f"weight must have the type of x ({x.dtype}), but got {weight.dtype}.")
    _want(weight.device == x.device, f"weight must be on {x.device}, but it is on {weight.device}.")
    _want(isinstance(activation, str) and activation in ACTIVATIONS,
          f"Unsupported activation: {activation!r}, expected one of {sorted(ACTIVATIONS)}.")
    n = weight.shape[0]
    if out_dtype is None:
        out_dtype = x.dtype if not fp8 else residual.dtype if isinstance(residual, torch.Tensor) else torch.bfloat16
    _want(out_dtype in (torch.bfloat16, torch.float16), f"out_dtype must be bfloat16 or float16, but got {out_dtype}.")
    if bias is not None:
        _check_optional("bias", bias, x)
        _want(bias.shape == (n,) and bias.dtype in _FLOATS, f"bias must be [{n}] in bfloat16, float16 or float32, but got "
              f"{tuple(bias.shape)} in {bias.dtype}.")
    if residual is not None:
        _check_optional("residual", residual, x)
        _want(residual.shape == x.shape[:-1] + (n,) and residual.dtype == out_dtype,
              f"residual must be {tuple(x.shape[:-1]) + (n,)} in {out_dtype}, but got {tuple(residual.shape)} in {residual.dtype}.")
    if gate is not None:
        _check_optional("gate", gate, x)
        single = gate.dim() >= 1 and gate.shape[-1] == n and gate.numel() == n
        _want(gate.dtype in _FLOATS and (single or (gate.dim() >= 2 and x.dim() >= 2 and gate.shape[-1] == n and
                                                    gate.shape[0] == x.shape[0] and gate.numel() == x.shape[0] * n)),
              f"gate must be [{n}] or [{x.shape[0]}, 1, {n}] in bfloat16, float16 or float32, but got {tuple(gate.shape)} "
              f"in {gate.dtype}.")
    if fp8:
        _want(x_scale is not None and weight_scale is not None, "e4m3 operands need x_scale and weight_scale.")
        rows = x.numel() // x.shape[-1]
        for name, t, count, lead in (("x_scale", x_scale, rows, x.shape[:-1]), ("weight_scale", weight_scale, n, (n,))):
            _check_optional(name, t, x)
            _want(t.dtype == torch.float32 and (t.numel() == 1 or t.shape == lead or t.shape == (*lead, 1)),
                  f"{name} must be float32 with one value in all or one per row ({count}), but got {tuple(t.shape)} in {t.dtype}.")
    else:
        _want(x_scale is None and weight_scale is None, "x_scale and weight_scale belong to e4m3 operands.")
    _want(max(weight.shape[0], weight.shape[1], x.numel() // x.shape[-1]) <= 0x7fff0000,
          f"Too many rows or columns: {tuple(x.shape)} and {tuple(weight.shape)}.")
    refuse_gradients("linear_forward", x, weight, bias, residual, gate, x_scale, weight_scale)
    _want(x.is_cuda or x.is_meta, f"linear_forward runs on a CUDA device, but x is on {x.device}.")


def linear_forward(x, weight, bias=None, activation="none", residual=None, gate=None, x_scale=None, weight_scale=None,
                   out_dtype=None):
    """out = residual + gate * act(x @ weight.T * x_scale * weight_scale + bias), accumulated and finished in fp32
    and rounded once.

    x [..., K], weight [N, K]: both bf16, both fp16 or both e4m3.  Rows whose start and stride are multiples of 32
    bytes are read in place; others are copied first (multiples of 16 bytes only where the copy is the shorter way).
    bias: [N], bf16, fp16 or fp32.  activation: "none", "relu", "silu", "gelu" (erf) or "gelu_tanh".
    gate: [N], or [B, N] / [B, 1, .., N] with B the first dimension of x; bf16, fp16 or fp32.
    residual: [..., N] in the output's type.
    x_scale, weight_scale: e4m3 operands only, where both are required: fp32, one value per row ([..., 1] or [...]
    for x, [N] or [N, 1] for weight) or one in all.
    out_dtype: bfloat16 or float16; by default the type of x, for e4m3 operands that of the residual or bfloat16."""
    try:
        if x.is_cuda:
            return checked(_op(x, weight, bias, residual, gate, x_scale, weight_scale, activation, out_dtype), "linear_forward")
    except (RuntimeError, TypeError, AttributeError):
        _explain(x, weight, bias, activation, residual, gate, x_scale, weight_scale, out_dtype)
        raise
    _explain(x, weight, bias, activation, residual, gate, x_scale, weight_scale, out_dtype)
    return _op(x, weight, bias, residual, gate, x_scale, weight_scale, activation, out_dtype)  # shapes only (meta tensors)
