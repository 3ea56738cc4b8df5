"""The norms in front of a transformer block's projections: `add_rms_norm` (residual addition and
root-mean-square norm in one pass; `RMSNorm` of mindiesd/layers/norm.py of MindIE-SD with the addition
that precedes it) and `add_rms_norm_quant`, whose output is e4m3 with one scale per token, ready for
`linear_forward`.

Inference only: there is no backward pass and no forward-mode derivative, so tensors that require gradients are
refused while gradients are recorded, and so are tensors that carry a tangent.
"""
import torch
from torch.autograd import forward_ad

from . import _custom_ops  # noqa: F401  (registers the fake implementations)
from ..utils.exception import ParametersInvalid

_op = torch.ops.mindiesd.add_rms_norm.default
_TYPES = (torch.bfloat16, torch.float16, torch.float32)


def refuse_gradients(where, *tensors):
    given = [t for t in tensors if t is not None]
    if torch.is_grad_enabled() and any(t.requires_grad for t in given):
        raise ParametersInvalid(f"{where} has no backward pass; call it under torch.no_grad() or torch.inference_mode().")
    if torch._C._is_fwd_grad_enabled() and any(forward_ad.unpack_dual(t).tangent is not None for t in given):
        raise ParametersInvalid(f"{where} has no forward-mode derivative, but an input carries a tangent.")


def _explain(where, x, weight, residual, eps):
    """Raises ParametersInvalid for arguments the operator does not take.  The operator makes the same checks on
    the way to the kernel; this says what was wrong, and costs a valid call nothing."""
    if not isinstance(x, torch.Tensor):
        raise ParametersInvalid(f"The data type of input x must be torch.Tensor, but got {type(x)}.")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ParametersInvalid(f"The input x must be [..., D] with D > 0, but got {tuple(x.shape)}.")
    if x.dtype not in _TYPES:
        raise ParametersInvalid(f"{where} supports bfloat16, float16 and float32, but got {x.dtype}.")
    if weight is not None:
        if not isinstance(weight, torch.Tensor):
            raise ParametersInvalid(f"The data type of input weight must be torch.Tensor, but got {type(weight)}.")
        if weight.shape != x.shape[-1:] or weight.device != x.device:
            raise ParametersInvalid(f"The input weight must be [{x.shape[-1]}] on {x.device}, but got "
                                    f"{tuple(weight.shape)} on {weight.device}.")
        if weight.dtype != x.dtype and weight.dtype != torch.float32:
            raise ParametersInvalid(f"The input weight must be {x.dtype} or float32, but got {weight.dtype}.")
    if residual is not None:
        if not isinstance(residual, torch.Tensor):
            raise ParametersInvalid(f"The data type of input residual must be torch.Tensor, but got {type(residual)}.")
        if residual.shape != x.shape or residual.device != x.device:
            raise ParametersInvalid(f"The input residual must be {tuple(x.shape)} on {x.device}, but got "
                                    f"{tuple(residual.shape)} on {residual.device}.")
        if residual.dtype != x.dtype and residual.dtype != torch.float32:
            raise ParametersInvalid(f"The input residual must be {x.dtype} or float32, but got {residual.dtype}.")
    if not isinstance(eps, float) or not 1e-38 < eps < 1e30:
        raise ParametersInvalid(f"The input eps must be a positive float (normal in float32), but got {eps!r}.")
    if x.shape[-1] > 0x3fffffff or x.numel() // x.shape[-1] > 0x7fffffff:
        raise ParametersInvalid(f"{where} takes at most 2^30 - 1 channels and 2^31 - 1 rows, but got {tuple(x.shape)}.")
    refuse_gradients(where, x, weight, residual)
    if not x.is_cuda and not x.is_meta:
        raise ParametersInvalid(f"{where} runs on a CUDA device, but x is on {x.device}.")


def _run(where, x, weight, residual, eps, quant):
    try:
        if x.is_cuda:
            return _op(x, weight, residual, eps, quant, False)
    except (RuntimeError, TypeError, AttributeError):
        _explain(where, x, weight, residual, eps)
        raise
    _explain(where, x, weight, residual, eps)
    return _op(x, weight, residual, eps, quant, False)  # shapes only (meta tensors)


def add_rms_norm(x, weight=None, residual=None, eps=1e-6):
    """y = v * weight / sqrt(mean(v^2) + eps) over the last dimension, with v = x + residual in fp32 (v = x
    without a residual) and one rounding to the type of x.  x: [..., D] bf16, fp16 or fp32; weight [D] (None:
    ones) and residual [..., D] in the type of x or fp32.  Returns y, or (y, v rounded to the residual's type)
    when a residual is given.  Leading dimensions that share one row stride (slices of a packed projection)
    are read in place.  The squares are summed in fp32: a row whose sum passes 3.4e38 (a root mean square of 1.8e19 /
    sqrt(D), 2.6e17 for 5120 channels) gives zeros."""
    y, _, total = _run("add_rms_norm", x, weight, residual, eps, False)
    return y if residual is None else (y, total)


def add_rms_norm_quant(x, weight=None, residual=None, eps=1e-6):
    """The same norm with its output in e4m3 and one scale per token, taken on the fp32 values: returns
    (e4m3 [..., D], fp32 scales [..., 1]), with the residual's sum as a third where one is given; real value =
    stored * scale, scale = max|y| / 448 (1 for a token of zeros, or one whose sum of squares overflows as there; NaN for
    one that holds a NaN or an infinity)."""
    q, scale, total = _run("add_rms_norm_quant", x, weight, residual, eps, True)
    return (q, scale) if residual is None else (q, scale, total)
