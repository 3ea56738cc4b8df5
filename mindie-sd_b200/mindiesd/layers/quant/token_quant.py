"""`token_quant_preprocess`: dynamic quantisation of the input of an e4m3 linear layer, one scale per token
(the activation side of the dynamic quantised linear layers of mindiesd/quantization/layer.py of MindIE-SD)."""
import torch

from ..norm import refuse_gradients
from ...utils.exception import ParametersInvalid

_op = torch.ops.mindiesd.add_rms_norm.default


def _explain(input_tensor):
    if not isinstance(input_tensor, torch.Tensor):
        raise ParametersInvalid(f"The data type of input_tensor must be torch.Tensor, but got {type(input_tensor)}.")
    if input_tensor.dim() < 1 or input_tensor.shape[-1] < 1:
        raise ParametersInvalid(f"input_tensor must be [..., D] with D > 0, but got {tuple(input_tensor.shape)}.")
    if input_tensor.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise ParametersInvalid(f"token_quant_preprocess supports bfloat16, float16 and float32, but got "
                                f"{input_tensor.dtype}.")
    if input_tensor.shape[-1] > 0x3fffffff or input_tensor.numel() // input_tensor.shape[-1] > 0x7fffffff:
        raise ParametersInvalid(f"token_quant_preprocess takes at most 2^30 - 1 channels and 2^31 - 1 rows, but got "
                                f"{tuple(input_tensor.shape)}.")
    refuse_gradients("token_quant_preprocess", input_tensor)
    if not input_tensor.is_cuda and not input_tensor.is_meta:
        raise ParametersInvalid(f"token_quant_preprocess runs on a CUDA device, but input_tensor is on "
                                f"{input_tensor.device}.")


def token_quant_preprocess(input_tensor):
    """input_tensor: [..., D] bf16, fp16 or fp32.  Returns (e4m3 [..., D], fp32 scales [..., 1]); real = stored *
    scale, scale = absmax / 448 of the token (1 for a token of zeros).  Rows of a weight matrix [N, K] quantised
    this way have one scale per output channel."""
    try:
        if input_tensor.is_cuda:
            return _op(input_tensor, None, None, 1.0, True, True)[:2]
    except (RuntimeError, AttributeError):
        _explain(input_tensor)
        raise
    _explain(input_tensor)
    return _op(input_tensor, None, None, 1.0, True, True)[:2]  # shapes only (meta tensors)
