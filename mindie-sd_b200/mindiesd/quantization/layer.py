"""The layers of a quantised model: `FP8RotateQuantFA`, the FP8 attention hook it calls instead of
attention_forward (mindiesd/quantization/layer.py:274-324 of MindIE-SD), and `FP8DynamicLinear`, a linear layer
on e4m3 operands whose input is quantised per token as it comes (the dynamic linear layers of that file)."""
import math

import torch
from torch import nn

from ..layers.linear import linear_forward
from ..layers.quant.token_quant import token_quant_preprocess
from ..layers.quant.block_quant import fa_block_quant_preprocess, fa_channel_quant_preprocess
from ..utils.exception import ParametersInvalid
from ..utils.status import checked


def get_quant_weight(weights, name):
    if weights is None or name not in weights:
        return None
    w = weights[name]
    return w if isinstance(w, torch.Tensor) else torch.as_tensor(w)


class FP8RotateQuantFA(nn.Module):
    """forward(query, key, value, layout=): rotate q and k by the learned 128x128 matrices (fused into
    the quantisation kernel), quantise
    q (128-token blocks), k and v (256-token blocks) to e4m3, run FP8 attention, return the input
    dtype and layout.  Without learned matrices q and k are rotated by the fixed Hadamard matrix
    inside the quantisation kernel.  `v_per_channel=True` quantises v with one scale per channel."""

    def __init__(self, prefix=None, weights=None, v_per_channel=False):
        super().__init__()
        self.register_buffer("q_rot", get_quant_weight(weights, f"{prefix}.q_rot"), persistent=False)
        self.register_buffer("k_rot", get_quant_weight(weights, f"{prefix}.k_rot"), persistent=False)
        self.v_per_channel = v_per_channel
        if (self.q_rot is None) != (self.k_rot is None):
            # q k^T is only preserved when both operands are rotated by matching matrices; the
            # reference fails in its first matmul when one of them is missing (layer.py:284-285).
            missing = "k_rot" if self.k_rot is None else "q_rot"
            raise ParametersInvalid(f"FP8RotateQuantFA needs both {prefix}.q_rot and {prefix}.k_rot, or neither "
                                    f"(fixed Hadamard rotation); {prefix}.{missing} is missing.")

    def forward(self, query, key, value, **kwargs):
        layout = kwargs.get("layout", "BNSD")
        if layout not in ("BNSD", "BSND"):
            raise ValueError(f"Unsupported layout: {layout}, expected 'BNSD' or 'BSND'.")
        d = query.shape[-1]
        fixed = self.q_rot is None and self.k_rot is None
        # A learned rotation runs on the tensor cores inside the quantisation kernel; without learned
        # matrices both operands get the fixed Hadamard rotation, also inside that kernel.
        q, q_scale = fa_block_quant_preprocess(query, block_size=128, layout=layout, rotate=fixed, rot=self.q_rot)
        k, k_scale = fa_block_quant_preprocess(key, block_size=256, layout=layout, rotate=fixed, rot=self.k_rot)
        if self.v_per_channel:
            v, v_scale = fa_channel_quant_preprocess(value, layout=layout)
            v_block = 0
        else:
            v, v_scale = fa_block_quant_preprocess(value, block_size=256, layout=layout)
            v_block = 256
        out = torch.ops.mindiesd.fp8_attention(q, k, v, q_scale, k_scale, v_scale, 1.0 / math.sqrt(d), 256, v_block,
                                               query.dtype)
        return checked(out.transpose(1, 2) if layout == "BSND" else out, "FP8RotateQuantFA")


class FP8DynamicLinear(nn.Module):
    """A linear layer with e4m3 weights, one scale per output channel, and its input quantised per token.

    weights[f"{prefix}.weight"]: [N, K], e4m3 together with f"{prefix}.weight_scale" ([N] or [N, 1] fp32), or a
    bf16 / fp16 / fp32 CUDA tensor that is quantised once, here; f"{prefix}.bias" is optional.

    forward(x, activation=, residual=, gate=, out_dtype=): x is a bf16 / fp16 / fp32 tensor [..., K], or the pair
    (e4m3 [..., K], scales [..., 1]) that add_rms_norm_quant returns; the other arguments are linear_forward's.
    The output has the type of x (bfloat16 for fp32 and for a pair) unless out_dtype or a residual says otherwise.

    Converting the module to another dtype converts the bias alone."""

    def __init__(self, prefix=None, weights=None):
        super().__init__()
        weight, scale = get_quant_weight(weights, f"{prefix}.weight"), get_quant_weight(weights, f"{prefix}.weight_scale")
        if weight is None or weight.dim() != 2:
            raise ParametersInvalid(f"FP8DynamicLinear needs {prefix}.weight [N, K], but got "
                                    f"{None if weight is None else tuple(weight.shape)}.")
        if (weight.dtype == torch.float8_e4m3fn) != (scale is not None):
            raise ParametersInvalid(f"FP8DynamicLinear takes {prefix}.weight_scale exactly with e4m3 weights, but "
                                    f"{prefix}.weight is {weight.dtype}.")
        if scale is None:
            weight, scale = token_quant_preprocess(weight.detach())
        elif scale.dtype != torch.float32 or scale.numel() != weight.shape[0]:
            raise ParametersInvalid(f"{prefix}.weight_scale must be float32 with {weight.shape[0]} values, but got "
                                    f"{tuple(scale.shape)} in {scale.dtype}.")
        bias = get_quant_weight(weights, f"{prefix}.bias")
        self.register_buffer("weight", weight.detach())
        self.register_buffer("weight_scale", scale.detach().reshape(-1))
        self.register_buffer("bias", None if bias is None else bias.detach())

    @classmethod
    def from_linear(cls, linear):
        """The quantised form of a torch.nn.Linear on a CUDA device."""
        weights = {"linear.weight": linear.weight}
        if linear.bias is not None:
            weights["linear.bias"] = linear.bias
        return cls("linear", weights)

    def _apply(self, fn, recurse=True):
        # What is stored is the e4m3 values and their fp32 scales: module.to(dtype), .half() and the like, which convert
        # every floating-point buffer, leave these two as they are; a move to another device takes them along.
        def same_type(t):
            moved = fn(t)
            return moved if moved.dtype == t.dtype else t.to(moved.device)
        return super()._apply(lambda t: same_type(t) if t is self.weight or t is self.weight_scale else fn(t), recurse)

    def forward(self, x, activation="none", residual=None, gate=None, out_dtype=None):
        if isinstance(x, tuple):
            if len(x) != 2:
                raise ParametersInvalid(f"A quantised input is the pair (e4m3 tensor, scales), but got {len(x)} items.")
            q, scale = x
        else:
            if out_dtype is None and residual is None and isinstance(x, torch.Tensor) and x.dtype == torch.float16:
                out_dtype = torch.float16
            q, scale = token_quant_preprocess(x)
        return linear_forward(q, self.weight, self.bias, activation=activation, residual=residual, gate=gate, x_scale=scale,
                              weight_scale=self.weight_scale, out_dtype=out_dtype)


def add_fa_quant(module, prefix=None, weights=None):
    """Attaches the hook as `module.fa_quant` (mindiesd/quantization/quantize.py:158-161)."""
    module.fa_quant = FP8RotateQuantFA(prefix, weights)
    return module
