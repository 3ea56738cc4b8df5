"""The operators around attention restated in 64 bits on the tensors' own device: residual addition with RMS
norm, per-token quantisation, and the matrix product with its epilogue.  Test infrastructure only.

The values are the real-number results before the last rounding; `half_step` is what one rounding to a type
may be off by, relative to the value."""
from __future__ import annotations

import math

import torch

E4M3_MAX = 448.0


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def smallest_half_step(dtype):
    """Half the distance between neighbouring subnormal values."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def rms_norm(x, weight=None, residual=None, eps=1e-6):
    """(y, v) in fp64."""
    v = x.double()
    if residual is not None:
        v = v + residual.double()
    y = v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps)
    if weight is not None:
        y = y * weight.double()
    return y, v


def token_scale(y):
    top = y.abs().amax(-1, keepdim=True)
    return torch.where(top == 0, torch.ones_like(top), (top / E4M3_MAX).clamp_min(2.0 ** -126))


def activation(v, name):
    if name == "relu":
        return torch.where(v > 0, v, torch.zeros_like(v)) if not torch.isnan(v).any() else v.clamp_min(0)
    if name == "silu":
        return v / (1 + torch.exp(-v))
    if name == "gelu":
        return v * 0.5 * torch.erfc(-v / math.sqrt(2.0))
    if name == "gelu_tanh":
        return v / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)))
    assert name == "none"
    return v


def linear(x, weight, bias=None, act="none", residual=None, gate=None, x_scale=None, weight_scale=None):
    """(value, bound): the result in fp64, and the sum of |x||w| of every element -- what the rounding of a
    32-bit accumulation is relative to -- carried through the epilogue.  gate: [N] or [B, 1.., N]."""
    xd, wd = x.double(), weight.double()
    if x_scale is not None:
        xd = xd * x_scale.double()
    if weight_scale is not None:
        wd = wd * weight_scale.double().reshape(-1, 1)
    v = xd @ wd.T
    size = xd.abs() @ wd.abs().T
    if bias is not None:
        v = v + bias.double()
        size = size + bias.double().abs()
    v = activation(v, act)
    if act != "none":
        size = 1.2 * size  # no activation here is steeper than 1.13
    if gate is not None:
        v = v * gate.double()
        size = size * gate.double().abs()
    if residual is not None:
        v = v + residual.double()
        size = size + residual.double().abs()
    return v, size
