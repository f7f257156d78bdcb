"""Layer norm of features, with its backward pass.

    from yggdrasil_b200 import layer_norm
    y = layer_norm(x, weight, bias)     # (x - mean) / sqrt(var + eps) weight + bias, over the last dimension

The kernels are csrc/ygg_norm.cu; means, variances and the sums of the gradients are held in 32 bits whatever the types, and the
gradients of weight and bias repeat bit for bit. There is no second derivative and no forward-mode one: both are refused
with NotImplementedError.
"""
from __future__ import annotations

import math

import torch

from . import _ops
from .logprobs import DTYPES


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """x (..., D) float32, float16 or bfloat16 on a CUDA device; weight and bias (D,) of any of these types, or None. Returns x's
    type. x, weight and bias may require a gradient."""
    y = _ops.layer_norm(x, weight, bias, eps)   # rows as the kernels read them
    return y if y is not None else _prepared(x, weight, bias, eps)


def _prepared(x, weight, bias, eps):
    """The same with whatever else the arguments may be: checked, and brought into the plain form."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda or x.dtype not in DTYPES or x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("x must be a float32, float16 or bfloat16 CUDA tensor (..., D), D at least 1")
    for name, v in (("weight", weight), ("bias", bias)):
        if v is not None and (not isinstance(v, torch.Tensor) or v.dtype not in DTYPES or v.shape != x.shape[-1:]
                              or v.device != x.device):
            raise ValueError(f"{name} must be a float tensor ({x.shape[-1]},) on {x.device}")
    if isinstance(eps, bool) or not isinstance(eps, (int, float)) or not 0 <= eps < math.inf:
        raise ValueError(f"eps {eps}: a finite number, 0 or more")
    weight, bias = (v if v is None else v.resolve_neg().contiguous() for v in (weight, bias))
    return _ops.layer_norm(x.resolve_neg().contiguous(), weight, bias, float(eps))
