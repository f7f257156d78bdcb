"""Linear layers in 8-bit integers: a scale for each row of activations, found as it comes, and one for each channel.

    from yggdrasil_b200 import int8_linear, quantize_rows
    head = quantize_rows(weight)                        # once: (N, K) floats -> codes and a scale for each channel
    y = int8_linear(x, head.codes, head.scale, bias)    # (..., K) -> (..., N) in x's type

y = (codes(x) . codes(w)) scale_w scale_x + bias, the sums exact in int32 (csrc/ygg_linear.cu): a row's outputs have the same
bits alone and in any batch. The weights are frozen: there is no gradient, and rows, scales or a bias that ask for one are
refused with NotImplementedError (detach() them, or call under torch.no_grad()).
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import _ops
from ._native import check, ops
from .inference import _raw_stream
from .logprobs import DTYPES

MAX_K = 131072


class QuantizedRows(NamedTuple):
    codes: torch.Tensor   # int8 (..., K), rows a multiple of 16 bytes apart
    scale: torch.Tensor   # float32 (...)


def quantize_rows(x):
    """x (..., K) float32, float16 or bfloat16 -> QuantizedRows. The scale of a row is its largest magnitude / 127, a
    code the nearest integer (ties to even) of the value times 127 / that magnitude. A row of zeros, or of magnitudes
    below 3.73e-37, has scale 0; a row that holds NaN or infinity has scale NaN."""
    out = _ops.quantize_rows(x)
    if out is None:
        codes, scale = _ops.quantize_rows(_rows(x))
        lead, k = x.shape[:-1], x.shape[-1]
        step = codes.stride(0)
        out = codes.as_strided((*lead, k), (*_strides(lead, step), 1)), scale.view(lead)
    return QuantizedRows(*out)


def int8_linear(x, weight, scale, bias=None, out_dtype=None):
    """x (..., K) @ weight.T with scales: x float32, float16 or bfloat16 (quantised here, a scale for each row) or a
    QuantizedRows; weight int8 (N, K) and scale float32 (N,), as quantize_rows gives them; bias (N,) or None. Returns
    (..., N) in out_dtype: x's type by default, float32 for QuantizedRows.

    Weights whose rows are not a multiple of 16 bytes apart are copied at each call: keep them as quantize_rows lays
    them out."""
    out = _ops.int8_linear(x, weight, scale, bias, out_dtype)   # (rows, K) and weights as the kernels read them
    return out if out is not None else _prepared(x, weight, scale, bias, out_dtype)


def _prepared(x, weight, scale, bias, out_dtype):
    """The same with whatever else the arguments may be: checked, and brought into the plain form."""
    if isinstance(x, QuantizedRows):
        codes, row_scale = x
        if codes.dtype != torch.int8 or not codes.is_cuda or codes.dim() < 1 or row_scale.dtype != torch.float32 \
                or row_scale.shape != codes.shape[:-1] or row_scale.device != codes.device:
            raise ValueError("QuantizedRows: int8 codes (..., K) and a float32 scale (...) on one CUDA device")
        lead, k, device = codes.shape[:-1], codes.shape[-1], codes.device
        _frozen(row_scale)
        if not 1 <= k <= MAX_K:
            raise ValueError(f"codes: K {k}: 1 to {MAX_K}")
    else:
        rows = _rows(x)
        lead, k, device = x.shape[:-1], x.shape[-1], x.device
    if out_dtype is not None and out_dtype not in DTYPES:
        raise ValueError(f"out_dtype {out_dtype}: float32, float16 or bfloat16")
    if not isinstance(weight, torch.Tensor) or weight.dtype != torch.int8 or weight.dim() != 2 or weight.shape[1] != k \
            or weight.device != device or weight.shape[0] < 1:
        raise ValueError(f"weight must be an int8 tensor (N, {k}) on {device}")
    n = weight.shape[0]
    if not isinstance(scale, torch.Tensor) or scale.dtype != torch.float32 or scale.shape != (n,) \
            or scale.device != device:
        raise ValueError(f"scale must be a float32 tensor ({n},) on {device}")
    if bias is not None:
        if not isinstance(bias, torch.Tensor) or bias.shape != (n,) or bias.device != device or bias.dtype not in DTYPES:
            raise ValueError(f"bias must be a float tensor ({n},) on {device}")
        _frozen(bias)
        bias = bias.detach().float().contiguous()
    _frozen(scale)
    with torch.cuda.device(device):
        weights = _laid_out(weight), scale.contiguous(), bias, out_dtype
        if isinstance(x, QuantizedRows):
            out = _ops.int8_linear_rows(_laid_out(codes.reshape(-1, k)), row_scale.reshape(-1).contiguous(), *weights)
        else:
            out = _ops.int8_linear(rows, *weights)
    return out.view(*lead, n)


def _rows(x):
    """x as (rows, K) with its entries side by side."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda or x.dtype not in DTYPES or x.dim() < 1:
        raise ValueError("x must be a float32, float16 or bfloat16 CUDA tensor (..., K)")
    k = x.shape[-1]
    if not 1 <= k <= MAX_K:
        raise ValueError(f"x: K {k}: 1 to {MAX_K}")
    _frozen(x)
    rows = x.reshape(-1, k)
    return rows if k == 1 or rows.stride(1) == 1 else rows.contiguous()


def _frozen(*tensors):
    """Refuse tensors through which a gradient, or a forward-mode derivative, is asked for."""
    if any(_ops.tracked(t) for t in tensors):
        raise NotImplementedError("the int8 product has no gradient: use detach() or torch.no_grad()")


def _strides(lead, step):
    """The strides of leading dimensions whose rows lie `step` apart."""
    out = []
    for size in reversed(lead):
        out.insert(0, step)
        step *= size
    return out


def linear_status(device="cuda"):
    """Raise YggError if a bounded wait of an int8 product on the device gave up since the last call: outputs since then
    are not to be used. Waits for the current stream. The record is one for the device and all of its callers: the first
    that asks is told, and clears it."""
    device = torch.device(device)
    index = device.index if device.index is not None else torch.cuda.current_device()
    out = ctypes.c_int(0)
    check(ops().ygg_linear_status(index, _raw_stream(index), ctypes.byref(out)), "ygg_linear_status")
    check(out.value, "int8 product")


def _laid_out(codes):
    """codes (rows, K) with their entries side by side and rows a multiple of 16 bytes apart."""
    rows, k = codes.shape
    step, one = codes.stride()
    if one == 1 and step % 16 == 0 and step >= k and codes.data_ptr() % 16 == 0:
        return codes
    out = torch.empty((rows, (k + 15) // 16 * 16), dtype=torch.int8, device=codes.device)[:, :k]
    return out.copy_(codes)
