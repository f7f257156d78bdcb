"""Linear layers in 8-bit integers: a scale for each row of activations, found as it comes, and one for each channel.

    from yggdrasil_b200 import int8_linear, quantize_rows
    head = quantize_rows(weight)                        # once: (N, K) floats -> codes and a scale for each channel
    y = int8_linear(x, head.codes, head.scale, bias)    # (..., K) -> (..., N) in x's type

y = (codes(x) . codes(w)) scale_x scale_w + bias, the sums exact in int32 (csrc/ygg_linear.cu). The weights are frozen:
there is no gradient.
"""
from __future__ import annotations

import ctypes
import functools
from typing import NamedTuple

import torch

from ._native import check, ops
from .inference import _raw_stream
from .logprobs import DTYPES, _nothing

MAX_K = 131072


class QuantizedRows(NamedTuple):
    codes: torch.Tensor   # int8 (..., K), rows a multiple of 16 bytes apart
    scale: torch.Tensor   # float32 (...)


def _rows(x, what):
    """x as (rows, K) with its entries side by side."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda or x.dtype not in DTYPES or x.dim() < 1:
        raise ValueError(f"{what} must be a float32, float16 or bfloat16 CUDA tensor (..., K)")
    k = x.shape[-1]
    if not 1 <= k <= MAX_K:
        raise ValueError(f"{what}: K {k}: 1 to {MAX_K}")
    if x.requires_grad and torch.is_grad_enabled():   # the weights are frozen
        raise NotImplementedError("the int8 product has no gradient: use detach() or torch.no_grad()")
    x2 = x if x.dim() == 2 else x.reshape(-1, k)
    return x2 if x2.stride(1) == 1 or k == 1 else x2.contiguous()


def _on(device):
    return torch.cuda.device(device) if device.index != torch.cuda.current_device() else _nothing


def _aligned(t):   # (rows, K) bytes
    step, one = t.stride()
    return one == 1 and step % 16 == 0 and step >= t.shape[1] and t.data_ptr() % 16 == 0


def quantize_rows(x):
    """x (..., K) float32, float16 or bfloat16 -> QuantizedRows. The scale of a row is its largest magnitude / 127, a
    code the nearest integer (ties to even) of the value times 127 / that magnitude. A row of zeros has scale 0; a row
    that holds NaN or infinity has scale NaN."""
    lead = x.shape[:-1] if isinstance(x, torch.Tensor) else None
    x2 = _rows(x, "x")
    rows, k = x2.shape
    padded = (k + 15) // 16 * 16
    codes = torch.empty((rows, padded), dtype=torch.int8, device=x2.device)
    scale = torch.empty(rows, dtype=torch.float32, device=x2.device)
    with _on(x2.device):
        dev = x2.device.index
        check(ops().ygg_quantize_rows(dev, DTYPES[x2.dtype], rows, k, x2.data_ptr(), x2.stride(0), codes.data_ptr(),
                                      padded, scale.data_ptr(), _raw_stream(dev)), "ygg_quantize_rows")
    return QuantizedRows(codes.view(*lead, padded)[..., :k], scale.view(lead))


def int8_linear(x, weight, scale, bias=None, out_dtype=None):
    """x (..., K) @ weight.T with scales: x float32, float16 or bfloat16 (quantised here, a scale for each row) or a
    QuantizedRows; weight int8 (N, K) and scale float32 (N,), as quantize_rows gives them; bias (N,) or None. Returns
    (..., N) in out_dtype: x's type by default, float32 for QuantizedRows.

    Weights whose rows are not a multiple of 16 bytes apart are copied at each call: keep them as quantize_rows lays
    them out."""
    if isinstance(x, QuantizedRows):
        codes, row_scale = x
        if codes.dtype != torch.int8 or not codes.is_cuda or codes.dim() < 1 or row_scale.dtype != torch.float32 \
                or row_scale.shape != codes.shape[:-1] or row_scale.device != codes.device:
            raise ValueError("QuantizedRows: int8 codes (..., K) and a float32 scale (...) on one CUDA device")
        lead, k, index = codes.shape[:-1], codes.shape[-1], codes.get_device()
        if not 1 <= k <= MAX_K:
            raise ValueError(f"codes: K {k}: 1 to {MAX_K}")
        x2, out_dtype = None, out_dtype or torch.float32
    else:
        x2 = _rows(x, "x")
        shape = x.shape
        lead, k, index = shape[:-1], shape[-1], x.get_device()
        out_dtype = out_dtype or x.dtype
    if out_dtype not in DTYPES:
        raise ValueError(f"out_dtype {out_dtype}: float32, float16 or bfloat16")
    if not isinstance(weight, torch.Tensor) or weight.dtype is not torch.int8 or weight.dim() != 2 \
            or weight.shape[1] != k or weight.get_device() != index or weight.shape[0] < 1:
        raise ValueError(f"weight must be an int8 tensor (N, {k}) on cuda:{index}")
    n = weight.shape[0]
    if not isinstance(scale, torch.Tensor) or scale.dtype is not torch.float32 or scale.shape != (n,) \
            or scale.get_device() != index:
        raise ValueError(f"scale must be a float32 tensor ({n},) on cuda:{index}")
    if bias is not None and (not isinstance(bias, torch.Tensor) or bias.shape != (n,) or bias.get_device() != index
                             or bias.dtype not in DTYPES):
        raise ValueError(f"bias must be a float tensor ({n},) on cuda:{index}")
    with _nothing if index == torch.cuda.current_device() else torch.cuda.device(index):
        w = weight if _aligned(weight) else _laid_out(weight)
        s = scale if scale.is_contiguous() else scale.contiguous()
        b = bias_at = None
        if bias is not None:
            b = bias if bias.dtype is torch.float32 and bias.is_contiguous() else bias.float().contiguous()
            bias_at = b.data_ptr()
        if x2 is None:
            c = codes.reshape(-1, k)
            c = c if _aligned(c) else _laid_out(c)
            rows, r = c.shape[0], row_scale.reshape(-1).contiguous()
            out = torch.empty_strided((rows, n), (n, 1), dtype=out_dtype, device=c.device)
            code = ops().ygg_linear_quantized(
                index, rows, k, n, c.data_ptr(), c.stride(0), r.data_ptr(), w.data_ptr(), w.stride(0), s.data_ptr(),
                bias_at, DTYPES[out_dtype], out.data_ptr(), n, _raw_stream(index))
        else:
            rows, device = x2.shape[0], x2.device
            out = torch.empty_strided((rows, n), (n, 1), dtype=out_dtype, device=device)
            nbytes = _workspace(rows, k)
            ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
            code = ops().ygg_linear(
                index, DTYPES[x2.dtype], rows, k, n, x2.data_ptr(), x2.stride(0), w.data_ptr(), w.stride(0),
                s.data_ptr(), bias_at, DTYPES[out_dtype], out.data_ptr(), n, ws.data_ptr(), nbytes, _raw_stream(index))
        if code:
            check(code, "ygg_linear")
    return out if len(lead) == 1 else out.view(*lead, n)


@functools.lru_cache(maxsize=1024)
def _workspace(rows, k):
    return ops().ygg_linear_workspace(rows, k)


def linear_status(device="cuda"):
    """Raise YggError if a bounded wait of an int8 product on the device gave up since the last call: outputs since then
    are not to be used. Waits for the current stream."""
    device = torch.device(device)
    index = device.index if device.index is not None else torch.cuda.current_device()
    out = ctypes.c_int(0)
    check(ops().ygg_linear_status(index, _raw_stream(index), ctypes.byref(out)), "ygg_linear_status")
    check(out.value, "int8 product")


def _laid_out(codes):
    """codes (rows, K) with rows a multiple of 16 bytes apart."""
    rows, k = codes.shape
    out = torch.empty((rows, (k + 15) // 16 * 16), dtype=torch.int8, device=codes.device)[:, :k]
    return out.copy_(codes)
