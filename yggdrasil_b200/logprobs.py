"""Log-probabilities of given tokens, with the entropy and the top alternatives of each row, and their gradient.

    from yggdrasil_b200 import token_logprobs
    logits, state = model.step(tokens, state)
    out = token_logprobs(logits, sampled, top=5)
    out.logprob       # (B,) float32: log softmax(logits)[sampled]
    out.entropy       # (B,) float32, nats
    out.lse           # (B,) float32: log sum exp
    out.top_ids       # (B, 5) int32, by value descending, ties by the lower index (int32: they feed model.step)
    out.top_logprobs  # (B, 5) float32

The kernels are csrc/ygg_logprobs.cu; the sums are held in 32 bits whatever the logits' type. With logits that require
a gradient, logprob, entropy, lse and top_logprobs carry one (top_ids does not).
"""
from __future__ import annotations

from typing import NamedTuple

import numpy as np
import torch

from ._native import check, ops
from .inference import _raw_stream

DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
TOP_MAX = 64


class TokenLogprobs(NamedTuple):
    logprob: torch.Tensor
    entropy: torch.Tensor
    lse: torch.Tensor
    top_ids: torch.Tensor | None
    top_logprobs: torch.Tensor | None


def _forward(logits, tokens, top, stats):
    rows, vocab = logits.shape
    dev = logits.device
    values = torch.empty((3, rows), dtype=torch.float32, device=dev)
    ids = tops = None
    if top:
        ids = torch.empty((rows, top), dtype=torch.int32, device=dev)
        tops = torch.empty((rows, top), dtype=torch.float32, device=dev)
    at = values.data_ptr()
    code = ops().ygg_token_logprobs(
        dev.index, DTYPES[logits.dtype], rows, vocab, logits.data_ptr(), logits.stride(0), tokens.data_ptr(),
        tokens.element_size(), top, at, at + 4 * rows, at + 8 * rows, ids.data_ptr() if top else None,
        tops.data_ptr() if top else None, stats.data_ptr() if stats is not None else None, _raw_stream(dev.index))
    if code:
        check(code, "ygg_token_logprobs")
    return *values.unbind(0), ids, tops


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, top):
        stats = torch.empty((logits.shape[0], 4), dtype=torch.float32, device=logits.device)
        out = _forward(logits, tokens, top, stats)
        ctx.save_for_backward(logits, tokens, stats, out[3])
        ctx.top = top
        ctx.set_materialize_grads(False)
        if top:
            ctx.mark_non_differentiable(out[3])
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_logprob, g_entropy, g_lse, _, g_top):
        logits, tokens, stats, ids = ctx.saved_tensors
        rows, vocab = logits.shape
        # rows that lie to the 16-byte boundary as the logits' do move 16 bytes at a time
        per = 16 // logits.element_size()
        wide = -(-vocab // per) * per if logits.stride(0) % per == 0 else vocab
        grad = torch.empty((rows, wide), dtype=logits.dtype, device=logits.device)[:, :vocab]
        # what arrives may be expanded (a sum's gradient) or of another type
        arriving = [None if g is None else g.float().contiguous() for g in (g_logprob, g_entropy, g_lse, g_top)]
        dev = logits.device.index
        code = ops().ygg_token_logprobs_backward(
            dev, DTYPES[logits.dtype], rows, vocab, logits.data_ptr(), logits.stride(0), tokens.data_ptr(),
            tokens.element_size(), ctx.top, ids.data_ptr() if ids is not None else None, stats.data_ptr(),
            *[None if g is None else g.data_ptr() for g in arriving], grad.data_ptr(), wide, _raw_stream(dev))
        if code:
            check(code, "ygg_token_logprobs_backward")
        return grad, None, None


def token_logprobs(logits, tokens, top=0):
    """logits (..., V) float32, float16 or bfloat16 on a CUDA device, any row stride; tokens (...) the given token of
    each row: an int32 or int64 tensor, or host integers (range-checked: < V). A negative token is padding: logprob 0
    and no gradient from it. top: how many alternatives, 0 to min(V, 64).

    -inf logits (masked tokens) have probability 0. A row of -inf alone has logprob and lse -inf, entropy 0, gradient
    0, and alternatives by the lower index; a row that holds NaN or +inf has NaN values."""
    if not isinstance(logits, torch.Tensor) or not logits.is_cuda or logits.dtype not in DTYPES or logits.dim() < 1:
        raise ValueError("logits must be a float32, float16 or bfloat16 CUDA tensor (..., V)")
    lead, vocab = logits.shape[:-1], logits.shape[-1]
    if vocab < 1:
        raise ValueError("logits: the vocabulary is empty")
    if not 0 <= top <= min(vocab, TOP_MAX):
        raise ValueError(f"top {top}: 0 to {min(vocab, TOP_MAX)}")
    if not isinstance(tokens, torch.Tensor) or not tokens.is_cuda:
        host = np.asarray(tokens)
        if host.size and (host.dtype.kind not in "iu" or host.max() >= vocab):
            raise ValueError(f"tokens must be integers below {vocab}")
        tokens = torch.as_tensor(np.array(host, np.int64)).to(logits.device)
    if tokens.dtype not in (torch.int32, torch.int64) or tokens.device != logits.device:
        raise ValueError(f"tokens must be int32 or int64 on {logits.device}")
    if tokens.shape != lead:
        raise ValueError(f"tokens {tuple(tokens.shape)} for logits {tuple(logits.shape)}: one token for each row")
    x = logits if logits.dim() == 2 else logits.reshape(-1, vocab)
    if x.stride(1) != 1 and vocab > 1:
        x = x.contiguous()
    t = tokens.contiguous()
    with torch.cuda.device(x.device) if x.device.index != torch.cuda.current_device() else _nothing:
        if x.requires_grad and torch.is_grad_enabled():
            out = _TokenLogprobs.apply(x, t, top)
        else:
            out = _forward(x, t, top, None)
    if len(lead) != 1:
        out = [None if v is None else v.reshape(lead + v.shape[1:]) for v in out]
    return TokenLogprobs(*out)


class _Nothing:
    def __enter__(self):
        return None

    def __exit__(self, *_):
        return False


_nothing = _Nothing()
