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
a gradient, logprob, entropy, lse and top_logprobs carry one (top_ids does not). There is no second derivative and no
forward-mode one: logits with a tangent are refused with NotImplementedError.
"""
from __future__ import annotations

from typing import NamedTuple

import numpy as np
import torch

from . import _ops

DTYPES = (torch.float32, torch.float16, torch.bfloat16)
TOP_MAX = 64


class TokenLogprobs(NamedTuple):
    logprob: torch.Tensor
    entropy: torch.Tensor
    lse: torch.Tensor
    top_ids: torch.Tensor | None
    top_logprobs: torch.Tensor | None


def token_logprobs(logits, tokens, top=0):
    """logits (..., V) float32, float16 or bfloat16 on a CUDA device, any row stride; tokens (...) the given token of
    each row: an int32 or int64 tensor, or host integers (range-checked: < V). A negative token is padding: logprob 0
    and no gradient from it. top: how many alternatives, 0 to min(V, 64).

    -inf logits (masked tokens) have probability 0. A row of -inf alone has logprob and lse -inf, entropy 0, gradient
    0, and alternatives by the lower index; a row that holds NaN or +inf has NaN values."""
    out = _ops.token_logprobs(logits, tokens, top)   # (rows, V) and (rows,) as the kernels read them
    return tuple.__new__(TokenLogprobs, out if out is not None else _prepared(logits, tokens, top))


def _prepared(logits, tokens, top):
    """The same with whatever else the arguments may be: checked, and brought into the plain form."""
    if not isinstance(logits, torch.Tensor) or not logits.is_cuda or logits.dtype not in DTYPES or logits.dim() < 1:
        raise ValueError("logits must be a float32, float16 or bfloat16 CUDA tensor (..., V)")
    lead, vocab = logits.shape[:-1], logits.shape[-1]
    if vocab < 1:
        raise ValueError("logits: the vocabulary is empty")
    if not hasattr(top, "__index__") or not 0 <= top <= min(vocab, TOP_MAX):   # 2.5 is no number of alternatives
        raise ValueError(f"top {top}: an integer, 0 to {min(vocab, TOP_MAX)}")
    if not isinstance(tokens, torch.Tensor) or not tokens.is_cuda:
        host = np.asarray(tokens)
        if host.size and (host.dtype.kind not in "iu" or host.max() >= vocab):
            raise ValueError(f"tokens must be integers below {vocab}")
        tokens = torch.as_tensor(np.array(host, np.int64)).to(logits.device)
    if tokens.dtype not in (torch.int32, torch.int64) or tokens.device != logits.device:
        raise ValueError(f"tokens must be int32 or int64 on {logits.device}")
    if tokens.shape != lead:
        raise ValueError(f"tokens {tuple(tokens.shape)} for logits {tuple(logits.shape)}: one token for each row")
    x = logits.reshape(-1, vocab)
    out = _ops.token_logprobs(x if vocab == 1 or x.stride(1) == 1 else x.contiguous(),
                              tokens.reshape(-1).contiguous(), int(top))
    return [None if v is None else v.view(lead + v.shape[1:]) for v in out]
