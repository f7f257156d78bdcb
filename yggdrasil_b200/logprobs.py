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

import numpy as np
import torch

from ._native import check, ops
from .inference import _raw_stream

DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
TOP_MAX = 64


class TokenLogprobs:
    """logprob, entropy, lse, top_ids, top_logprobs, by name or in this order."""
    __slots__ = ("logprob", "entropy", "top_ids", "top_logprobs", "_lse")

    def __init__(self, logprob, entropy, lse, top_ids, top_logprobs):
        self.logprob, self.entropy, self.top_ids, self.top_logprobs = logprob, entropy, top_ids, top_logprobs
        self._lse = lse

    @property
    def lse(self):
        if type(self._lse) is tuple:   # (buffer of all three, rows, leading shape): a view is made when it is asked for
            buf, rows, lead = self._lse
            self._lse = buf[2 * rows:].view(lead)
        return self._lse

    def __iter__(self):
        return iter((self.logprob, self.entropy, self.lse, self.top_ids, self.top_logprobs))


def _forward(logits, rows, vocab, tokens, top, stats, index):
    """logprob and entropy (rows,), the buffer that holds them and lse, and the alternatives."""
    device = logits.device
    buf = torch.empty(3 * rows, dtype=torch.float32, device=device)
    at = buf.data_ptr()
    if top:
        shape, strides = (rows, top), (top, 1)
        ids = torch.empty_strided(shape, strides, dtype=torch.int32, device=device)
        tops = torch.empty_strided(shape, strides, dtype=torch.float32, device=device)
        ids_at, tops_at = ids.data_ptr(), tops.data_ptr()
    else:
        ids = tops = ids_at = tops_at = None
    code = ops().ygg_token_logprobs(
        index, DTYPES[logits.dtype], rows, vocab, logits.data_ptr(), logits.stride(0), tokens.data_ptr(),
        tokens.element_size(), top, at, at + 4 * rows, at + 8 * rows, ids_at, tops_at,
        stats.data_ptr() if stats is not None else None, _raw_stream(index))
    if code:
        check(code, "ygg_token_logprobs")
    one = (rows,)
    return buf.as_strided(one, (1,), 0), buf.as_strided(one, (1,), rows), buf, ids, tops


class _TokenLogprobs(torch.autograd.Function):
    """logprob, entropy, lse and top_logprobs of logits; the ids, which carry no gradient, are put into `box`."""

    @staticmethod
    def forward(ctx, logits, tokens, top, box):
        rows, vocab = logits.shape
        index = logits.get_device()
        stats = torch.empty_strided((rows, 4), (4, 1), dtype=torch.float32, device=logits.device)
        logprob, entropy, buf, ids, tops = _forward(logits, rows, vocab, tokens, top, stats, index)
        ctx.save_for_backward(logits, tokens, stats, ids)
        ctx.sizes = rows, vocab, top, index
        ctx.set_materialize_grads(False)
        box.append(ids)
        return logprob, entropy, buf.as_strided((rows,), (1,), 2 * rows), tops

    @staticmethod
    def backward(ctx, g_logprob, g_entropy, g_lse, g_top):
        if torch.is_grad_enabled():   # create_graph
            raise NotImplementedError("token_logprobs has no second derivative")
        logits, tokens, stats, ids = ctx.saved_tensors
        rows, vocab, top, index = ctx.sizes
        step, dtype = logits.stride(0), logits.dtype
        # rows that lie to the 16-byte boundary as the logits' do move 16 bytes at a time
        per = 16 // logits.element_size()
        wide = -(-vocab // per) * per if step % per == 0 else vocab
        grad = torch.empty_strided((rows, vocab), (wide, 1), dtype=dtype, device=logits.device)
        keep = [_arrived(g) for g in (g_logprob, g_entropy, g_lse, g_top)]
        code = ops().ygg_token_logprobs_backward(
            index, DTYPES[dtype], rows, vocab, logits.data_ptr(), step, tokens.data_ptr(), tokens.element_size(), top,
            ids.data_ptr() if top else None, stats.data_ptr(), *[None if g is None else g.data_ptr() for g in keep],
            grad.data_ptr(), wide, _raw_stream(index))
        if code:
            check(code, "ygg_token_logprobs_backward")
        return grad, None, None, None


def _arrived(g):
    """A gradient that arrives, as the kernel reads it: it may be expanded (a sum's) or of another type."""
    if g is None or (g.dtype is torch.float32 and g.is_contiguous()):
        return g
    return g.float().contiguous()


def token_logprobs(logits, tokens, top=0):
    """logits (..., V) float32, float16 or bfloat16 on a CUDA device, any row stride; tokens (...) the given token of
    each row: an int32 or int64 tensor, or host integers (range-checked: < V). A negative token is padding: logprob 0
    and no gradient from it. top: how many alternatives, 0 to min(V, 64).

    -inf logits (masked tokens) have probability 0. A row of -inf alone has logprob and lse -inf, entropy 0, gradient
    0, and alternatives by the lower index; a row that holds NaN or +inf has NaN values."""
    if not isinstance(logits, torch.Tensor) or not logits.is_cuda or logits.dtype not in DTYPES or logits.dim() < 1:
        raise ValueError("logits must be a float32, float16 or bfloat16 CUDA tensor (..., V)")
    shape = logits.shape
    lead, vocab, index = shape[:-1], shape[-1], logits.get_device()
    if vocab < 1:
        raise ValueError("logits: the vocabulary is empty")
    if not 0 <= top <= min(vocab, TOP_MAX):
        raise ValueError(f"top {top}: 0 to {min(vocab, TOP_MAX)}")
    if not isinstance(tokens, torch.Tensor) or not tokens.is_cuda:
        host = np.asarray(tokens)
        if host.size and (host.dtype.kind not in "iu" or host.max() >= vocab):
            raise ValueError(f"tokens must be integers below {vocab}")
        tokens = torch.as_tensor(np.array(host, np.int64)).to(logits.device)
    if (tokens.dtype is not torch.int32 and tokens.dtype is not torch.int64) or tokens.get_device() != index:
        raise ValueError(f"tokens must be int32 or int64 on {logits.device}")
    if tokens.shape != lead:
        raise ValueError(f"tokens {tuple(tokens.shape)} for logits {tuple(shape)}: one token for each row")
    x = logits if len(shape) == 2 else logits.reshape(-1, vocab)
    if vocab > 1 and x.stride(1) != 1:
        x = x.contiguous()
    t = tokens if tokens.is_contiguous() else tokens.contiguous()
    rows = x.shape[0]
    with _nothing if index == torch.cuda.current_device() else torch.cuda.device(index):
        if x.requires_grad and torch.is_grad_enabled():
            box = []
            logprob, entropy, lse, tops = _TokenLogprobs.apply(x, t, top, box)
            out = logprob, entropy, lse, box[0], tops
            if len(lead) != 1:
                out = [None if v is None else v.reshape(lead + v.shape[1:]) for v in out]
            return TokenLogprobs(*out)
        logprob, entropy, buf, ids, tops = _forward(x, rows, vocab, t, top, None, index)
    if len(lead) != 1:
        logprob, entropy = logprob.view(lead), entropy.view(lead)
        if top:
            ids, tops = ids.view(*lead, top), tops.view(*lead, top)
    return TokenLogprobs(logprob, entropy, (buf, rows, lead), ids, tops)


class _Nothing:
    def __enter__(self):
        return None

    def __exit__(self, *_):
        return False


_nothing = _Nothing()
