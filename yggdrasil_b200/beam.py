"""Beam search: the choice over beams and alternatives, the states of the streams that go on in its order, and, if asked for, an
output head of one's own with 8-bit or 4-bit weights on the (normalised) states, run together.

    from yggdrasil_b200 import Yggdrasil
    from yggdrasil_b200.beam import beam_search
    model = Yggdrasil.load("model.bin", backend="b200")
    tokens, scores = beam_search(model, prompt, n=32, width=4)   # (B, 4, L + 32), (B, 4) nats, best first

Every step: model.step (or the head on the new states) -> beam_select over the beams' continuations -> reorder_states of the
states and the tokens so far -> the next step.
"""
from __future__ import annotations

import numpy as np
import torch

from .linear import Int4Weights, QuantizedRows, int4_linear, int8_linear, linear_status
from .norm import layer_norm
from .select import beam_select, reorder_states


def state_features(state):
    """The states of a batch (B, layers, n) as rows (B, layers n) for int8_linear: int8 states are codes already, with a
    scale of 1; float states are quantised row by row."""
    rows = state.reshape(state.shape[0], -1)
    if rows.dtype == torch.int8:
        return QuantizedRows(rows, torch.ones(rows.shape[0], dtype=torch.float32, device=rows.device))
    return rows


def state_head(weight, scale=None, bias=None, norm=None):
    """An output head on the states: weight int8 (classes, layers n) and scale (classes,) as quantize_rows gives them, or
    Int4Weights of as many inputs (and no scale); norm: a weight and a bias (layers n,) of a layer norm that the states go
    through first. Returns a function state -> logits (B, classes) float32."""
    if isinstance(weight, Int4Weights) and scale is not None:
        raise ValueError("Int4Weights hold their scales")

    def head(state):
        if norm is None and not isinstance(weight, Int4Weights):
            return int8_linear(state_features(state), weight, scale, bias, out_dtype=torch.float32)
        x = state.reshape(state.shape[0], -1)
        if x.dtype == torch.int8:   # codes up to 127 are exact in either
            x = x.to(torch.bfloat16 if norm is None else torch.float32)
        if norm is not None:
            x = layer_norm(x, *norm)
        if isinstance(weight, Int4Weights):
            return int4_linear(x, weight, bias, out_dtype=torch.float32)
        return int8_linear(x, weight, scale, bias, out_dtype=torch.float32)

    return head


def beam_search(model, prompt, n, width=4, head=None, end=None):
    """The `width` best continuations by n tokens that a beam search finds, for prompt (L,) or (B, L) with L >= 1.

    model: a backend with init_state and step (b200 or b200f). head: state -> logits (B, classes), for instance
    state_head(...), in place of the step's own logits; its classes must be tokens of the model. end: a token after which
    a beam is done and keeps its score (it is filled up with `end`).
    Returns tokens (B, width, L + n) int64 and scores (B, width) float64 as numpy arrays, best first: the log-probability
    of the n tokens given the prompt, ties by the lower beam, then the lower token."""
    prompt = np.asarray(prompt, np.int64)
    x = np.atleast_2d(prompt)
    if x.ndim != 2 or x.shape[1] < 1:
        raise ValueError("prompt must be (L,) or (B, L) with L >= 1")
    if n < 0 or width < 1:
        raise ValueError("beam_search needs n >= 0 and width >= 1")
    rows, dev = x.shape[0], model.device
    with torch.cuda.device(dev), torch.no_grad():
        state = model.init_state(rows)
        logits = None
        for t in range(x.shape[1]):
            logits, state = model.step(x[:, t], state)
        head_of = (lambda logits, state: logits) if head is None else (lambda logits, state: head(state))
        logits = head_of(logits, state)
        classes = logits.shape[1]
        if width > min(classes, 64):
            raise ValueError(f"width {width}: at most {min(classes, 64)}")
        if end is not None and not 0 <= end < classes:
            raise ValueError(f"end {end}: a token below {classes}")
        end = None if end is None else int(end)
        scores = torch.zeros(rows, 1, dtype=torch.float64, device=dev)
        done = None if end is None else torch.zeros(rows, 1, dtype=torch.bool, device=dev)
        tokens = torch.as_tensor(x, device=dev)   # a row for each beam
        for i in range(n):
            best = beam_select(logits.reshape(rows, -1, classes), scores, width, done=done, end=end)
            scores, done = best.scores, best.done
            new = best.tokens.reshape(-1)
            if i + 1 == n:
                tokens = reorder_states(best.parents, tokens)
            else:
                tokens, state = reorder_states(best.parents, tokens, state)
            tokens = torch.cat([tokens, new[:, None].long()], 1)
            if i + 1 < n:
                logits, state = model.step(new, state)
                logits = head_of(logits, state)
        tokens = tokens.view(rows, -1, tokens.shape[1])
        if hasattr(model, "status"):
            model.status()
        if head is not None:   # its products may have given up a wait: then the logits are not to be used
            linear_status(dev)
        if n == 0:
            tokens, scores = tokens.expand(rows, width, -1), scores.expand(rows, width)
        tokens, scores = tokens.cpu().numpy(), scores.cpu().numpy()
    return (tokens[0], scores[0]) if prompt.ndim == 1 else (tokens, scores)
