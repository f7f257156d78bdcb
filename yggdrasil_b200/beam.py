"""Beam search: a step's alternatives, the states of the streams that go on from them, and, if asked for, an int8 output
head of one's own, run together.

    from yggdrasil_b200 import Yggdrasil
    from yggdrasil_b200.beam import beam_search
    model = Yggdrasil.load("model.bin", backend="b200")
    tokens, scores = beam_search(model, prompt, n=32, width=4)   # (B, 4, L + 32), (B, 4) nats, best first

Every step: model.step (or the head on the new states) -> token_logprobs with `width` alternatives -> the best `width`
of the beams' alternatives -> StateCache.fork of the beams that go on, free of the others, compact -> the next step.
"""
from __future__ import annotations

import numpy as np
import torch

from .cache import StateCache
from .linear import QuantizedRows, int8_linear, linear_status
from .logprobs import token_logprobs


def state_features(state):
    """The states of a batch (B, layers, n) as rows (B, layers n) for int8_linear: int8 states are codes already, with a
    scale of 1; float states are quantised row by row."""
    rows = state.reshape(state.shape[0], -1)
    if rows.dtype == torch.int8:
        return QuantizedRows(rows, torch.ones(rows.shape[0], dtype=torch.float32, device=rows.device))
    return rows


def state_head(weight, scale, bias=None):
    """An output head on the states: weight int8 (classes, layers n) and scale (classes,) as quantize_rows gives them.
    Returns a function state -> logits (B, classes) float32."""
    return lambda state: int8_linear(state_features(state), weight, scale, bias, out_dtype=torch.float32)


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
        # two banks of beams: a step forks one into the other. A step's new pages are taken before the old ones are free.
        beams = rows * width
        cache = StateCache.empty(2 * beams + rows, 2 * beams + rows, like=model.init_state(1))
        first = torch.arange(rows, dtype=torch.int32, device=dev) + 2 * beams
        cache.grow(first)
        cache.write(first, state)
        banks = [torch.arange(beams, dtype=torch.int32, device=dev) + k * beams for k in range(2)]
        none = torch.full((beams,), -1, dtype=torch.int32, device=dev)
        scores = torch.zeros(rows, 1, dtype=torch.float64, device=dev)
        done = torch.zeros(rows, 1, dtype=torch.bool, device=dev)
        tokens = torch.as_tensor(x, device=dev)[:, None]
        parents_of = first.view(rows, 1)
        for i in range(n):
            held = parents_of.shape[1]
            out = token_logprobs(logits, none[:rows * held], top=width)
            more = out.top_logprobs.view(rows, held, width).double()
            ids = out.top_ids.view(rows, held, width)
            if end is not None:   # a beam that is done goes on with `end` alone, at no cost
                only = torch.full_like(more, -torch.inf)
                only[:, :, 0] = 0.0
                more = torch.where(done[:, :, None], only, more)
                ids = torch.where(done[:, :, None], end, ids)
            total = (scores[:, :, None] + more).reshape(rows, -1)
            total, pick = total.sort(dim=1, descending=True, stable=True)
            scores, pick = total[:, :width], pick[:, :width]
            beam, new = pick // width, ids.reshape(rows, -1).gather(1, pick)
            tokens = torch.cat([tokens.gather(1, beam[:, :, None].expand(-1, -1, tokens.shape[2])),
                                new[:, :, None].long()], 2)
            if end is not None:
                done = done.gather(1, beam) | (new == end)
            if i + 1 == n:
                break
            children = banks[i % 2].view(rows, -1)[:, :width]
            cache.fork(parents_of.gather(1, beam).reshape(-1), children.reshape(-1))
            cache.free(parents_of.reshape(-1))
            cache.compact()   # the beams' states are pages[:beams] now: one contiguous batch, in the order of `page`
            parents_of = children
            page = cache.table[children.reshape(-1).long(), 0].long()
            batch = cache.pages[:beams]
            order = torch.empty_like(new.reshape(-1))
            order[page] = new.reshape(-1)
            logits, state = model.step(order, batch)
            batch.copy_(state)
            logits = head_of(logits, state)[page]
        cache.status()
        if hasattr(model, "status"):
            model.status()
        if head is not None:   # its products may have given up a wait: then the logits are not to be used
            linear_status(dev)
        if n == 0:
            tokens, scores = tokens.expand(rows, width, -1), scores.expand(rows, width)
        tokens, scores = tokens.cpu().numpy(), scores.cpu().numpy()
    return (tokens[0], scores[0]) if prompt.ndim == 1 else (tokens, scores)
