"""Cases that measure the operators between a beam's state and its next token: layer norm of the states' features with its
backward pass (`layer_norm`), an output head with 4-bit weights and group scales (`int4_linear`), the choice over beams and
vocabulary (`beam_select`) and the states in the order of that choice (`reorder_states`). `run` computes them in plain torch
operations, or through yggdrasil_b200 where `own` is true.
"""
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16, "int8": torch.int8}
END = 0   # the token after which a beam is done


def listed():
    return [
        # a 4-bit output head on one stream's state (5 layers of 256 coordinates), 256 classes: latency
        dict(name="int4_stream", op="int4", rows=1, k=1280, n=256, group=32, dtype="float32", bias=True),
        # one token through a wide head: the weights are read once
        dict(name="int4_token", op="int4", rows=1, k=4096, n=32768, group=128, dtype="bfloat16", bias=False),
        # a few beams, no size a multiple of a tile, the last group of a row cut off
        dict(name="int4_beams", op="int4", rows=7, k=1000, n=5003, group=64, dtype="float16", bias=True),
        # 64 prompts of 4 beams through a wide head
        dict(name="int4_batch", op="int4", rows=256, k=4096, n=16384, group=128, dtype="bfloat16", bias=False),
        # one prompt's 4 beams, the vocabulary of the enwik8 shapes: latency
        dict(name="select_prompt", op="select", prompts=1, beams=4, vocab=256, width=4, dtype="float32", masked=0.0,
             done=0.0),
        # the benchmark's 65 536 streams as 16 384 prompts of 4 beams, some of them done
        dict(name="select_prompts", op="select", prompts=16384, beams=4, vocab=256, width=4, dtype="float32", masked=0.0,
             done=0.1),
        # three prompts over a wide, odd vocabulary, half of it closed by a grammar
        dict(name="select_wide", op="select", prompts=3, beams=5, vocab=100003, width=5, dtype="bfloat16", masked=0.5,
             done=0.0),
        # a served batch of 8 beams over a wide vocabulary
        dict(name="select_batch", op="select", prompts=256, beams=8, vocab=32768, width=8, dtype="bfloat16", masked=0.0,
             done=0.1),
        # two prompts of 4 beams with float states of 5 layers of 256 and 57 tokens so far: latency
        dict(name="reorder_beams", op="reorder", prompts=2, beams=4, width=4, layers=5, n=256, dtype="float32", tokens=57),
        # 65 536 streams with float states of 5 layers of 256 and 64 tokens so far
        dict(name="reorder_streams", op="reorder", prompts=16384, beams=4, width=4, layers=5, n=256, dtype="float32",
             tokens=64),
        # the features of a ragged training batch, forward and backward
        dict(name="norm_ragged", op="norm", rows=1003, dim=1000, dtype="float16", grad=True),
        # a training batch, forward and backward
        dict(name="norm_train", op="norm", rows=16384, dim=4096, dtype="bfloat16", grad=True),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["int4", "int4", "select", "select", "reorder", "norm"])
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    if op == "int4":
        rows = _log_uniform(rng, 1, 256)
        k = _log_uniform(rng, 16, 16384)
        n = _log_uniform(rng, 5, 32768)
        while rows * k * n > 256 * 4096 * 16384 or k * n > 4096 * 32768:
            n = max(5, n // 2)
        return dict(op=op, rows=rows, k=k, n=n, group=rng.choice([32, 64, 128]), dtype=dtype, bias=rng.random() < 0.5)
    if op == "select":
        beams = rng.randrange(1, 17)
        width = rng.randrange(1, 17)
        vocab = _log_uniform(rng, 20, 131072)
        prompts = _log_uniform(rng, 1, 16384)
        while prompts * beams * vocab > 256 * 8 * 32768 // (2 if dtype == "float32" else 1):
            prompts = max(1, prompts // 2)
        return dict(op=op, prompts=prompts, beams=beams, vocab=vocab, width=width, dtype=dtype,
                    masked=rng.choice([0.0, 0.0, 0.3, 0.9]), done=rng.choice([0.0, 0.1, 0.5]))
    if op == "reorder":
        beams = rng.randrange(1, 17)
        width = rng.randrange(1, 17)
        prompts = _log_uniform(rng, 1, 65536 // max(beams, width))
        return dict(op=op, prompts=prompts, beams=beams, width=width, layers=rng.choice([2, 3, 4, 5]),
                    n=rng.choice([64, 96, 128, 256]), dtype=rng.choice(["int8", "float32"]), tokens=rng.randrange(1, 65))
    rows = _log_uniform(rng, 1, 65536)
    dim = _log_uniform(rng, 5, 16384)
    while rows * dim > 16384 * 4096 // (2 if dtype == "float32" else 1):
        rows = max(1, rows // 2)
    return dict(op=op, rows=rows, dim=dim, dtype=dtype, grad=rng.random() < 0.7)


# ------------------------------------------------------------------------------------------------------- prepare


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    return {"int4": _prepare_int4, "select": _prepare_select, "reorder": _prepare_reorder,
            "norm": _prepare_norm}[case["op"]](case, gen)


def _prepare_int4(c, gen):
    """Activations with a few strong channels; weights kept as 4-bit codes -8..7 with a scale for each channel and each
    group of inputs, laid out once at load. A row of codes is padded with zeros to a multiple of 128 inputs. Of 128 inputs
    (four runs of 32, each four pieces of 8), piece t of run i is the 32-bit word 4 t + i: inputs 0, 2, 4, 6 of the piece
    in its four lowest 4-bit fields, 1, 3, 5, 7 in the upper ones, each as code + 8."""
    rows, k, n, group = c["rows"], c["k"], c["n"], c["group"]
    x = torch.randn(rows, k, device="cuda", generator=gen)
    x[:, torch.randint(0, k, (max(1, k // 100),), device="cuda", generator=gen)] *= 8
    groups = -(-k // group)
    w = torch.randn(n, groups * group, device="cuda", generator=gen)
    w[:, k:] = 0
    w = w.view(n, groups, group)
    scale = (w.abs().amax(-1) / 7).to(DTYPES[c["dtype"]])
    codes = (w / scale[:, :, None].float()).round().clamp(-8, 7).view(n, -1).to(torch.int8)
    padded = torch.zeros(n, -(-k // 128) * 128, dtype=torch.uint8, device="cuda")
    padded[:, :k] = (codes[:, :k] & 15).to(torch.uint8)
    fields = (padded ^ 8).view(n, -1, 4, 4, 4, 2).permute(0, 1, 3, 2, 5, 4).reshape(n, -1, 2)
    packed = fields[:, :, 0] | fields[:, :, 1] << 4
    scale = (scale.float() / math.sqrt(k)).to(scale.dtype)
    bias = torch.randn(n, device="cuda", generator=gen) if c["bias"] else None
    return dict(c, x=x.to(DTYPES[c["dtype"]]), codes=packed, scale=scale, bias=bias)


def _prepare_select(c, gen):
    """Logits as a trained head gives them (a spread of a few nats, rows of unlike sharpness), a mask of closed tokens as
    -inf (the end stays open), scores of beams that have gone apart, and which of them are done."""
    shape = c["prompts"], c["beams"]
    spread = torch.rand(*shape, 1, device="cuda", generator=gen) * 3 + 1
    logits = torch.randn(*shape, c["vocab"], device="cuda", generator=gen) * spread
    if c["masked"]:
        closed = torch.rand(*shape, c["vocab"], device="cuda", generator=gen) < c["masked"]
        closed[:, :, :c["width"]] = False
        logits.masked_fill_(closed, -math.inf)
    scores = -30 - 3 * torch.randn(shape, device="cuda", generator=gen).abs()
    done = torch.rand(shape, device="cuda", generator=gen) < c["done"]
    done[:, 0] = False
    return dict(c, logits=logits.to(DTYPES[c["dtype"]]), scores=scores, done_before=done)


def _prepare_reorder(c, gen):
    """The states of all beams, the tokens that each has so far, and the beams that the next ones go on from."""
    rows = c["prompts"] * c["beams"]
    shape = (rows, c["layers"], c["n"])
    if c["dtype"] == "int8":
        states = torch.randint(-127, 128, shape, device="cuda", generator=gen, dtype=torch.int8)
    else:
        states = torch.randn(shape, device="cuda", generator=gen)
    tokens = torch.randint(0, 256, (rows, c["tokens"]), device="cuda", generator=gen, dtype=torch.int32)
    parents = torch.randint(0, c["beams"], (c["prompts"], c["width"]), device="cuda", generator=gen, dtype=torch.int32)
    return dict(c, states=states, history=tokens, parents=parents)


def _prepare_norm(c, gen):
    """Features whose rows differ in mean and spread, a trained weight and bias, and the gradient that arrives."""
    rows, dim = c["rows"], c["dim"]
    spread = torch.rand(rows, 1, device="cuda", generator=gen) * 2 + 0.5
    x = torch.randn(rows, dim, device="cuda", generator=gen) * spread + torch.randn(rows, 1, device="cuda", generator=gen)
    w = 1 + 0.2 * torch.randn(dim, device="cuda", generator=gen)
    b = 0.2 * torch.randn(dim, device="cuda", generator=gen)
    dtype = DTYPES[c["dtype"]]
    s = dict(c, x=x.to(dtype), weight=w.to(dtype), bias=b.to(dtype))
    if c["grad"]:
        for v in (s["x"], s["weight"], s["bias"]):
            v.requires_grad_()
        s["g"] = torch.randn(rows, dim, device="cuda", generator=gen).to(dtype)
    return s


# ----------------------------------------------------------------------------------------------------------- run


def run(state):
    return {"int4": _run_int4, "select": _run_select, "reorder": _run_reorder, "norm": _run_norm}[state["op"]](state)


def _codes(s):
    """The codes -8..7 as they are laid out (see _prepare_int4), (n, k) float32."""
    n, k = s["codes"].shape[0], s["k"]
    fields = torch.stack([s["codes"] & 15, s["codes"] >> 4], -1).view(n, -1, 4, 4, 2, 4)
    return fields.permute(0, 1, 3, 2, 5, 4).reshape(n, -1)[:, :k].float() - 8


def _run_int4(s):
    if own:
        from yggdrasil_b200 import Int4Weights, int4_linear
        return int4_linear(s["x"], Int4Weights(s["codes"], s["scale"], s["k"], s["group"]), bias=s["bias"])
    w = _codes(s) * s["scale"].float().repeat_interleave(s["group"], 1)[:, :s["k"]]
    y = s["x"].float() @ w.T
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(s["x"].dtype)


def _run_select(s):
    if own:
        from yggdrasil_b200 import beam_select
        out = beam_select(s["logits"], s["scores"], s["width"], done=s["done_before"], end=END)
        return {"scores": out.scores, "tokens": out.tokens, "parents": out.parents, "done": out.done}
    # in 64 bits: continuations of two beams may be nearer to each other than 32 bits tell
    x = s["logits"].double()
    shifted = x - x.amax(-1, keepdim=True)
    total = s["scores"].double()[:, :, None] + (shifted - shifted.exp().sum(-1, keepdim=True).log())
    only = torch.full_like(total, -math.inf)
    only[:, :, END] = s["scores"].double()
    total = torch.where(s["done_before"][:, :, None], only, total)
    value, at = total.flatten(1).sort(dim=1, descending=True, stable=True)
    value, at = value[:, :s["width"]], at[:, :s["width"]]
    parents, tokens = at // s["vocab"], at % s["vocab"]
    done = s["done_before"].gather(1, parents)
    tokens = torch.where(done, END, tokens)
    return {"scores": value.float(), "tokens": tokens.int(), "parents": parents.int(), "done": done | (tokens == END)}


def _run_reorder(s):
    if own:
        from yggdrasil_b200 import reorder_states
        states, history = reorder_states(s["parents"], s["states"], s["history"])
        return {"states": states, "history": history}
    first = torch.arange(s["prompts"], device="cuda")[:, None] * s["beams"]
    rows = (first + s["parents"]).flatten()
    return {"states": s["states"][rows], "history": s["history"][rows]}


def _run_norm(s, eps=1e-5):
    if own:
        from yggdrasil_b200 import layer_norm
        y = layer_norm(s["x"], s["weight"], s["bias"], eps)
        if not s["grad"]:
            return y
        dx, dw, db = torch.autograd.grad(y, [s["x"], s["weight"], s["bias"]], s["g"])
        return {"y": y, "dx": dx, "dw": dw, "db": db}
    dtype = s["x"].dtype
    x, w, b = (s[name].detach().float() for name in ("x", "weight", "bias"))
    centred = x - x.mean(-1, keepdim=True)
    r = ((centred * centred).mean(-1, keepdim=True) + eps).rsqrt()
    hat = centred * r
    y = (hat * w + b).to(dtype)
    if not s["grad"]:
        return y
    g = s["g"].float()
    gw = g * w
    dx = r * (gw - gw.mean(-1, keepdim=True) - hat * (gw * hat).mean(-1, keepdim=True))
    return {"y": y, "dx": dx.to(dtype), "dw": (g * hat).sum(0).to(dtype), "db": g.sum(0).to(dtype)}


# ---------------------------------------------------------------------------------------------------------- work


def work(case):
    c = case
    size = {"float32": 4, "int8": 1}.get(c["dtype"], 2)
    if c["op"] == "int4":
        rows, k, n = c["rows"], c["k"], c["n"]
        weights = n * (k / 2 + size * -(-k // c["group"]) + (4 if c["bias"] else 0))
        return {"bytes": weights + rows * (k + n) * size, "flops": 2 * rows * k * n}
    if c["op"] == "select":
        # a done beam's logits are not needed: it goes on with the end alone
        beams = c["prompts"] * c["beams"]
        read = c["prompts"] + (beams - c["prompts"]) * (1 - c["done"])
        return {"bytes": read * c["vocab"] * size + 5 * beams + c["prompts"] * c["width"] * 13,
                "flops": 4 * read * c["vocab"]}
    if c["op"] == "reorder":
        # each of a prompt's `width` next beams goes on from any of its beams: some are read for several, some for none
        row = c["layers"] * c["n"] * size + 4 * c["tokens"]
        read = c["prompts"] * c["beams"] * (1 - (1 - 1 / c["beams"]) ** c["width"])
        return {"bytes": row * (read + c["prompts"] * c["width"]) + 4 * c["prompts"] * c["width"], "flops": 0}
    cells = c["rows"] * c["dim"]
    return {"bytes": cells * size * (4 if c["grad"] else 2) + c["dim"] * size * (4 if c["grad"] else 2),
            "flops": cells * (20 if c["grad"] else 7)}


# --------------------------------------------------------------------------------------------------------- exact


def exact(case, seed):
    s = prepare(case, seed)
    return {"int4": _exact_int4, "select": _exact_select, "reorder": _exact_reorder, "norm": _exact_norm}[case["op"]](s)


def _exact_int4(s):
    """sum_k x_k (code_k scale_g(k)) + b, the code of input k looked up where the layout has it."""
    k = torch.arange(s["k"], device="cuda")
    word = k // 128 * 16 + k % 32 // 8 * 4 + k % 128 // 32
    field = k % 8 // 2 + k % 2 * 4
    code = (s["codes"].long()[:, word * 4 + field // 2] >> (field % 2 * 4)) % 16 - 8
    y = s["x"].double() @ (code * s["scale"].double()[:, k // s["group"]]).T
    return y if s["bias"] is None else y + s["bias"].double()


def _exact_select(s):
    """The log-probability of each continuation, a done beam's end alone at 0, with the beam's score; ordered by prompt."""
    out = {"scores": [], "tokens": [], "parents": [], "done": []}
    step = max(1, (1 << 24) // (s["beams"] * s["vocab"]))
    for i in range(0, s["prompts"], step):
        x, done = s["logits"][i:i + step].double(), s["done_before"][i:i + step]
        total = x - torch.logsumexp(x, -1, keepdim=True)
        total[done] = -math.inf
        total[:, :, END].masked_fill_(done, 0.0)
        total += s["scores"][i:i + step].double()[:, :, None]
        flat = total.reshape(len(x), -1)
        best = torch.argsort(flat, dim=1, descending=True, stable=True)[:, :s["width"]]
        parent = torch.div(best, s["vocab"], rounding_mode="floor")
        was = torch.take_along_dim(done, parent, 1)
        token = (best - parent * s["vocab"]).masked_fill(was, END)
        out["scores"].append(torch.take_along_dim(flat, best, 1))
        out["tokens"].append(token.int())
        out["parents"].append(parent.int())
        out["done"].append(was | (token == END))
    return {name: torch.cat(v) for name, v in out.items()}


def _exact_reorder(s):
    parents = s["parents"].tolist()
    rows = [p * s["beams"] + b for p, chosen in enumerate(parents) for b in chosen]
    rows = torch.tensor(rows, device="cuda")
    return {"states": s["states"].index_select(0, rows), "history": s["history"].index_select(0, rows)}


def _exact_norm(s, eps=1e-5):
    x, w, b = (s[name].detach().double().requires_grad_() for name in ("x", "weight", "bias"))
    mean = x.sum(-1, keepdim=True) / s["dim"]
    var = ((x - mean) ** 2).sum(-1, keepdim=True) / s["dim"]
    y = (x - mean) / torch.sqrt(var + eps) * w + b
    if not s["grad"]:
        return y.detach()
    dx, dw, db = torch.autograd.grad(y, [x, w, b], s["g"].double())
    return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}
