"""Cases that measure the operators a served model's answers go through: the int8 output head (`int8_linear`), the
log-probabilities of its logits (`token_logprobs`, with its gradient) and the pages of the streams' states
(`StateCache`). `run` computes them in plain torch operations, or through yggdrasil_b200 where `own` is true.
"""
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16, "int8": torch.int8}


def listed():
    return [
        # one stream's decode step with 5 alternatives, the vocabulary of the enwik8 shapes: latency
        dict(name="logprobs_stream", op="logprobs", rows=1, vocab=256, dtype="float32", top=5, masked=0.0, grad=False),
        # the benchmark's 65 536 streams on the 730M enwik8 shape: one decode step's answers
        dict(name="logprobs_streams", op="logprobs", rows=65536, vocab=256, dtype="float32", top=5, masked=0.0,
             grad=False),
        # a few beams over a wide, odd vocabulary, half of it closed by a grammar
        dict(name="logprobs_wide", op="logprobs", rows=7, vocab=100003, dtype="bfloat16", top=20, masked=0.5,
             grad=False),
        # a training batch: log-probability and entropy of the targets, and the gradient of the logits
        dict(name="logprobs_train", op="logprobs", rows=8192, vocab=32768, dtype="bfloat16", top=0, masked=0.0,
             grad=True),
        # an output head on one stream's state (5 layers of 256 coordinates), 256 classes: latency
        dict(name="head_stream", op="linear", rows=1, k=1280, n=256, dtype="float32", bias=True),
        # one token through a wide head: the weights are read once
        dict(name="linear_token", op="linear", rows=1, k=4096, n=32768, dtype="bfloat16", bias=False),
        # a ragged batch, no size a multiple of a tile
        dict(name="linear_ragged", op="linear", rows=77, k=1000, n=5003, dtype="float16", bias=True),
        # a prompt's or a training batch's rows: bound by the tensor cores
        dict(name="linear_batch", op="linear", rows=8192, k=4096, n=16384, dtype="bfloat16", bias=False),
        # 8 beams forked from a few parents (states of the enwik8 large shape, fp32): latency
        dict(name="fork_beams", op="fork", streams=64, active=32, forks=8, pages=1, layers=5, n=256, dtype="float32"),
        # half of the benchmark's streams forked (int8 states of 4 layers of 128), a snapshot behind each
        dict(name="fork_streams", op="fork", streams=131072, active=65536, forks=65536, pages=2, layers=4, n=128,
             dtype="int8"),
        # a few streams of a server end, the rest moves together
        dict(name="retire_some", op="retire", streams=300, active=257, forks=33, pages=3, layers=4, n=96,
             dtype="int8"),
        # half of 65 536 streams with fp32 states end at once
        dict(name="retire_half", op="retire", streams=65536, active=65536, forks=32768, pages=2, layers=5, n=256,
             dtype="float32"),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["logprobs", "logprobs", "linear", "linear", "fork", "retire"])
    if op == "logprobs":
        rows = _log_uniform(rng, 1, 65536)
        vocab = _log_uniform(rng, 5, min(131072, max(256, (1 << 28) // rows)))
        vocab = rng.choice([vocab, vocab, 5, 256]) if rows > 1024 else vocab
        return dict(op=op, rows=rows, vocab=vocab, dtype=rng.choice(["float32", "bfloat16", "float16"]),
                    top=min(vocab, rng.choice([0, 1, 5, 20, 32])), masked=rng.choice([0.0, 0.0, 0.3, 0.9]),
                    grad=rng.random() < 0.4)
    if op == "linear":
        rows = _log_uniform(rng, 1, 8192)
        k = _log_uniform(rng, 16, 8192)
        n = _log_uniform(rng, 5, 32768)
        while rows * k * n > 8192 * 4096 * 16384:
            n = max(5, n // 2)
        return dict(op=op, rows=rows, k=k, n=n, dtype=rng.choice(["float32", "bfloat16", "float16"]),
                    bias=rng.random() < 0.5)
    active = _log_uniform(rng, 16, 65536)
    layers, n = rng.choice([2, 3, 4, 5, 6]), rng.choice([64, 96, 128, 256])
    dtype = rng.choice(["int8", "float32"])
    pages = rng.choice([1, 2, 3, 5])
    forks = max(1, int(active * rng.uniform(0.05, 0.9)))
    while active * (pages + 1) * layers * n * (4 if dtype == "float32" else 1) > 600_000_000:
        active, forks = max(16, active // 2), max(1, forks // 2)
    return dict(op=op, streams=active + (forks if op == "fork" else rng.randrange(0, 50)), active=active, forks=forks,
                pages=pages, layers=layers, n=n, dtype=dtype)


# ------------------------------------------------------------------------------------------------------- prepare


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    return {"logprobs": _prepare_logprobs, "linear": _prepare_linear, "fork": _prepare_cache,
            "retire": _prepare_cache}[case["op"]](case, gen)


def _prepare_logprobs(c, gen):
    """Logits as a trained head gives them (a spread of a few nats, rows of unlike sharpness), the given tokens (3 in
    100 are padding, -1), a mask of closed tokens as -inf, and the gradients that arrive from the loss."""
    rows, vocab = c["rows"], c["vocab"]
    spread = torch.rand(rows, 1, device="cuda", generator=gen) * 3 + 1
    logits = torch.randn(rows, vocab, device="cuda", generator=gen) * spread
    tokens = torch.randint(0, vocab, (rows,), device="cuda", generator=gen, dtype=torch.int32)
    if c["masked"]:
        closed = torch.rand(rows, vocab, device="cuda", generator=gen) < c["masked"]
        closed.scatter_(1, tokens.long()[:, None], False)
        logits.masked_fill_(closed, -math.inf)
    padding = torch.rand(rows, device="cuda", generator=gen) < 0.03
    if rows > 32:
        tokens.masked_fill_(padding, -1)
    s = dict(c, logits=logits.to(DTYPES[c["dtype"]]), tokens=tokens)
    if c["grad"]:
        s["logits"].requires_grad_()
        s["g_logprob"] = torch.randn(rows, device="cuda", generator=gen)
        s["g_entropy"] = torch.randn(rows, device="cuda", generator=gen) * 0.1
        if c["top"]:
            s["g_top"] = torch.randn(rows, c["top"], device="cuda", generator=gen) * 0.1
    return s


def _prepare_linear(c, gen):
    """Activations with a few strong channels; weights kept in int8 with a scale for each output channel, their rows
    padded to 16 bytes as they are laid out once at load."""
    rows, k, n = c["rows"], c["k"], c["n"]
    x = torch.randn(rows, k, device="cuda", generator=gen)
    x[:, torch.randint(0, k, (max(1, k // 100),), device="cuda", generator=gen)] *= 8
    w = torch.randn(n, k, device="cuda", generator=gen) / math.sqrt(k)
    codes, scale = _quantize(w)
    weight = torch.zeros(n, (k + 15) // 16 * 16, dtype=torch.int8, device="cuda")[:, :k]
    weight.copy_(codes)
    bias = torch.randn(n, device="cuda", generator=gen) if c["bias"] else None
    return dict(c, x=x.to(DTYPES[c["dtype"]]), weight=weight, scale=scale, bias=bias)


def _prepare_cache(c, gen):
    """A cache in use: `active` streams hold 1 to `pages` pages each, scattered over the pool; some share all pages
    but the last with a neighbour that they were forked from. `book` holds the table, the lengths and the counts of
    references one after another; `before` is its state before the call, which a pass starts from."""
    streams, active, forks, m = c["streams"], c["active"], c["forks"], c["pages"]
    pool = active * m + (forks if c["op"] == "fork" else 0) + 8
    book = torch.zeros(streams * (m + 1) + pool, dtype=torch.int32, device="cuda")
    table, length, refs = _book(book, streams, m)
    table.fill_(-1)
    which = torch.randperm(streams, device="cuda", generator=gen)
    used, rest = which[:active], which[active:]
    lens = torch.randint(1, m + 1, (active,), device="cuda", generator=gen, dtype=torch.int32)
    rows = torch.randperm(pool, device="cuda", generator=gen)[:active * m].view(active, m).int()
    even = torch.arange(active, device="cuda") // 2 * 2
    shared = (torch.rand(active, device="cuda", generator=gen) < 0.5) & (even != torch.arange(active, device="cuda"))
    lens = torch.where(shared, lens[even], lens)
    behind = torch.arange(m, device="cuda")[None] < lens[:, None] - 1
    rows = torch.where(shared[:, None] & behind, rows[even], rows)
    held = torch.arange(m, device="cuda")[None] < lens[:, None]
    table[used] = torch.where(held, rows, -1)
    length[used] = lens
    refs.copy_(torch.bincount(rows[held].long(), minlength=pool))
    shape = (pool, c["layers"], c["n"])
    if c["dtype"] == "int8":
        pages = torch.randint(-127, 128, shape, device="cuda", generator=gen, dtype=torch.int8)
    else:
        pages = torch.randn(shape, device="cuda", generator=gen)
    s = dict(c, book=book, before=book.clone(), page_data=pages)
    if c["op"] == "fork":
        s["parents"] = used[torch.randint(0, active, (forks,), device="cuda", generator=gen)].int()
        s["children"] = rest[:forks].int()
    else:
        s["ended"] = used[torch.randperm(active, device="cuda", generator=gen)[:forks]].int()
    return s


def _book(book, streams, m):
    return book[:streams * m].view(streams, m), book[streams * m:streams * (m + 1)], book[streams * (m + 1):]


# ----------------------------------------------------------------------------------------------------------- run


def run(state):
    return {"logprobs": _run_logprobs, "linear": _run_linear, "fork": _run_cache,
            "retire": _run_cache}[state["op"]](state)


def _run_logprobs(s):
    if own:
        from yggdrasil_b200 import token_logprobs
        out = token_logprobs(s["logits"], s["tokens"], top=s["top"])
        got = {"logprob": out.logprob, "entropy": out.entropy}
        if s["top"]:
            got |= {"top_ids": out.top_ids, "top_logprobs": out.top_logprobs}
        if s["grad"]:
            back = [(out.logprob, s["g_logprob"]), (out.entropy, s["g_entropy"])]
            back += [(out.top_logprobs, s["g_top"])] if s["top"] else []
            got["grad"], = torch.autograd.grad([o for o, _ in back], [s["logits"]], [g for _, g in back])
        return got
    logits = s["logits"].detach().float()
    tokens = s["tokens"].long()
    at = tokens.clamp(min=0)[:, None]
    given = (tokens >= 0).float()
    shifted = logits - logits.amax(-1, keepdim=True)
    e = shifted.exp()
    total = e.sum(-1, keepdim=True)
    logp = shifted - total.log()
    p = e / total
    entropy = -torch.where(p > 0, p * logp, 0.0).sum(-1)
    got = {"logprob": torch.where(tokens >= 0, logp.gather(1, at)[:, 0], 0.0), "entropy": entropy}
    top = s["top"]
    if top:
        ids = logits.sort(stable=True, dim=-1, descending=True)[1][:, :top]
        got |= {"top_ids": ids.int(), "top_logprobs": logp.gather(1, ids)}
    if s["grad"]:
        g = s["g_logprob"] * given
        total = g + (s["g_top"].sum(-1) if top else 0.0)
        open_ = torch.where(p > 0, logp, 0.0)
        grad = -p * (total[:, None] + s["g_entropy"][:, None] * (open_ + entropy[:, None]))
        grad.scatter_add_(1, at, g[:, None])
        if top:
            grad.scatter_add_(1, ids, s["g_top"])
        got["grad"] = grad.to(s["logits"].dtype)
    return got


def _quantize(x):
    """Codes in [-127, 127] and the scale of each row: the scale is the row's largest magnitude / 127, a code the
    nearest integer (ties to even) of the value times 127 / that magnitude. (Both divisions are tensor by tensor, so
    that they round once; torch multiplies by a reciprocal for plain numbers.)"""
    most = x.abs().amax(-1)
    full = torch.full_like(most, 127.0)
    inverse = torch.where(most > 0, full / most, 0.0)
    return (x * inverse[:, None]).round().clamp(-127, 127), most / full


def _run_linear(s):
    if own:
        from yggdrasil_b200 import int8_linear
        return int8_linear(s["x"], s["weight"], s["scale"], bias=s["bias"])
    codes, scale = _quantize(s["x"].float())
    y = (codes @ s["weight"].float().T) * scale[:, None] * s["scale"]
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(s["x"].dtype)


def _run_cache(s):
    book, pages = s["book"], s["page_data"]
    book.copy_(s["before"])
    table, length, refs = _book(book, s["streams"], s["pages"])
    if own:
        from yggdrasil_b200 import StateCache
        cache = StateCache(pages, table, length, refs)
        if s["op"] == "fork":
            cache.fork(s["parents"], s["children"])
            return {"book": book, "pages": pages}
        cache.free(s["ended"])
        return {"live": cache.compact(), "book": book, "pages": pages}
    ids = torch.arange(len(refs), device=refs.device)
    if s["op"] == "fork":  # every parent here holds pages, and the pool has one for each fork
        parents, children = s["parents"].long(), s["children"].long()
        fresh = (refs == 0).nonzero()[:len(parents), 0]
        rows, last = table[parents], length[parents].long()[:, None] - 1
        pages[fresh] = pages[rows.gather(1, last)[:, 0].long()]
        behind = torch.arange(s["pages"], device=refs.device)[None] < last
        refs.scatter_add_(0, rows.clamp(min=0).long().flatten(), behind.int().flatten())
        refs[fresh] = 1
        table[children] = rows.scatter(1, last, fresh[:, None].int())
        length[children] = length[parents]
        return {"book": book, "pages": pages}
    ended = s["ended"].long()
    rows = table[ended]
    refs.scatter_add_(0, rows.clamp(min=0).long().flatten(), -(rows >= 0).int().flatten())
    table[ended] = -1
    length[ended] = 0
    live = (refs > 0).sum()
    hole, mover = ((refs == 0) & (ids < live)).nonzero()[:, 0], ((refs > 0) & (ids >= live)).nonzero()[:, 0]
    pages[hole] = pages[mover]
    refs[hole] = refs[mover]
    refs[mover] = 0
    ids[mover] = hole
    table.copy_(torch.where(table >= 0, ids[table.clamp(min=0).long()].int(), -1))
    return {"live": live.int(), "book": book, "pages": pages}


# ---------------------------------------------------------------------------------------------------------- work


def work(case):
    c = case
    size = {"float32": 4, "int8": 1}.get(c["dtype"], 2)
    if c["op"] == "logprobs":
        rows, vocab = c["rows"], c["vocab"]
        each = 4 + 8 + 8 * c["top"] + (4 * (2 + c["top"]) if c["grad"] else 0)
        cells = rows * vocab
        return {"bytes": cells * size * (2 if c["grad"] else 1) + rows * each,
                "flops": cells * (13 if c["grad"] else 7)}
    if c["op"] == "linear":
        rows, k, n = c["rows"], c["k"], c["n"]
        return {"bytes": rows * k * size + n * k + rows * n * size + n * (8 if c["bias"] else 4),
                "flops": 2 * rows * k * n}
    page = c["layers"] * c["n"] * size
    mean = (c["pages"] + 1) / 2
    pool = c["active"] * c["pages"] + (c["forks"] if c["op"] == "fork" else 0) + 8
    book = 8 * (c["streams"] * (c["pages"] + 1) + pool)   # read and written once to start from
    if c["op"] == "fork":
        return {"bytes": book + c["forks"] * (2 * page + 8 + 8 * mean), "flops": 0}
    # a stream's last page is its own; a quarter of the streams share the others with a neighbour
    left = (c["active"] - c["forks"]) * (1 + 0.8 * (mean - 1))
    moved = left * (1 - left / pool)
    return {"bytes": book + 4 * c["forks"] + 2 * page * moved, "flops": 0}


# --------------------------------------------------------------------------------------------------------- exact


def exact(case, seed):
    s = prepare(case, seed)
    return {"logprobs": _exact_logprobs, "linear": _exact_linear, "fork": _exact_fork,
            "retire": _exact_retire}[case["op"]](s)


def _exact_logprobs(s):
    """log softmax, -sum p log p, the largest entries, and the derivative of g . log p + g_H H, in blocks of rows."""
    got = {}
    rows, step = len(s["tokens"]), max(1, (1 << 26) // s["logits"].shape[1])
    for i in range(0, rows, step):
        x = s["logits"].detach()[i:i + step].double()
        t = s["tokens"][i:i + step].long()
        row = torch.arange(len(t), device=t.device)
        logp = x - torch.logsumexp(x, -1, keepdim=True)
        p = torch.exp(logp)
        plogp = torch.nan_to_num(p * logp, nan=0.0)
        h = -plogp.sum(-1)
        part = {"logprob": torch.where(t < 0, 0.0, logp[row, t]), "entropy": h}
        if s["top"]:
            ids = torch.argsort(x, dim=-1, descending=True, stable=True)[:, :s["top"]]
            part |= {"top_ids": ids.int(), "top_logprobs": torch.take_along_dim(logp, ids, 1)}
        if s["grad"]:
            g = torch.where(t < 0, 0.0, s["g_logprob"][i:i + step].double())
            weight = torch.zeros_like(x)
            weight[row, t.clamp(min=0)] = g
            if s["top"]:
                weight.scatter_add_(1, ids, s["g_top"][i:i + step].double())
            ge = s["g_entropy"][i:i + step].double()[:, None]
            part["grad"] = weight - p * weight.sum(-1, keepdim=True) - ge * (plogp + p * h[:, None])
        for name, v in part.items():
            got.setdefault(name, []).append(v)
    return {name: torch.cat(v) for name, v in got.items()}


def _exact_linear(s):
    x = s["x"].double()
    most = x.abs().max(-1, keepdim=True).values
    codes = torch.round(x * 127 / most.clamp(min=1e-300))
    y = (codes * (most / 127)) @ (s["weight"].double() * s["scale"].double()[:, None]).T
    return y if s["bias"] is None else y + s["bias"].double()


def _host_cache(s):
    table, length, refs = (v.tolist() for v in _book(s["before"].cpu(), s["streams"], s["pages"]))
    return table, length, refs, s["page_data"].cpu().numpy().copy()


def _as_book(table, length, refs):
    return torch.tensor([p for row in table for p in row] + length + refs, dtype=torch.int32)


def _exact_fork(s):
    table, length, refs, pages = _host_cache(s)
    free = iter([p for p, r in enumerate(refs) if r == 0])
    for parent, child in zip(s["parents"].tolist(), s["children"].tolist()):
        row = list(table[parent])
        for j in range(length[parent] - 1):
            refs[row[j]] += 1
        fresh = next(free)
        pages[fresh] = pages[row[length[parent] - 1]]
        refs[fresh] = 1
        row[length[parent] - 1] = fresh
        table[child], length[child] = row, length[parent]
    return {"book": _as_book(table, length, refs), "pages": pages}


def _exact_retire(s):
    table, length, refs, pages = _host_cache(s)
    for stream in s["ended"].tolist():
        for p in table[stream][:length[stream]]:
            refs[p] -= 1
        table[stream], length[stream] = [-1] * s["pages"], 0
    live = sum(r > 0 for r in refs)
    high = iter([p for p in range(live, len(refs)) if refs[p] > 0])
    new = list(range(len(refs)))
    for hole in [p for p in range(live) if refs[p] == 0]:
        p = next(high)
        new[p], refs[hole], refs[p], pages[hole] = hole, refs[p], 0, pages[p]
    table = [[new[p] if p >= 0 else -1 for p in row] for row in table]
    return {"live": torch.tensor(live, dtype=torch.int32), "book": _as_book(table, length, refs), "pages": pages}
