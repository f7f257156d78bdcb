"""token_logprobs against its definition in 64 bits: values, alternatives and gradients, at the sizes and masks where the
kernels change shape or can go wrong, and its refusals.

Tolerances. A row's sum of exponentials has a relative error of at most rel(V): 2^-21 for exp2 and its argument, and
2^-24 for each addition of the longest chain (at most 64 + V / 256 additions one after another). A log-probability
then is off by rel(V), plus the roundings of its argument: 2^-22 of (|logprob| + max |x|). The entropy log s - t / s is
off by rel(V) (1 + 3 log2 V). A gradient p (...) is off by its p's relative error, rel(V) + 2^-22 (|log p| + max |x|),
times the magnitudes of its terms, plus the rounding to its type.
"""
import math

import numpy as np
import pytest
import torch

from yggdrasil_b200 import _native

INF = math.inf
STEP = {torch.float32: 2.0 ** -23, torch.float16: 2.0 ** -10, torch.bfloat16: 2.0 ** -7}   # spacing of 1.0


def rel(vocab):
    return 2.0 ** -21 + (64 + vocab / 256) * 2.0 ** -24


def op():
    from yggdrasil_b200 import token_logprobs
    return token_logprobs


def make(rows, vocab, dtype, mask="none", seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g) * (torch.rand(rows, 1, generator=g) * 5 + 0.5) + 3
    t = torch.randint(0, vocab, (rows,), generator=g)
    if mask == "half":
        x[torch.rand(rows, vocab, generator=g) < 0.5] = -INF
    elif mask == "lowest":
        x[torch.rand(rows, vocab, generator=g) < 0.5] = torch.finfo(dtype).min
    elif mask == "one":       # one open token in a row
        keep = x.gather(1, t[:, None])
        x.fill_(-INF)
        x.scatter_(1, t[:, None], keep)
    elif mask == "empty":     # every third row has none
        x[::3] = -INF
    elif mask == "equal":
        x.fill_(1.5)
    elif mask == "coarse":    # many ties
        x = (x * 2).round() / 2
    if rows > 3:
        t[1] = -1
        t[3] = -100
    return x.to(dtype).cuda(), t.cuda()


def definition(x, t, top):
    """In 64 bits: logprob, entropy, lse, ids, top_logprobs."""
    x, t = x.detach().double().cpu(), t.cpu().long()
    lse = torch.logsumexp(x, -1)
    logp = torch.where(lse[:, None] == -INF, -INF, x - lse[:, None])
    p = torch.where(logp == -INF, 0.0, logp.exp())
    h = -torch.where(p == 0, 0.0, p * logp).sum(-1)
    lp = torch.where(t < 0, 0.0, logp.gather(1, t.clamp(min=0)[:, None])[:, 0])
    ids = x.sort(stable=True, dim=-1, descending=True)[1][:, :top]
    return lp, h, lse, ids, logp.gather(1, ids), logp, p


def close(got, want, tol, what):
    got, want = got.detach().double().cpu(), want.double()
    tol = torch.as_tensor(tol, dtype=torch.float64).expand(want.shape)
    inf = ~torch.isfinite(want)
    assert torch.equal(got[inf], want[inf]), what
    off = (got - want).abs()[~inf]
    assert bool((off <= tol[~inf]).all()), f"{what}: off by {float((off / tol[~inf]).max())} of the tolerance"


def span(x):
    x = x.detach().double().cpu()
    return torch.where(x.abs() < 1e4, x.abs(), 0.0).amax(-1)


def check_values(x, t, top, out):
    vocab = x.shape[1]
    lp, h, lse, ids, tops, logp, p = definition(x, t, top)
    most, r = span(x), rel(vocab)
    fin = lambda v: torch.where(torch.isfinite(v), v.abs(), 0.0)  # noqa: E731
    close(out.logprob, lp, r + 2.0 ** -22 * (fin(lp) + most), "logprob")
    close(out.lse, lse, r + 2.0 ** -22 * (fin(lse) + most), "lse")
    close(out.entropy, h, r * (1 + 3 * math.log2(max(2, vocab))), "entropy")
    if top:
        assert out.top_ids.dtype == torch.int32
        assert torch.equal(out.top_ids.cpu().long(), ids)
        close(out.top_logprobs, tops, r + 2.0 ** -22 * (fin(tops) + most[:, None]), "top_logprobs")
    else:
        assert out.top_ids is None and out.top_logprobs is None


SIZES = [(1, 1), (1, 2), (7, 5), (300, 5), (1, 31), (5, 33), (1, 256), (67, 256), (3, 257), (2, 1000), (3, 1024),
         (2, 1025), (5, 2049), (4, 4099), (300, 4100), (3, 8191), (2, 32768), (1, 50001), (3, 100003), (1, 262147)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,vocab", SIZES)
def test_values(rows, vocab, dtype):
    x, t = make(rows, vocab, dtype, seed=vocab)
    for top in {0, 1, min(5, vocab), min(20, vocab), min(64, vocab)}:
        check_values(x, t, top, op()(x, t, top=top))


@pytest.mark.gpu
@pytest.mark.parametrize("mask", ["half", "lowest", "one", "empty", "equal", "coarse"])
@pytest.mark.parametrize("rows,vocab", [(7, 5), (9, 256), (6, 777), (5, 5001), (4, 40000), (150, 20001)])
def test_masks_and_ties(rows, vocab, mask):
    for dtype in (torch.float32, torch.bfloat16):
        x, t = make(rows, vocab, dtype, mask, seed=vocab + 1)
        top = min(33, vocab)
        check_values(x, t, top, op()(x, t, top=top))


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [5, 256, 3000, 70000])
def test_nan_and_infinity_make_the_row_nan(vocab):
    x, t = make(6, vocab, torch.float32, seed=3)
    x[0, vocab // 2] = math.nan
    x[2, vocab - 1] = INF
    x[4] = math.nan
    t[:] = 0
    top = min(4, vocab)
    out = op()(x, t, top=top)
    for row in (0, 2, 4):
        assert all(bool(torch.isnan(v[row]).all()) for v in (out.logprob, out.entropy, out.top_logprobs))
    ranked = torch.where(torch.isnan(x), -INF, x).cpu().sort(stable=True, dim=-1, descending=True)[1][:, :top]
    assert torch.equal(out.top_ids.cpu().long(), ranked)
    keep = [1, 3, 5]
    check_values(x[keep], t[keep], top, op()(x[keep], t[keep], top=top))
    assert torch.equal(out.logprob[keep], op()(x[keep], t[keep], top=top).logprob)


@pytest.mark.gpu
def test_token_beyond_the_vocabulary_gives_nan():
    x, t = make(4, 100, torch.float32)
    t[2] = 100
    out = op()(x, t)
    assert torch.isnan(out.logprob).tolist() == [False, False, True, False]
    assert torch.isfinite(out.entropy).all()


@pytest.mark.gpu
def test_signed_zeros_tie():
    x = torch.tensor([[-0.0, 0.0, -1.0, 0.0, -0.0]], device="cuda")
    assert op()(x, [0], top=4).top_ids.tolist() == [[0, 1, 3, 4]]


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [40, 1000, 9000])
def test_strides_offsets_and_leading_shapes(vocab):
    wide, t = make(24, vocab + 3, torch.bfloat16, seed=5)
    t = (t % vocab).int()
    t[0] = -1
    for x in (wide[:, :vocab], wide[:, 1:vocab + 1], wide[:, 3:], wide[:, :vocab].T.contiguous().T, wide[::2, :vocab]):
        rows = x.shape[0]
        check_values(x, t[:rows], 7, op()(x, t[:rows], top=7))
    x = wide[:, 1:vocab + 1].unflatten(0, (2, 3, 4))
    out = op()(x, t.view(2, 3, 4), top=5)
    flat = op()(wide[:, 1:vocab + 1], t, top=5)
    assert out.top_ids.shape == (2, 3, 4, 5) and out.logprob.shape == (2, 3, 4)
    assert torch.equal(out.top_ids.flatten(0, 2), flat.top_ids) and torch.equal(out.logprob.flatten(), flat.logprob)
    one = op()(wide[0, :vocab], int(t[2]), top=2)
    assert one.logprob.shape == () and one.top_ids.shape == (2,)
    # rows that share their memory
    same = op()(wide[:1, :vocab].expand(5, vocab), t[:5], top=3)
    assert torch.equal(same.top_ids, same.top_ids[:1].expand(5, 3))


@pytest.mark.gpu
def test_no_rows():
    out = op()(torch.empty(0, 77, device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda"), top=3)
    assert out.logprob.shape == (0,) and out.top_ids.shape == (0, 3)


@pytest.mark.gpu
def test_host_tokens_and_int64_tokens_agree():
    x, t = make(9, 300, torch.float32)
    a, b, c = op()(x, t), op()(x, t.int()), op()(x, t.cpu().numpy())
    assert torch.equal(a.logprob, b.logprob) and torch.equal(a.logprob, c.logprob)


def check_grad(x, t, top, seed=0, parts=("logprob", "entropy", "lse", "top")):
    rows, vocab = x.shape
    g = torch.Generator().manual_seed(seed)
    gl, gh, gs = (torch.randn(rows, generator=g) if k in parts else None for k in ("logprob", "entropy", "lse"))
    gt = torch.randn(rows, top, generator=g) if top and "top" in parts else None
    leaf = x.detach().requires_grad_()
    out = op()(leaf, t, top=top)
    pairs = [(o, v.cuda()) for o, v in ((out.logprob, gl), (out.entropy, gh), (out.lse, gs), (out.top_logprobs, gt))
             if v is not None]
    got, = torch.autograd.grad([o for o, _ in pairs], [leaf], [v for _, v in pairs])
    assert got.dtype == x.dtype and got.shape == x.shape

    lp, h, lse, ids, tops, logp, p = definition(x, t, top)
    tc = t.cpu().long()
    zero = torch.zeros(rows, dtype=torch.float64)
    gl, gh, gs = (zero if v is None else v.double() for v in (gl, gh, gs))
    gl = torch.where(tc < 0, 0.0, gl)
    w = torch.zeros(rows, vocab, dtype=torch.float64)
    w.scatter_add_(1, tc.clamp(min=0)[:, None], gl[:, None])
    size = gl.abs() + gs.abs()
    if gt is not None:
        w.scatter_add_(1, ids, gt.double())
        size = size + gt.double().abs().sum(-1)
    open_logp = torch.where(p == 0, 0.0, logp)
    want = w + p * (gs - w.sum(-1))[:, None] - gh[:, None] * p * (open_logp + h[:, None])
    dead = lse == -INF
    want[dead] = 0
    err = rel(vocab) * (1 + 3 * math.log2(max(2, vocab))) + 2.0 ** -22 * (open_logp.abs() + span(x)[:, None])
    tol = p * err * (size[:, None] + gh.abs()[:, None] * (open_logp.abs() + h[:, None] + 1))
    tol = tol + want.abs() * STEP[x.dtype] + 2.0 ** -22 * w.abs()
    tol = tol + (2.0 ** -25 if x.dtype == torch.float16 else 1e-37)
    close(got, want, tol, "grad")
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (7, 5), (67, 256), (3, 257), (2, 1025), (4, 4099), (3, 32768),
                                        (2, 100003)])
def test_gradients(rows, vocab, dtype):
    x, t = make(rows, vocab, dtype, seed=vocab + 7)
    check_grad(x, t, min(20, vocab))
    check_grad(x, t, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("mask", ["half", "lowest", "one", "empty", "equal", "coarse"])
def test_gradients_with_masks(mask):
    for rows, vocab in ((6, 5), (9, 256), (5, 5001)):
        x, t = make(rows, vocab, torch.float32, mask, seed=11)
        got = check_grad(x, t, min(8, vocab))
        assert bool(torch.isfinite(got).all())


@pytest.mark.gpu
@pytest.mark.parametrize("parts", [("logprob",), ("entropy",), ("lse",), ("top",), ("entropy", "top")])
def test_gradients_of_single_outputs(parts):
    x, t = make(5, 1500, torch.float32, seed=13)
    check_grad(x, t, 6, parts=parts)


@pytest.mark.gpu
def test_gradients_of_strided_logits_and_expanded_arriving_gradients():
    wide, t = make(12, 3003, torch.float32, seed=17)
    for x in (wide[:, 1:3001], wide[::2, :2999], wide[:, :3000].T.contiguous().T):
        check_grad(x, (t % 2999)[:x.shape[0]], 4)
    a, b = wide.clone().requires_grad_(), wide.clone().requires_grad_()
    op()(a, t).logprob.sum().backward()               # arrives as an expanded scalar
    (op()(b, t).logprob * torch.ones(12, device="cuda")).sum().backward()
    assert torch.equal(a.grad, b.grad)
    # broadcast logits: the rows' gradients add up
    row = wide[0].clone().requires_grad_()
    op()(row.expand(12, -1), t).logprob.sum().backward()
    torch.testing.assert_close(row.grad, op_grad_sum(wide[0], t), rtol=1e-4, atol=1e-5)


def op_grad_sum(row, t):
    x = row.double().requires_grad_()
    lp = torch.log_softmax(x.expand(len(t), -1), -1).gather(1, t.clamp(min=0)[:, None])[:, 0]
    torch.where(t < 0, 0.0, lp).sum().backward()
    return x.grad.float()


@pytest.mark.gpu
def test_gradient_against_differences():
    """The directional derivative of g . logprob + g_H H in 64 bits by central differences: h = 1e-5 leaves an error of
    about h^2 in the difference and 1e-11 / h from rounding; the kernel's 32-bit gradient adds 300 terms at 2^-22."""
    x, t = make(6, 300, torch.float32, seed=19)
    g = torch.Generator().manual_seed(1)
    gl, gh = torch.randn(6, generator=g).double(), torch.randn(6, generator=g).double()
    v = torch.randn(6, 300, generator=g).double()

    def f(y):
        lp, h, *_ = definition(y, t, 0)
        return (gl * lp).sum() + (gh * h).sum()

    step = 1e-5
    want = (f(x.double().cpu() + step * v) - f(x.double().cpu() - step * v)) / (2 * step)
    leaf = x.clone().requires_grad_()
    out = op()(leaf, t)
    got, = torch.autograd.grad([out.logprob, out.entropy], [leaf], [gl.float().cuda(), gh.float().cuda()])
    assert abs(float((got.double().cpu() * v).sum()) - float(want)) < 1e-5 * (1 + abs(float(want)))


@pytest.mark.gpu
def test_another_stream_and_repeatable():
    x, t = make(40, 20000, torch.bfloat16, seed=23)
    want = op()(x, t, top=9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = op()(x, t, top=9)
    side.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_capture_into_a_graph():
    x, t = make(3, 60000, torch.float32, seed=29)
    want = op()(x, t, top=4)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = op()(x, t, top=4)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_refusals():
    f = op()
    x, t = make(4, 50, torch.float32)
    for bad in (x.double(), x.int(), x.cpu(), "x"):
        with pytest.raises(ValueError):
            f(bad, t)
    for top in (-1, 51):
        with pytest.raises(ValueError):
            f(x, t, top=top)
    with pytest.raises(ValueError):
        f(torch.randn(2, 100, device="cuda"), [0, 1], top=65)
    for bad in (t[:3], t.float(), [0, 1, 2, 50], [0.5, 1, 2, 3], t[:, None]):
        with pytest.raises(ValueError):
            f(x, bad)
    with pytest.raises(ValueError):
        f(torch.empty(3, 0, device="cuda"), [0, 0, 0])


def test_c_entry_refuses_bad_arguments():
    """Checked before any CUDA call."""
    lib = _native.ops()
    p = 256   # a pointer that nothing reads: every call below is refused
    f = lib.ygg_token_logprobs
    assert f(0, 0, -1, 5, p, 5, p, 4, 0, p, p, p, None, None, None, None) == _native.YGG_E_ARG
    assert f(0, 0, 1, 0, p, 5, p, 4, 0, p, p, p, None, None, None, None) == _native.YGG_E_ARG
    assert f(0, 0, 1, 5, p, 5, p, 3, 0, p, p, p, None, None, None, None) == _native.YGG_E_ARG
    assert f(0, 0, 1, 5, p, 5, p, 4, 6, p, p, p, p, p, None, None) == _native.YGG_E_ARG
    assert f(0, 0, 1, 100, p, 100, p, 4, 65, p, p, p, p, p, None, None) == _native.YGG_E_ARG
    assert f(0, 0, 1, 5, None, 5, p, 4, 0, p, p, p, None, None, None, None) == _native.YGG_E_ARG
    assert f(0, 0, 1, 5, p, 5, p, 4, 2, p, p, p, None, None, None, None) == _native.YGG_E_ARG
    assert f(0, 0, 1, 5, p, 5, p, 4, 0, p, p, p, None, None, p + 4, None) == _native.YGG_E_ARG
    assert f(0, 0, 0, 5, None, 5, None, 4, 0, None, None, None, None, None, None, None) == _native.YGG_OK
    b = lib.ygg_token_logprobs_backward
    assert b(0, 0, 1, 5, p, 5, p, 4, 2, None, p, None, None, None, p, p, 5, None) == _native.YGG_E_ARG
    assert b(0, 0, 1, 5, p, 5, p, 4, 0, None, None, None, None, None, None, p, 5, None) == _native.YGG_E_ARG
    assert b(0, 0, 0, 5, None, 5, None, 4, 0, None, None, None, None, None, None, None, 5, None) == _native.YGG_OK


def test_host_tensors_are_refused():
    with pytest.raises(ValueError):
        op()(torch.zeros(2, 5), [0, 1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [17, 64, 256, 700, 1024, 1100, 2600, 9000, 70001])
def test_sorted_rows_and_few_open_tokens(vocab, dtype):
    """Rows whose best entries lie side by side, and rows with fewer open tokens than alternatives."""
    x, t = make(8, vocab, dtype, seed=31)
    x[0] = x[0].sort()[0]
    x[1] = x[1].sort(descending=True)[0]
    for row, open_ in ((2, 1), (3, 3), (4, min(vocab, 40))):
        at = torch.randperm(vocab, generator=torch.Generator().manual_seed(row))[:open_].cuda()
        keep = x[row, at]
        x[row] = -INF
        x[row, at] = keep
    x[5, : vocab // 2] = x[5].max()
    x[6, vocab // 3:] = x[6].max() + 1
    for top in {1, min(5, vocab), min(32, vocab), min(33, vocab), min(64, vocab)}:
        check_values(x, t, top, op()(x, t, top=top))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab", [(1, 600001), (2, 1 << 20), (1, 3000000)])
def test_very_wide_rows(rows, vocab):
    """Rows cut into segments of more than one run."""
    for dtype in (torch.float32, torch.float16):
        x, t = make(rows, vocab, dtype, "coarse", seed=37)
        for top in (0, 3, 64):
            check_values(x, t, top, op()(x, t, top=top))
    x[0] = -INF
    x[0, vocab - 2] = 0.5
    check_values(x, t, 20, op()(x, t, top=20))


@pytest.mark.gpu
def test_no_second_derivative():
    x, t = make(3, 40, torch.float32)
    leaf = x.requires_grad_()
    with pytest.raises(NotImplementedError):
        torch.autograd.grad(op()(leaf, t).logprob.sum(), leaf, create_graph=True)


@pytest.mark.gpu
def test_gradient_of_the_alternatives_alone_and_of_float64_arrivals():
    x, t = make(6, 700, torch.bfloat16, seed=41)
    a, b = x.clone().requires_grad_(), x.clone().requires_grad_()
    out = op()(a, t, top=3)
    assert not out.top_ids.requires_grad and out.top_logprobs.requires_grad
    g = torch.randn(6, 3, device="cuda")
    out.top_logprobs.backward(g)
    out = op()(b, t, top=3)
    (out.top_logprobs.double() * g.double()).sum().backward()
    assert torch.equal(a.grad, b.grad) and a.grad.shape == x.shape


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab,step", [(1100, 128), (8192, 512), (8192, 1024), (32768, 1024), (32768, 4096), (120000, 16384)])
def test_best_entries_a_fixed_step_apart(vocab, step, dtype):
    """The best entries lie `step` apart, in few of the bins that a bound is taken from, alone or with a tie of most others."""
    x, t = make(6, vocab, dtype, seed=41)
    x = torch.where(torch.arange(vocab, device="cuda") % step < 8, x + 50, x)
    x[3:] = torch.where(x[3:] > 30, x[3:], torch.tensor(1.0, device="cuda", dtype=dtype))
    for top in (1, 9, 20, 33, 64):
        check_values(x, t, top, op()(x, t, top=top))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [5, 8, 9, 20, 200, 5000])
def test_empty_rows_have_no_gradient_whatever_arrives(vocab, dtype):
    """What arrives at a row of -inf alone is often not finite (its logprob is -inf, a difference of two such NaN)."""
    x, t = make(9, vocab, dtype, "empty", seed=43)
    t = t.abs() % vocab
    empty = torch.arange(9, device="cuda") % 3 == 0
    for bad in (math.nan, INF, -INF):
        for which in ("logprob", "entropy", "lse", "top_logprobs"):
            leaf = x.clone().requires_grad_()
            out = op()(leaf, t, top=4)
            g = torch.where(empty, bad, 0.5)
            o = getattr(out, which)
            got, = torch.autograd.grad(o, leaf, g if o.dim() == 1 else g[:, None].expand(o.shape))
            assert not bool(got[empty].any()), (bad, which)
            g = torch.where(empty, 0.0, 0.5)
            out = op()(leaf, t, top=4)
            o = getattr(out, which)
            want, = torch.autograd.grad(o, leaf, g if o.dim() == 1 else g[:, None].expand(o.shape))
            assert torch.equal(got, want)


@pytest.mark.gpu
def test_tangents_are_refused():
    """A forward-mode derivative is refused, not lost: of the logits, and of what arrives at the gradient."""
    import torch.autograd.forward_ad as fw
    x, t = make(4, 60, torch.float32)
    one = torch.ones_like(x)
    with fw.dual_level():
        dual = fw.make_dual(x, one)
        for logits in (dual, dual[:, 1:], dual.unflatten(0, (2, 2)), dual.T.contiguous().T, dual.half(),
                       fw.make_dual(x.clone().requires_grad_(), one)):
            with pytest.raises(NotImplementedError):
                op()(logits, t.view(logits.shape[:-1]) % 50, top=2)
            with pytest.raises(NotImplementedError), torch.no_grad():
                op()(logits, t.view(logits.shape[:-1]) % 50, top=2)
        leaf = x.clone().requires_grad_()
        out = op()(leaf, t)
        with pytest.raises(NotImplementedError):
            torch.autograd.grad(out.lse, leaf, fw.make_dual(torch.ones(4, device="cuda"), torch.ones(4, device="cuda")))
        primal = fw.unpack_dual(dual).primal
        assert torch.equal(op()(primal, t).logprob, op()(x, t).logprob)
    assert torch.equal(op()(x, t).logprob, op()(x.clone().requires_grad_(), t).logprob)


@pytest.mark.gpu
def test_a_number_of_alternatives_is_an_integer():
    x, t = make(4, 50, torch.float32)
    for bad in (2.5, 2.0, "2", None, [2]):
        with pytest.raises(ValueError):
            op()(x, t, top=bad)
    assert op()(x, t, top=np.int64(2)).top_ids.shape == (4, 2) and op()(x[None], t[None], top=np.uint8(3)).top_ids.shape == (1, 4, 3)
