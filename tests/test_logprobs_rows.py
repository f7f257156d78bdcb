"""token_logprobs at numbers of rows that fill the SMs, where a warp takes four short rows, or one or few warps a long row:
values and alternatives against the definition in 64 bits, on the device. Rows of every kind stand side by side (masks, ties,
sorted, empty, NaN), so that the rows of one warp differ. The tolerances are those of test_logprobs.py; one warp a row adds
at most 17 + V / 512 terms one after another, less than the 64 + V / 256 that they allow for."""
import math

import pytest
import torch

from test_logprobs import INF, op, rel

pytestmark = pytest.mark.gpu

KINDS = 9   # odd: four rows side by side are of other kinds in the next warp


def sms():
    return torch.cuda.get_device_properties(0).multi_processor_count


def mixed(rows, vocab, dtype, seed):
    """Rows by turns: plain, half of -inf, half of the type's lowest value, one open token, empty, all equal, many ties,
    ascending, NaN among them. Every eleventh token is padding."""
    g = torch.Generator("cuda").manual_seed(seed)
    rand = lambda *s: torch.rand(*s, device="cuda", generator=g)  # noqa: E731
    x = torch.randn(rows, vocab, device="cuda", generator=g) * (rand(rows, 1) * 5 + 0.5) + 3
    t = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
    kind = (torch.arange(rows, device="cuda") % KINDS)[:, None]
    half = rand(rows, vocab) < 0.5
    at = torch.arange(vocab, device="cuda")[None]
    x = torch.where((kind == 1) & half, -INF, x)
    x = torch.where(((kind == 3) & (at != t[:, None])) | (kind == 4), -INF, x)
    x = torch.where(kind == 5, 1.5, x)
    x = torch.where(kind == 6, (x * 2).round() / 2, x)
    x = torch.where(kind == 7, x.sort(1)[0], x).to(dtype)
    x = torch.where((kind == 2) & half, torch.finfo(dtype).min, x)
    x = torch.where((kind == 8) & (rand(rows, vocab) < 0.1), math.nan, x)
    t[5::11] = -1
    return x, t if seed % 2 else t.int()


def near(got, want, tol, what):
    got = got.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), what
    off = torch.where(torch.isfinite(want), (got - want).abs() / tol, 0.0)
    assert float(off.max()) <= 1, f"{what}: off by {float(off.max())} of the tolerance"


def check(x, t, tops):
    rows, vocab = x.shape
    xd, t64 = x.double(), t.long()
    m = xd.amax(-1, keepdim=True)
    y = xd - torch.where(m == -INF, 0.0, m)   # first: beside the type's lowest value log s is lost, in 64 bits too
    ls = y.exp().sum(-1, keepdim=True).log()
    lse, logp = (m + ls)[:, 0], torch.where(ls == -INF, -INF, y - ls)
    p = torch.where(logp == -INF, 0.0, logp.exp())
    h = -torch.where(p == 0, 0.0, p * logp).sum(-1)
    lp = torch.where(t64 < 0, 0.0, logp.gather(1, t64.clamp(min=0)[:, None])[:, 0])
    most = torch.where(xd.abs() < 1e4, xd.abs(), 0.0).amax(-1)
    order = torch.where(torch.isnan(xd), -INF, xd).sort(stable=True, dim=-1, descending=True)[1]
    fin = lambda v: torch.where(torch.isfinite(v), v.abs(), 0.0)  # noqa: E731
    r = rel(vocab)
    for top in sorted({min(top, vocab) for top in tops}):
        out = op()(x, t, top=top)
        near(out.logprob, lp, r + 2.0 ** -22 * (fin(lp) + most), "logprob")
        near(out.lse, lse, r + 2.0 ** -22 * (fin(lse) + most), "lse")
        near(out.entropy, h, torch.full_like(h, r * (1 + 3 * math.log2(max(2, vocab)))), "entropy")
        if top:
            ids = order[:, :top]
            assert torch.equal(out.top_ids.long(), ids)
            want = logp.gather(1, ids)
            # an alternative that is NaN ranks as -inf; the values of its row are NaN
            near(out.top_logprobs, want, r + 2.0 ** -22 * (fin(want) + most[:, None]), "top_logprobs")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("vocab", [9, 20, 128, 256, 257, 512, 1000, 1024])
def test_short_rows_four_a_warp(vocab, dtype):
    x, t = mixed(64 * sms() + 1 + vocab % 4, vocab, dtype, seed=vocab)
    check(x, t, (0, 5, 8, 20, 64))


def test_short_rows_that_all_tie():
    """Ranks by the values alone come twice in every row, and are written over by those that count the indices."""
    for vocab in (40, 200, 700):
        x, t = mixed(64 * sms() + 3, vocab, torch.float32, seed=vocab)
        x = (x.nan_to_num(0, 0, 0) / 2).round()
        check(x, t, (3, 20, 64))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("per_sm,vocab", [(2.5, 4099), (5, 4099), (10, 4099), (20, 1100), (20, 2600), (20, 9001), (50, 1100),
                                          (50, 2600)])
def test_long_rows_few_warps_a_row(per_sm, vocab, dtype):
    """Eight, four and two warps a row, and one from 20 rows an SM on: it joins the sums and picks the segments itself, and
    its 32 threads have up to 64 alternatives to find."""
    x, t = mixed(int(per_sm * sms()) + 3, vocab, dtype, seed=vocab)
    check(x, t, (0, 1, 5, 20, 33, 64))


@pytest.mark.parametrize("dtype,vocab", [(torch.float32, 8003), (torch.bfloat16, 16001), (torch.float16, 16384)])
def test_long_rows_two_warps_where_one_would_leave_a_round_half_empty(dtype, vocab):
    x, t = mixed(34 * sms(), vocab, dtype, seed=7)
    check(x, t, (0, 20, 64))


def test_long_rows_that_all_tie():
    for vocab in (1100, 5000):
        x, t = mixed(21 * sms(), vocab, torch.float32, seed=vocab)
        x = (x.nan_to_num(0, 0, 0) / 2).round()
        check(x, t, (3, 33, 64))


def test_many_rows_of_unlike_alignment():
    """Rows that begin anywhere: short ones four a warp, and long ones."""
    for rows, vocab in ((64 * sms() + 2, 200), (64 * sms() + 2, 900), (21 * sms(), 3001)):
        wide, t = mixed(rows, vocab + 5, torch.bfloat16, seed=vocab)
        t = t.clamp(max=vocab - 1)
        for x in (wide[:, 1:vocab + 1], wide[:, 5:]):
            check(x, t, (0, 7, 40))


def gradient(x, t, top, g, gh, gs, gt):
    """The formula in 64 bits, and the magnitude of its terms at each entry."""
    xd, t64 = x.double(), t.long()
    m = xd.amax(-1, keepdim=True)
    y = xd - torch.where(m == -INF, 0.0, m)
    ls = y.exp().sum(-1, keepdim=True).log()
    logp = torch.where(ls == -INF, -INF, y - ls)
    p = torch.where(logp == -INF, 0.0, logp.exp())
    plogp = torch.where(p == 0, 0.0, p * logp)
    h = -plogp.sum(-1, keepdim=True)
    w = torch.zeros_like(xd)
    g = torch.where(t64 < 0, 0.0, g.double())
    w.scatter_add_(1, t64.clamp(min=0)[:, None], g[:, None])
    ids = xd.sort(stable=True, dim=-1, descending=True)[1][:, :top]
    w.scatter_add_(1, ids, gt.double())
    want = w + p * (gs.double() - g - gt.double().sum(-1))[:, None] - gh.double()[:, None] * (plogp + p * h)
    want = torch.where(ls == -INF, 0.0, want)
    size = (g.abs() + gs.abs() + gt.abs().sum(-1))[:, None]
    r = rel(x.shape[1])
    open_logp = torch.where(p == 0, 0.0, logp.abs())
    most = torch.where(xd.abs() < 1e4, xd.abs(), 0.0).amax(-1, keepdim=True)
    err = r * (1 + 3 * math.log2(max(2, x.shape[1]))) + 2.0 ** -22 * (open_logp + most)
    tol = p * err * (size + gh.abs()[:, None] * (open_logp + h + 1)) + 2.0 ** -22 * w.abs()
    step = {torch.float32: 2.0 ** -23, torch.float16: 2.0 ** -10, torch.bfloat16: 2.0 ** -7}[x.dtype]
    return want, tol + want.abs() * step + (2.0 ** -25 if x.dtype == torch.float16 else 1e-37)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("vocab", [9, 40, 128, 200, 256, 500, 1024, 2001])
def test_gradients_of_many_rows(vocab, dtype):
    x, t = mixed(64 * sms() + 3, vocab, dtype, seed=vocab)
    x = x[torch.arange(len(x), device="cuda") % KINDS != 8].contiguous()   # without the rows of NaN
    rows, top = len(x), 5
    t = t[:rows].contiguous()
    g = torch.Generator("cuda").manual_seed(3)
    arriving = [torch.randn(rows, device="cuda", generator=g) for _ in range(3)]
    arriving.append(torch.randn(rows, top, device="cuda", generator=g))
    leaf = x.clone().requires_grad_()
    out = op()(leaf, t, top=top)
    got, = torch.autograd.grad([out.logprob, out.entropy, out.lse, out.top_logprobs], leaf, arriving)
    want, tol = gradient(x, t, top, *arriving)
    near(got, want, tol, "gradient")
