"""int8_linear and quantize_rows against their definition, at the sizes where the kernels change shape or can go wrong,
and their refusals.

Tolerances. The codes and the scales of the rows are compared exactly: the definition's two divisions and one product
round once each in float32, here as there. The integer sums are exact; a product then rounds to float32 once for the
sum, once for each factor and once with the bias, so that it is off by at most 4 2^-24 of the magnitudes of its two
terms, and by half a spacing of its own type.
"""
import numpy as np
import pytest
import torch

from yggdrasil_b200 import _native

STEP = {torch.float32: 2.0 ** -23, torch.float16: 2.0 ** -10, torch.bfloat16: 2.0 ** -7}
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def ops():
    import yggdrasil_b200 as y
    return y.int8_linear, y.quantize_rows


def codes_of(x):
    """The definition in float32 on the host: codes (rows, k) int64, scale (rows,) float32."""
    x = x.detach().float().cpu().numpy()
    with np.errstate(all="ignore"):
        most = np.abs(x).max(-1)
        scale, inverse = most / np.float32(127), np.float32(127) / most
        dead = (scale == 0) | np.isinf(inverse)
        bad = ~np.isfinite(most)
        inverse = np.where(dead | bad, np.float32(0), inverse).astype(np.float32)
        prod = np.where(inverse[:, None] == 0, np.float32(0), x * inverse[:, None])
    codes = np.clip(np.rint(prod), -127, 127).astype(np.int64)
    return codes, np.where(bad, np.float32(np.nan), np.where(dead, np.float32(0), scale)).astype(np.float32)


def weights(n, k, seed=0, bias=True):
    g = torch.Generator().manual_seed(seed)
    w = torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8)
    laid = torch.full((n, (k + 15) // 16 * 16), 77, dtype=torch.int8)   # the bytes past k are nobody's
    laid[:, :k] = w
    scale = torch.rand(n, generator=g) * 0.01 + 0.001
    b = torch.randn(n, generator=g) if bias else None
    return laid.cuda()[:, :k], scale.cuda(), None if b is None else b.cuda()


def inputs(rows, k, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + 100)
    x = torch.randn(rows, k, generator=g) * (torch.rand(rows, 1, generator=g) * 10 + 0.01)
    return x.to(dtype).cuda()


def check(y, x, w, s, b, dtype):
    codes, sx = codes_of(x)
    acc = codes.astype(np.float64) @ w.cpu().numpy().astype(np.float64).T
    prod = acc * sx.astype(np.float64)[:, None] * s.cpu().numpy().astype(np.float64)[None]
    bias = np.zeros(w.shape[0]) if b is None else b.float().cpu().numpy().astype(np.float64)
    want = prod + bias
    tol = 4 * 2.0 ** -24 * (np.abs(prod) + np.abs(bias)) + STEP[dtype] / 2 * np.abs(want) + 2.0 ** -25
    got = y.double().cpu().numpy()
    assert y.dtype == dtype and got.shape == want.shape
    # a value beyond the type's range is infinite (float32's edge is its largest number and half a spacing)
    edge = {torch.float32: 2.0 ** 128 - 2.0 ** 103, torch.float16: 65520.0, torch.bfloat16: 2.0 ** 128 - 2.0 ** 119}[dtype]
    beyond = np.abs(want) >= edge
    assert np.array_equal(got[beyond], np.copysign(np.inf, want[beyond]))
    off = np.where(beyond, 0, np.abs(got - np.where(beyond, 0, want)) / tol)
    assert np.nanmax(off) <= 1 and np.array_equal(np.isnan(got), np.isnan(want)), f"off by {np.nanmax(off)}"


SIZES = [(1, 1, 1), (1, 16, 1), (1, 17, 5), (1, 1280, 256), (1, 4096, 1000), (2, 100, 33), (3, 4097, 257),
         (4, 512, 256), (5, 1000, 515), (7, 33, 129), (8, 2048, 2047), (9, 96, 128), (15, 8191, 130), (16, 512, 4099),
         (17, 64, 300), (31, 640, 1000), (32, 128, 127), (33, 129, 128), (64, 1000, 257), (77, 1000, 5003),
         (127, 512, 640), (128, 128, 128), (129, 257, 129), (200, 4096, 16), (255, 96, 2000), (256, 384, 256),
         (257, 1024, 513), (300, 5000, 1030), (513, 272, 5), (1000, 64, 256), (1025, 1500, 1100), (4099, 512, 256),
         (65537, 64, 5)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k,n", SIZES)
def test_values(rows, k, n, dtype):
    f, _ = ops()
    x = inputs(rows, k, dtype, seed=k)
    w, s, b = weights(n, k, seed=n, bias=n % 2 == 1)
    check(f(x, w, s, b), x, w, s, b, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,k,n", [(1, 131072, 40), (3, 131072, 5), (130, 65552, 130), (20, 100003, 300)])
def test_long_rows_with_the_largest_codes(rows, k, n):
    """Every code 127: the sums reach 127 127 k, near the end of int32 at the longest rows."""
    f, _ = ops()
    x = torch.full((rows, k), 3.0, device="cuda")
    w, s, b = weights(n, k)
    w.fill_(127)
    w[1::2] = -127
    check(f(x, w, s, b), x, w, s, b, torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k", [(1, 1), (3, 15), (5, 16), (2, 17), (9, 1000), (300, 255), (4, 4096), (2, 20001),
                                    (1, 131072)])
def test_codes_and_scales(rows, k, dtype):
    _, q = ops()
    x = inputs(rows, k, dtype, seed=3)
    if rows > 2:
        x[1] = 0
    got = q(x)
    codes, scale = codes_of(x)
    assert got.codes.shape == x.shape and got.codes.stride(0) % 16 == 0
    assert np.array_equal(got.codes.cpu().numpy(), codes)
    assert np.array_equal(got.scale.cpu().numpy(), scale)
    pad = got.codes.as_strided((rows, got.codes.stride(0)), (got.codes.stride(0), 1))[:, k:]
    assert not bool(pad.any())


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [6, 40])
def test_zero_tiny_nan_and_infinite_rows(rows):
    f, q = ops()
    x = inputs(rows, 300, torch.float32)
    x[0] = 0
    x[1] = 1e-44          # its scale rounds to nothing
    x[2, 7] = float("nan")
    x[3, 299] = float("inf")
    x[4, 0] = -float("inf")
    x[5] = 3e38
    w, s, b = weights(130, 300)
    got = q(x)
    codes, scale = codes_of(x)
    assert np.array_equal(got.codes.cpu().numpy(), codes)
    assert np.array_equal(got.scale.cpu().numpy(), scale, equal_nan=True)
    y = f(x, w, s, b)
    check(y, x, w, s, b, torch.float32)
    assert torch.equal(y[0], b) and torch.equal(y[1], b)
    assert torch.isnan(y[2:5]).all() and not torch.isnan(y[5:]).any()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 12, 150])
def test_strides_types_and_leading_shapes(rows):
    f, q = ops()
    wide = inputs(rows, 520, torch.bfloat16)
    w, s, b = weights(200, 515)
    for x in (wide[:, :515], wide[:, 1:516], wide[:, 5:], wide[:, :515].T.contiguous().T):
        check(f(x, w, s, b), x, w, s, b, torch.bfloat16)
        check(f(x, w, s, b, out_dtype=torch.float32), x, w, s, b, torch.float32)
        check(f(q(x), w, s, b), x, w, s, b, torch.float32)
        check(f(q(x), w, s, b, out_dtype=torch.float16), x, w, s, b, torch.float16)
    x = wide[:, :515]
    dense = w.contiguous()                      # rows 515 bytes apart: laid out at the call
    assert torch.equal(f(x, dense, s, b), f(x, w, s, b))
    spread = torch.zeros(200, 1040, dtype=torch.int8, device="cuda")[:, 16:531]
    spread.copy_(w)
    assert torch.equal(f(x, spread, s, b), f(x, w, s, b))
    c = q(x)
    tight = type(c)(c.codes.contiguous(), c.scale)
    assert torch.equal(f(tight, w, s, b), f(c, w, s, b))
    assert torch.equal(f(x, w, s, b.bfloat16()), f(x, w, s, b.bfloat16().float()))
    one = f(x[0], w, s, b)
    assert one.shape == (200,) and torch.equal(one, f(x, w, s, b)[0])
    if rows == 12:
        assert torch.equal(f(x.unflatten(0, (2, 3, 2)), w, s, b).flatten(0, 2), f(x, w, s, b))
        assert q(x.unflatten(0, (3, 4))).scale.shape == (3, 4)


@pytest.mark.gpu
def test_codes_whose_padding_is_not_zero():
    """Bytes past k count for nothing, whatever they hold."""
    f, q = ops()
    for rows in (1, 3, 70, 300):
        x = inputs(rows, 77, torch.float32)
        w, s, b = weights(150, 77)
        c = q(x)
        laid = torch.full((rows, 96), 101, dtype=torch.int8, device="cuda")
        laid[:, :77] = c.codes
        assert torch.equal(f(type(c)(laid[:, :77], c.scale), w, s, b), f(c, w, s, b))


@pytest.mark.gpu
def test_no_rows():
    f, q = ops()
    w, s, b = weights(20, 64)
    assert f(torch.empty(0, 64, device="cuda"), w, s, b).shape == (0, 20)
    assert q(torch.empty(0, 64, device="cuda")).codes.shape == (0, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,k,n", [(1, 4096, 4000), (20, 8192, 300), (300, 2000, 700)])
def test_another_stream_a_graph_and_repeats(rows, k, n):
    f, _ = ops()
    x = inputs(rows, k, torch.bfloat16)
    w, s, b = weights(n, k)
    want = f(x, w, s, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = f(x, w, s, b)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = f(x, w, s, b)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)


@pytest.mark.gpu
def test_outputs_stay_in_their_rows():
    """Nothing is written beside the output: its neighbours keep their values."""
    f, _ = ops()
    lib = _native.ops()
    for rows, k, n in ((1, 100, 77), (5, 100, 77), (50, 100, 77), (200, 300, 259)):
        x = inputs(rows, k, torch.float32)
        w, s, b = weights(n, k)
        frame = torch.full((rows + 2, n + 9), -5.0, device="cuda")
        ws = torch.empty(lib.ygg_linear_workspace(rows, k), dtype=torch.uint8, device="cuda")
        out = frame[1:-1, 4:4 + n]
        rc = lib.ygg_linear(0, 0, rows, k, n, x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0), s.data_ptr(),
                            b.data_ptr(), 0, out.data_ptr(), out.stride(0), ws.data_ptr(), ws.numel(),
                            torch.cuda.current_stream().cuda_stream)
        assert rc == _native.YGG_OK
        assert torch.equal(out, f(x, w, s, b))
        keep = frame.clone()
        keep[1:-1, 4:4 + n] = -5.0
        assert bool((keep == -5.0).all())


@pytest.mark.gpu
def test_refusals():
    f, q = ops()
    x = inputs(4, 64, torch.float32)
    w, s, b = weights(20, 64)
    for bad in (x.double(), x.cpu(), x[:, :63], torch.empty(4, 0, device="cuda"), "x"):
        with pytest.raises(ValueError):
            f(bad, w, s, b)
    for bad in (w.float(), w.cpu(), w[:, :48], w[None], w[:0]):
        with pytest.raises(ValueError):
            f(x, bad, s, b)
    for bad in (s[:19], s.half(), s.cpu(), None):
        with pytest.raises(ValueError):
            f(x, w, bad, b)
    for bad in (b[:19], b.double(), b.cpu()):
        with pytest.raises(ValueError):
            f(x, w, s, bad)
    with pytest.raises(ValueError):
        f(x, w, s, b, out_dtype=torch.int32)
    with pytest.raises(ValueError):
        q(torch.zeros(1, 131073, device="cuda"))
    with pytest.raises(NotImplementedError):
        f(x.clone().requires_grad_(), w, s, b)
    with torch.no_grad():
        f(x.clone().requires_grad_(), w, s, b)


def test_c_entry_refuses_bad_arguments():
    """Checked before any CUDA call."""
    lib = _native.ops()
    p, E = 4096, _native
    q = lib.ygg_quantize_rows
    assert q(0, 0, -1, 16, p, 16, p, 16, p, None) == E.YGG_E_ARG
    assert q(0, 0, 1, 0, p, 16, p, 16, p, None) == E.YGG_E_ARG
    assert q(0, 0, 1, 131073, p, 16, p, 131088, p, None) == E.YGG_E_UNSUPPORTED
    assert q(0, 0, 1, 20, p, 20, p, 16, p, None) == E.YGG_E_ARG
    assert q(0, 0, 1, 20, p, 20, p + 8, 32, p, None) == E.YGG_E_ARG
    assert q(0, 0, 1, 20, p, 20, p, 40, p, None) == E.YGG_E_ARG
    f = lib.ygg_linear_quantized
    assert f(0, 1, 16, 0, p, 16, p, p, 16, p, None, 0, p, 4, None) == E.YGG_E_ARG
    assert f(0, 1, 16, 4, p, 16, p, p + 4, 16, p, None, 0, p, 4, None) == E.YGG_E_ARG
    assert f(0, 1, 16, 4, p, 16, p, p, 20, p, None, 0, p, 4, None) == E.YGG_E_ARG
    assert f(0, 1, 32, 4, p, 16, p, p, 32, p, None, 0, p, 4, None) == E.YGG_E_ARG
    assert f(0, 1, 16, 4, None, 16, p, p, 16, p, None, 0, p, 4, None) == E.YGG_E_ARG
    assert f(0, 0, 16, 4, None, 16, p, p, 16, p, None, 0, p, 4, None) == E.YGG_OK
    g = lib.ygg_linear
    assert lib.ygg_linear_workspace(3, 17) >= 3 * 36
    assert lib.ygg_linear_workspace(-1, 17) == 0
    assert g(0, 0, 3, 17, 4, p, 17, p, 32, p, None, 0, p, 4, p, 8, None) == E.YGG_E_ARG
    assert g(0, 0, 3, 17, 4, p, 17, p, 32, p, None, 0, p, 4, None, 1 << 20, None) == E.YGG_E_ARG


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 3, 20, 300])
def test_weights_written_just_before_the_product(rows):
    """The product may begin under the launches before it, but reads weights, scales and rows only when they are written:
    weights quantised, rows computed and both used back to back."""
    f, q = ops()
    x = inputs(rows, 2048, torch.bfloat16)
    w = [torch.randn(3000, 2048, device="cuda", generator=torch.Generator("cuda").manual_seed(k)) for k in range(3)]
    want = []
    for v in w:
        c = q(v)
        torch.cuda.synchronize()
        want.append(f(x * 2, c.codes, c.scale))
        torch.cuda.synchronize()
    for _ in range(20):
        got = []
        for v in w:
            y = x * 2
            c = q(v)
            got.append(f(y, c.codes, c.scale))
            got.append(f(q(y), c.codes, c.scale, out_dtype=torch.bfloat16))
            c.codes.zero_()   # its memory is free to be used again
        assert all(torch.equal(got[2 * k], want[k]) and torch.equal(got[2 * k + 1], want[k]) for k in range(3))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 4, 16])
def test_weights_that_end_with_their_allocation(rows):
    """Weights of 128 MiB to the byte: nothing past them may be read."""
    f, _ = ops()
    x = inputs(rows, 4096, torch.bfloat16)
    w = [torch.randint(-127, 128, (32768, 4096), dtype=torch.int8, device="cuda") for _ in range(3)]
    s = torch.full((32768,), 0.01, device="cuda")
    for v in w:
        y = f(x, v, s)
        pick = torch.tensor([0, 1, 16383, 32766, 32767], device="cuda")
        check(y[:, pick], x, v[pick], s[pick], None, torch.bfloat16)


@pytest.mark.gpu
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("k,n", [(1280, 1300), (4000, 7000)])
def test_a_row_has_the_same_bits_in_any_batch(k, n, bias):
    """Few rows, shared K, one CTA a tile and (3000 rows) a pair: every cut of the product rounds alike."""
    f, q = ops()
    w, s, b = weights(n, k, seed=5)
    if not bias:
        b = None
    x = inputs(3000, k, torch.float32, seed=7)
    whole, codes = f(x, w, s, b), q(x)
    assert torch.equal(f(codes, w, s, b), whole)
    for rows in (1, 2, 3, 4, 5, 16, 33, 64, 100, 256, 300, 1000, 2047):
        assert torch.equal(f(x[:rows], w, s, b), whole[:rows]), rows
        assert torch.equal(f(x[-rows:], w, s, b), whole[-rows:]), rows
        assert torch.equal(f(type(codes)(codes.codes[:rows], codes.scale[:rows]), w, s, b), whole[:rows]), rows


@pytest.mark.gpu
def test_rows_of_magnitudes_below_the_inverse_of_the_range_count_as_zeros():
    """127 / 3.7e-37 is infinite in float32, 127 / 3.8e-37 is not."""
    f, q = ops()
    x = torch.zeros(4, 20, device="cuda")
    x[0, 3], x[1, 3], x[2, 3], x[3, 3] = 3.7e-37, 3.8e-37, -1e-38, 1e-44
    got = q(x)
    codes, scale = codes_of(x)
    assert np.array_equal(got.codes.cpu().numpy(), codes) and np.array_equal(got.scale.cpu().numpy(), scale)
    assert got.codes[:, 3].tolist() == [0, 127, 0, 0] and (got.scale > 0).tolist() == [False, True, False, False]


@pytest.mark.gpu
def test_status_is_clean_after_products_of_each_cut():
    from yggdrasil_b200.linear import linear_status
    f, q = ops()
    w, s, b = weights(7000, 4000)
    for rows in (1, 4, 5, 100, 3000):
        f(inputs(rows, 4000, torch.float32), w, s, b)
        linear_status()
        linear_status("cuda:0")


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [2, 40])
def test_derivatives_are_refused_of_every_input(rows):
    """Of the rows, their scales, the channels' scales and the bias, by gradients and by tangents; none is lost."""
    import torch.autograd.forward_ad as fw
    f, q = ops()
    x, (w, s, b) = inputs(rows, 64, torch.float32), weights(32, 64)
    c = q(x)
    want = f(x, w, s, b)

    def calls(mark):
        return [lambda: f(mark(x), w, s, b), lambda: f(mark(x)[None], w, s, b), lambda: q(mark(x)), lambda: q(mark(x).T),
                lambda: f(x, w, mark(s), b), lambda: f(x, w, s, mark(b)), lambda: f(x, w, s, mark(b.half())),
                lambda: f(x, w, mark(s.repeat_interleave(2))[::2], b), lambda: f(c, w, mark(s), b),
                lambda: f(type(c)(c.codes, mark(c.scale)), w, s, b), lambda: f(c, w, s, mark(b))]

    leaf = lambda t: t.detach().clone().requires_grad_()  # noqa: E731
    for call in calls(leaf):
        with pytest.raises(NotImplementedError):
            call()
        with torch.no_grad():
            call()
    with fw.dual_level():
        for call in calls(lambda t: fw.make_dual(t, torch.ones_like(t))):
            with pytest.raises(NotImplementedError):
                call()
    with torch.no_grad():
        assert torch.equal(f(leaf(x), w, leaf(s), leaf(b)), want)
    assert torch.equal(f(x, w, s, torch.nn.Parameter(b).detach()), want)


# CTA pairs over several rounds of tiles (the first two), one CTA over several rounds with bands of channel blocks, and narrow
# and short K on the tensor cores
LARGE = [(5001, 2001, 3003), (3000, 4000, 7000), (1025, 4096, 9000), (700, 300, 40000), (20000, 40, 700), (9001, 130, 1100),
         (20, 1, 40), (20, 5, 130), (300, 3, 70), (300, 15, 2000), (2000, 1, 5)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,k,n", LARGE)
def test_values_of_large_and_narrow_products(rows, k, n, dtype):
    f, _ = ops()
    x = inputs(rows, k, dtype, seed=k)
    w, s, b = weights(n, k, seed=n, bias=rows % 2 == 1)
    check(f(x, w, s, b), x, w, s, b, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("k", [1, 7, 128, 130, 255, 256, 500, 512, 513, 1000, 1024, 1030, 2000, 2048])
def test_codes_of_many_rows(k, dtype):
    """A warp a row, in one to eight vectors a lane, where rows fill the SMs; rows that end inside a vector of theirs."""
    _, q = ops()
    rows = 8 * torch.cuda.get_device_properties(0).multi_processor_count + 3
    for x in (inputs(rows, (k + 15) // 16 * 16, dtype, seed=k)[:, :k], inputs(rows, k, dtype, seed=k + 1)):
        x[5], x[rows - 1, k - 1], x[17, k // 2] = 0, float("inf"), float("nan")
        got = q(x)
        codes, scale = codes_of(x)
        assert np.array_equal(got.codes.cpu().numpy(), codes)
        assert np.array_equal(got.scale.cpu().numpy(), scale, equal_nan=True)
        padded = (k + 15) // 16 * 16
        assert not bool(got.codes.as_strided((rows, padded), (padded, 1))[:, k:].any())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("k", [1025, 2050, 4100, 8190, 16380, 16400])
def test_codes_of_long_rows(k, dtype):
    """A block a row, in one to eight vectors a thread, and beyond."""
    _, q = ops()
    x = inputs(9, (k + 15) // 16 * 16, dtype, seed=k)[:, :k]
    got = q(x)
    codes, scale = codes_of(x)
    assert np.array_equal(got.codes.cpu().numpy(), codes) and np.array_equal(got.scale.cpu().numpy(), scale)
