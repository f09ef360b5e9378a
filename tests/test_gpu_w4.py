"""linear_w4 and dequantize_w4 against float64, at the ends of their ranges and where a tile, a block or a group is
partial."""
import math

import pytest
import torch

from mamba_lite import _lib, ops

pytestmark = pytest.mark.gpu


def _matrix(n, k, group, zeros, scale_dtype, seed):
    """(W4, the same matrix in float64 by its definition)"""
    g = torch.Generator(device="cuda").manual_seed(seed)
    ng = -(-k // group)
    codes = torch.randint(0, 16, (n, k), device="cuda", generator=g, dtype=torch.uint8)
    scales = ((torch.rand(n, ng, device="cuda", generator=g) + 0.5) * 0.01).to(scale_dtype)
    z = torch.randint(0, 16, (n, ng), device="cuda", generator=g, dtype=torch.uint8) if zeros else None
    col = torch.arange(k, device="cuda") // group
    w = (codes.double() - (8.0 if z is None else z.double()[:, col])) * scales.double()[:, col]
    return ops.pack_w4(codes, scales, z, group), w


def _x(m, k, dtype, seed):
    return torch.randn(m, k, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).to(dtype)


def _tol(k, group, dtype):
    """Of the norm.  float32: a random walk of k rounded sums, 2^-24 sqrt(k); sums over a group may run over codes
    16 + q, six times the size of q - z, before 16 + z of the sum of x is taken off; splits, scales and the bias a few
    roundings more.  bfloat16: the output's rounding, 2^-8."""
    return 2.0 ** -24 * (math.sqrt(k) + 6 * math.sqrt(min(k, group)) + 4) + (2.0 ** -8 if dtype == torch.bfloat16 else 0)


def _check(y, ref, tol):
    assert y.shape == ref.shape
    e = float((y.double() - ref).norm() / ref.norm().clamp_min(1e-300))
    assert e < tol, (e, tol)
    # no value is far off either: 6 times the root mean square of what the norm allows, plus its own rounding
    worst = float(((y.double() - ref).abs() - tol * ref.abs()).max() / ref.norm() * math.sqrt(ref.numel()))
    assert worst < 6 * tol, (worst, tol)


SIZES = [(1, 1, 1), (1, 16, 128), (2, 15, 31), (3, 17, 129), (5, 768, 1536), (6, 33, 700), (16, 1001, 777),
         (17, 100, 2048), (33, 48, 96), (64, 257, 1300), (1, 8192, 2048), (4, 40, 9000), (48, 20, 8192)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("group,zeros,scale_dtype", [(32, True, torch.float32), (64, False, torch.bfloat16),
                                                     (128, True, torch.bfloat16), (128, False, torch.float32)])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_linear_matches_float64(m, n, k, group, zeros, scale_dtype, dtype):
    w4, w = _matrix(n, k, group, zeros, scale_dtype, n + k)
    x = _x(m, k, dtype, m)
    bias = _x(1, n, dtype, 7)[0] if m % 2 else None
    ref = x.double() @ w.t().contiguous() + (0 if bias is None else bias.double())
    y = ops.linear_w4(x, w4, bias)
    assert y.dtype == dtype
    _check(y, ref, _tol(k, group, dtype))
    assert torch.equal(y, ops.linear_w4(x, w4, bias))          # the same bits every time


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("group,zeros,scale_dtype", [(32, False, torch.bfloat16), (64, True, torch.float32),
                                                     (128, True, torch.bfloat16)])
@pytest.mark.parametrize("n,k", [(1, 1), (16, 128), (15, 31), (17, 129), (768, 1536), (1001, 777), (100, 130), (5, 5000)])
def test_matrix_is_the_rounded_product(n, k, group, zeros, scale_dtype, dtype):
    w4, w = _matrix(n, k, group, zeros, scale_dtype, n + k)
    got = ops.dequantize_w4(w4, dtype)
    assert got.shape == (n, k) and torch.equal(got, w.float().to(dtype))       # one rounding (a code times a scale
    # fits 24 bits + 5: float32 rounds it once, and so does the float64 value taken to float32)


def test_rows_with_strides_and_outputs_in_place():
    w4, w = _matrix(100, 300, 64, True, torch.bfloat16, 0)
    for dtype in (torch.float32, torch.bfloat16):
        big = _x(9, 700, dtype, 1)
        for x in (big[:, 3:303], big[::2, 5:305], big[:1, 1:301], big[:, ::2][:, :300], big[4:5].expand(3, 700)[:, :300],
                  big[:, :600].reshape(9, 2, 300)):
            ref = x.double() @ w.t().contiguous()
            _check(ops.linear_w4(x, w4), ref, _tol(300, 64, dtype))
        room = torch.full((6, 130), 3.0, device="cuda", dtype=dtype)
        got = ops.linear_w4(big[:4, :300], w4, out=room[1:5, 7:107])
        _check(got, big[:4, :300].double() @ w.t().contiguous(), _tol(300, 64, dtype))
        room[1:5, 7:107] = 3.0
        assert bool((room == 3.0).all())                       # nothing written beside the rows
        wide = torch.full((102, 311), 5.0, device="cuda", dtype=dtype)
        ops.dequantize_w4(w4, dtype, out=wide[1:101, 3:303])
        assert torch.equal(wide[1:101, 3:303], w.float().to(dtype))
        wide[1:101, 3:303] = 5.0
        assert bool((wide == 5.0).all())
    assert ops.linear_w4(torch.empty(0, 300, device="cuda"), w4).shape == (0, 100)
    assert ops.linear_w4(_x(1, 300, torch.float32, 2)[0], w4).shape == (100,)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("scale", [1e-30, 1e20, 3e35])
def test_large_and_small_values(dtype, scale):
    w4, w = _matrix(64, 512, 64, True, torch.float32, 3)
    x = (_x(3, 512, torch.float32, 4).clamp(-4, 4) * scale).to(dtype)
    ref = x.double() @ w.t().contiguous()
    assert bool(ref.abs().max() < 3e38)
    _check(ops.linear_w4(x, w4) / scale, ref / scale, _tol(512, 64, dtype) + 2.0 ** -24)
    # rows of very different size do not disturb each other
    x = _x(3, 512, torch.float32, 5) * torch.tensor([1e-12, 1.0, 1e12], device="cuda")[:, None]
    y, ref = ops.linear_w4(x.to(dtype), w4), x.to(dtype).double() @ w.t().contiguous()
    for m in range(3):
        _check(y[m:m + 1], ref[m:m + 1], _tol(512, 64, dtype))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,at", [(1, 0), (7, 3), (40, 39)])
def test_infinities_and_nan_stay_in_their_row(m, at, dtype):
    w4, w = _matrix(70, 400, 32, True, torch.bfloat16, 6)
    x = _x(m, 400, dtype, 8)
    clean = x.double() @ w.t().contiguous()
    for bad, where in ((float("inf"), 5), (float("-inf"), 399), (float("nan"), 130)):
        xb = x.clone()
        xb[at, where] = bad
        y = ops.linear_w4(xb, w4)
        ref = xb.double()[at] @ w.t().contiguous()             # inf * 0 is NaN, inf * w an infinity of its sign
        assert torch.equal(torch.isnan(y[at]), torch.isnan(ref))
        ok = ~torch.isnan(ref)
        assert torch.equal(y[at][ok].double(), ref[ok])
        rest = [i for i in range(m) if i != at]
        if rest:
            _check(y[rest], clean[rest], _tol(400, 32, dtype))


def test_streams_and_graph_replays():
    w4, w = _matrix(300, 1000, 128, False, torch.bfloat16, 9)
    x = _x(5, 1000, torch.float32, 10)
    want = ops.linear_w4(x, w4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.linear_w4(x, w4)
        ops.linear_w4(x, w4), ops.dequantize_w4(w4)            # warm for the capture
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    sx = x.clone()
    with torch.cuda.graph(graph):
        y = ops.linear_w4(sx, w4)
        wm = ops.dequantize_w4(w4)
    for i in range(4):
        sx.copy_(x * (i + 1))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ops.linear_w4(x * (i + 1), w4)) and torch.equal(wm, w.float())


def test_refusals_on_the_gpu():
    w4, _ = _matrix(20, 200, 64, True, torch.bfloat16, 11)
    x = _x(2, 200, torch.float32, 12)
    with pytest.raises(ValueError, match="at most 64"):
        ops.linear_w4(_x(65, 200, torch.float32, 0), w4)
    with pytest.raises(RuntimeError, match="operands"):
        ops.linear_w4(x.cpu(), w4)
    with pytest.raises(RuntimeError, match="operands"):
        ops.linear_w4(x, w4, out=torch.empty(2, 20))
    with pytest.raises(RuntimeError, match="backward"):
        ops.linear_w4(x.requires_grad_(), w4)
    with torch.no_grad():
        ops.linear_w4(x, w4)
    odd = torch.zeros(2000, device="cuda", dtype=torch.bfloat16)[1:1 + w4.scales.numel()].view_as(w4.scales)
    half = ops.W4(w4.codes, odd, w4.zeros, 20, 200, 64)
    with pytest.raises(AttributeError):
        half.scales = w4.scales
    with pytest.raises(_lib.MTLError, match="aligned"):
        ops.linear_w4(_x(2, 200, torch.float32, 12), half)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("k", [1, 5, 7, 8, 9, 15, 127, 128, 129, 136, 777, 1300, 9001])
def test_linear_on_rows_at_any_alignment(k, dtype):
    w4, w = _matrix(40, k, 32, True, torch.float32, k)
    for m, offset, gap in ((1, 1, 0), (5, 2, 3), (33, 7, 1), (64, 0, 5)):
        # what lies around the rows is NaN
        buffer = torch.full((offset + m * (k + gap),), torch.nan, device="cuda", dtype=dtype)
        x = buffer[offset:].view(m, k + gap)[:, :k]
        x.copy_(_x(m, k, dtype, k + m))
        _check(ops.linear_w4(x, w4), x.double() @ w.t().contiguous(), _tol(k, 32, dtype))
        # an infinity in the row's last column sends that row alone to infinities
        x[m - 1, k - 1] = torch.inf
        y = ops.linear_w4(x, w4)
        ref = x.double()[m - 1] @ w.t().contiguous()
        assert torch.equal(torch.isnan(y[m - 1]), torch.isnan(ref)) and torch.equal(y[m - 1] == torch.inf, ref == torch.inf)
        if m > 1:
            _check(y[:m - 1], x[:m - 1].double() @ w.t().contiguous(), _tol(k, 32, dtype))


def _each(y, x, w, bias=None):
    """Every value against float64, within what k fp32 products and sums may be off in any order: each of the k + 8
    operations rounds by 2^-24 of what it makes, or cuts off 2^-23, and what is made never passes sum |x| |w|; then the
    output's own rounding."""
    k = x.shape[-1]
    ref = x.double() @ w.t().contiguous()
    most = x.double().abs() @ w.abs().t().contiguous()
    if bias is not None:
        ref, most = ref + bias.double(), most + bias.double().abs()
    tol = (k + 8) * 2.0 ** -23 * most + (2.0 ** -8 * ref.abs() if y.dtype == torch.bfloat16 else 0) + 1e-37
    off = (y.double() - ref).abs()
    assert bool((off <= tol).all()), float((off / tol).max())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True), (128, False)])
@pytest.mark.parametrize("m,n,k", [(1, 40, 256), (6, 100, 777), (17, 33, 1024), (40, 50, 4000)])
def test_a_large_value_meets_a_weight_of_zero(m, n, k, group, zeros, dtype):
    """Columns whose code is their zero weigh nothing, whatever x holds there."""
    g = torch.Generator(device="cuda").manual_seed(n + k)
    ng = -(-k // group)
    codes = torch.randint(0, 16, (n, k), device="cuda", generator=g, dtype=torch.uint8)
    z = torch.randint(0, 16, (n, ng), device="cuda", generator=g, dtype=torch.uint8)
    z = z if zeros else torch.full_like(z, 8)
    col = torch.arange(k, device="cuda") // group
    large = torch.arange(0, k, 29, device="cuda")
    codes[:, large] = z[:, col[large]]
    scales = (torch.rand(n, ng, device="cuda", generator=g) + 0.5) * 0.01
    w4 = ops.pack_w4(codes, scales, z if zeros else None, group)
    w = (codes.double() - z.double()[:, col]) * scales.double()[:, col]
    for size in (1e3, 1e10, 1e20, 7e28):
        x = _x(m, k, dtype, m)
        x[:, large] = (x[:, large].sign() * size).to(dtype)
        _each(ops.linear_w4(x, w4), x, w)
        one = _x(m, k, dtype, m)                              # in a single row: no other row notices
        one[m // 2, large[1]] = size
        _each(ops.linear_w4(one, w4), one, w)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset", [0.0, 10.0, 1e4])
def test_rows_about_an_offset(offset, dtype):
    """x whose values share an offset: sums of x over a group are large, sums of x w are as large as x and w make them."""
    w4, w = _matrix(100, 2048, 128, True, torch.bfloat16, 21)
    x = (_x(5, 2048, torch.float32, 22) + offset).to(dtype)
    _each(ops.linear_w4(x, w4), x, w)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("m,n,k", [(2, 20, 5), (7, 70, 400), (16, 300, 1300), (40, 33, 777), (10, 40, 9001), (64, 17000, 300)])
def test_a_row_that_holds_an_infinity_changes_no_bit_of_another(m, n, k, zeros, dtype):
    w4, _ = _matrix(n, k, 64, zeros, torch.bfloat16, 31)
    x = _x(m, k, dtype, 32)
    clean = ops.linear_w4(x, w4)
    for bad in (float("inf"), float("nan"), 3e38):
        for rows in ([0], [m - 1], list(range(0, m, 2))):
            xb = x.clone()
            for i, row in enumerate(rows):
                xb[row, (i * 37 + k - 1) % k] = bad
            y = ops.linear_w4(xb, w4)
            rest = [i for i in range(m) if i not in rows]
            assert torch.equal(y[rest], clean[rest])
            assert bool((~torch.isfinite(y[rows]) | (y[rows] != clean[rows])).any(1).all())


# What few and short rows of W do not reach: two operand tiles, workgroups of 16 wavefronts, several tiles of W to a
# wavefront (the next one's loads under the last products), x in parts for each of them, a last tile that is partial.
LARGE = [(1, 50280, 2048), (16, 50280, 2048), (33, 50277, 777), (64, 33000, 520), (10, 20011, 9000), (64, 8192, 2048),
         (48, 2043, 4096), (33, 8190, 8192), (40, 50277, 6000)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("group,zeros,scale_dtype", [(32, True, torch.bfloat16), (64, False, torch.float32)])
@pytest.mark.parametrize("m,n,k", LARGE)
def test_large_matrices_match_float64(m, n, k, group, zeros, scale_dtype, dtype):
    w4, w = _matrix(n, k, group, zeros, scale_dtype, n + k)
    x = _x(m, k, dtype, m)
    bias = _x(1, n, dtype, 7)[0] if zeros else None
    y = ops.linear_w4(x, w4, bias)
    _check(y, x.double() @ w.t().contiguous() + (0 if bias is None else bias.double()), _tol(k, group, dtype))
    _each(y, x, w, bias)
    assert torch.equal(y, ops.linear_w4(x, w4, bias))
    xb = x.clone()
    at, where = m // 2, k - 3
    xb[at, where] = torch.inf
    yb = ops.linear_w4(xb, w4, bias)
    ref = torch.inf * w[:, where]                          # NaN where the weight is zero
    assert torch.equal(torch.isnan(yb[at]), torch.isnan(ref))
    assert torch.equal(yb[at][~torch.isnan(ref)].double(), ref[~torch.isnan(ref)])
    rest = [i for i in range(m) if i != at]
    assert torch.equal(yb[rest], y[rest])


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("scale", [1e-33, 1e-36, 1e-39])
def test_values_near_the_least_ones(scale, zeros):
    """fp32 x to 2^-133, where bf16's least values end: each of k values by less than that, on top of the sums' rounding."""
    k = 512
    w4, w = _matrix(64, k, 64, zeros, torch.float32, 3)
    x = _x(3, k, torch.float32, 4) * scale
    ref = x.double() @ w.t().contiguous()
    most = x.double().abs() @ w.abs().t().contiguous()
    tol = (k + 8) * 2.0 ** -23 * most + 2.0 ** -133 * w.abs().sum(1) + k * 2.0 ** -149
    assert bool(((ops.linear_w4(x, w4).double() - ref).abs() <= tol).all())
