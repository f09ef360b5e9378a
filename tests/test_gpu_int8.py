"""quantize_int8, add_rmsnorm_int8, linear_int8 and dequantize_int8 against float64, at the ends of their ranges and where
a tile, a run or a row is partial."""
import ctypes

import pytest
import torch

from mamba_lite import _lib, ops

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16]
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}          # half a step, relative to the value


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _codes(t):
    """(codes, largest magnitudes) of float32 rows, by the definition in 64 bits."""
    a = t.double().abs().amax(-1, keepdim=True)
    return torch.where(a > 0, (t.double() * 127 / a).round(), 0.0), a


def _matrix(n, k, seed, dtype=torch.float32):
    """(Int8, the same matrix in float64 without its scales, scales in float64)"""
    g = _gen(seed)
    codes = torch.randint(-127, 128, (n, k), device="cuda", generator=g, dtype=torch.int8)
    scales = (torch.rand(n, device="cuda", generator=g) + 0.5) * 0.01
    return ops.pack_int8(codes, scales, dtype), codes.double(), scales.double()


# ------------------------------------------------------------------ rows into codes
ROWS = [(1, 1), (1, 768), (3, 5), (2, 127), (4, 128), (5, 129), (7, 777), (33, 1536), (1, 2048), (9, 2049), (8, 4096),
        (5, 4100), (300, 1000), (3, 8192), (2, 16391), (1, 40000), (1, 131071), (0, 64), (70000, 3),
        (1025, 129), (1026, 1000), (1500, 1801), (1030, 2500), (1025, 4096), (6, 5121), (3, 9001), (2, 16384)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k", ROWS)
def test_quantize_is_the_definition(m, k, dtype):
    x = torch.randn(m, k, device="cuda", generator=_gen(m + k)).to(dtype)
    if m > 2:
        x[1] = 0.0                                          # padding
        x[2, 0] = 40.0                                      # an outlier
    q = ops.quantize_int8(x)
    want, a = _codes(x.float())
    assert q.dtype == dtype and tuple(q.shape) == (m, k)
    assert torch.equal(q.codes[:, :k].double(), want)
    assert not bool(q.codes[:, k:].any())
    assert bool(((q.scales.double() - a[:, 0] / 127).abs() <= 2.0 ** -24 * a[:, 0] / 127).all())       # one division
    back = ops.dequantize_int8(q)
    assert back.dtype == dtype and torch.equal(back, (want.float() * q.scales[:, None]).to(dtype))
    assert torch.equal(ops.dequantize_int8(q, torch.float32), want.float() * q.scales[:, None])
    # half a step of the code, the scale's and the product's rounding, and the output's
    assert bool(((back.double() - x.double()).abs() <=
                 0.5 * a / 127 + (2.0 ** -23 + HALF[dtype]) * x.double().abs() + 2.0 ** -22 * a).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_halves_go_to_the_even_code(dtype):
    # a = 127: the codes are the values; a = 2 x: 63.5; and halves that no rounding of 1 / a may move
    for top in (127.0, 254.0, 1.0, 2.0 ** -90, 3 * 2.0 ** 100):
        x = torch.arange(-127, 127.5, 0.5, device="cuda") * (top / 127 if top in (127.0, 254.0) else 1.0)
        x = x.to(dtype).clamp(-top, top) if top >= 127 else torch.tensor([1.0, 0.5, -0.5, 0.25, 0.0], device="cuda").to(dtype) * top
        x[0] = top
        q = ops.quantize_int8(x[None])
        assert torch.equal(q.codes[:, :x.numel()].double(), _codes(x.float()[None])[0])
    # every float32 next to a border of a = 1: (c + 1/2) / 127 rounded down and up
    c = torch.arange(0, 127, device="cuda").double() + 0.5
    near = (c / 127).float()
    x = torch.cat([torch.ones(1, device="cuda"), near, torch.nextafter(near, torch.zeros_like(near)),
                   torch.nextafter(near, torch.ones_like(near))])[None]
    assert torch.equal(ops.quantize_int8(x).codes[:, :x.shape[1]].double(), _codes(x)[0])


@pytest.mark.parametrize("scale", [1e-45, 3e-44, 1e-41, 1.2e-38, 1e-30, 1e30, 3.4e38])
@pytest.mark.parametrize("k", [5, 777, 2048, 40000])
def test_quantize_at_the_ends_of_the_range(scale, k):
    x = torch.rand(3, k, device="cuda", generator=_gen(k)) * 2 - 1
    x[:, k // 2] = 1.0
    x = (x.double() * scale).float()
    q = ops.quantize_int8(x)
    want, a = _codes(x)
    assert torch.equal(q.codes[:, :k].double(), want)
    assert bool(((q.scales.double() - a[:, 0] / 127).abs() <= 2.0 ** -24 * a[:, 0] / 127 + 2.0 ** -150).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k", [6, 200, 4096, 50000])
def test_infinities_and_nan_stay_in_their_row(k, dtype):
    x = torch.randn(6, k, device="cuda", generator=_gen(k)).to(dtype)
    clean = ops.quantize_int8(x)
    x[1, k - 1], x[3, 0], x[4, k // 2] = float("inf"), float("nan"), -float("inf")
    q = ops.quantize_int8(x)
    bad = torch.tensor([False, True, False, True, True, False], device="cuda")
    assert torch.equal(q.scales.isnan(), bad) and not bool(q.codes[bad].any())
    assert torch.equal(q.codes[~bad], clean.codes[~bad]) and torch.equal(q.scales[~bad], clean.scales[~bad])
    w, _, _ = _matrix(20, k, 3)
    y = ops.linear_int8(q, w)
    assert bool(y[bad].isnan().all()) and bool(y[~bad].isfinite().all())
    assert bool(ops.dequantize_int8(q)[bad].isnan().all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_takes_rows_at_any_stride(dtype):
    big = torch.randn(9, 700, device="cuda", generator=_gen(0)).to(dtype)
    for x in (big[:, 3:303], big[::2, 5:305], big[:1, 1:301], big[:, ::2], big.t(), big[4:5].expand(3, 700),
              big[:, :600].reshape(9, 2, 300), big[:, 1:601].view(9, 2, 300), big[0], big[0, 1:]):
        q, c = ops.quantize_int8(x), ops.quantize_int8(x.contiguous())
        assert torch.equal(q.codes, c.codes) and torch.equal(q.scales, c.scales)
        assert tuple(q.shape) == tuple(x.shape)
        assert torch.equal(q.codes[..., :x.shape[-1]].double(), _codes(x.float())[0])


# ------------------------------------------------------------------ the norm
@pytest.mark.parametrize("wt", DTYPES)
@pytest.mark.parametrize("yt", [None, torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,k", ROWS)
def test_norm_is_the_definition(m, k, yt, wt):
    g = _gen(m * 3 + k)
    x = torch.randn(m, k, device="cuda", generator=g) * 3
    y = None if yt is None else torch.randn(m, k, device="cuda", generator=g).to(yt)
    w = (1 + 0.3 * torch.randn(k, device="cuda", generator=g)).to(wt)
    if m > 2:
        x[1] = 0.0
        if y is not None:
            y[1] = 0.0
    h = x if y is None else x + y.float()
    keep = x.clone()
    out = torch.full_like(x, 7.0)
    q = ops.add_rmsnorm_int8(x, w, 1e-5, y=y, x_out=out, dtype=wt)
    assert torch.equal(x, keep) and torch.equal(out, h) and q.dtype == wt
    want, a = _codes(h * w.float())
    assert torch.equal(q.codes[:, :k].double(), want) and not bool(q.codes[:, k:].any())
    r = (h.double().pow(2).mean(-1) + 1e-5).rsqrt()
    # the sum of squares: every lane's run of them and a few steps of a tree, all positive; half of that in its root;
    # the root itself, the product, the division
    tol = 2.0 ** -24 * (0.5 * (k / 64 + 12) + 8)
    assert bool(((q.scales.double() - a[:, 0] * r / 127).abs() <= tol * a[:, 0] * r / 127).all())
    # in place, over a float y, and without a stored sum
    for over in (["x"] if y is None else ["x", "y"] if yt == torch.float32 else ["x"]):
        x2, y2 = x.clone(), None if y is None else y.clone()
        to = x2 if over == "x" else y2
        p = ops.add_rmsnorm_int8(x2, w, 1e-5, y=y2, x_out=to)
        assert torch.equal(to, h) and torch.equal(p.codes, q.codes) and torch.equal(p.scales, q.scales)
    p = ops.add_rmsnorm_int8(x, w, 1e-5, y=y)
    assert torch.equal(p.codes, q.codes) and torch.equal(p.scales, q.scales) and torch.equal(x, keep)


def test_norm_agrees_with_the_float_norm():
    x = torch.randn(4, 6, 768, device="cuda", generator=_gen(1))
    y = torch.randn(4, 6, 768, device="cuda", generator=_gen(2))
    w = 1 + 0.3 * torch.randn(768, device="cuda", generator=_gen(3))
    q = ops.add_rmsnorm_int8(x, w, 1e-5, y=y)
    ref = ops.add_rmsnorm(x, w, 1e-5, y=y)
    assert tuple(q.shape) == (4, 6, 768)
    # half a step of each row's codes, and float roundings
    assert bool(((ops.dequantize_int8(q) - ref).abs() <= 0.5 * q.scales[..., None] + 2.0 ** -20 * ref.abs().amax(-1, True)).all())


@pytest.mark.parametrize("k", [6, 200, 2048, 50000])
def test_norm_keeps_infinities_and_nan_in_their_row(k):
    x = torch.randn(5, k, device="cuda", generator=_gen(k))
    y = torch.randn(5, k, device="cuda", generator=_gen(k + 1))
    w = torch.ones(k, device="cuda")
    clean = ops.add_rmsnorm_int8(x, w, 1e-5, y=y)
    x[1, k - 1], y[3, 0] = float("inf"), float("nan")
    q = ops.add_rmsnorm_int8(x, w, 1e-5, y=y)
    bad = torch.tensor([False, True, False, True, False], device="cuda")
    assert torch.equal(q.scales.isnan(), bad) and not bool(q.codes[bad].any())
    assert torch.equal(q.codes[~bad], clean.codes[~bad]) and torch.equal(q.scales[~bad], clean.scales[~bad])
    w[k // 2] = float("nan")
    assert bool(ops.add_rmsnorm_int8(x, w, 1e-5).scales.isnan().all())


# ------------------------------------------------------------------ the product
SIZES = [(1, 1, 1), (1, 16, 128), (2, 15, 31), (3, 17, 129), (1, 768, 1536), (5, 768, 1536), (8, 33, 700), (16, 1001, 777),
         (17, 100, 2048), (33, 48, 96), (64, 257, 1300), (65, 130, 300), (1, 8192, 2048), (4, 40, 9000), (100, 1000, 1000),
         (130, 768, 1536), (256, 512, 640), (257, 513, 129), (300, 3, 4097), (1000, 777, 333), (512, 2048, 256),
         (1025, 1027, 1030), (1, 70000, 64), (2000, 5, 131), (3, 300, 131071)]


def _reference(x, w, xs, ws, bias):
    """(the product in float64, what its rounding to float32 may be off by)"""
    p = (x @ w.t().contiguous()) * xs[:, None] * ws
    y = p if bias is None else p + bias.double()
    # the sum as a float, times one scale, times the other, and with a bias
    return y, 3.01 * 2.0 ** -24 * p.abs() + 2.0 ** -24 * y.abs()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_linear_matches_float64(m, n, k, dtype):
    x, xc, xs = _matrix(m, k, m + k, dtype)
    w, wc, ws = _matrix(n, k, n + k)
    bias = torch.randn(n, device="cuda", generator=_gen(7)).to(dtype) if m % 2 else None
    ref, off = _reference(xc, wc, xs, ws, bias)
    y = ops.linear_int8(x, w, bias)
    assert y.dtype == dtype and y.shape == (m, n)
    assert bool(((y.double() - ref).abs() <= off + HALF[dtype] * (ref.abs() + off)).all())
    assert torch.equal(y, ops.linear_int8(x, w, bias))          # the same bits every time


# (each form that mtl_linear_int8 chooses, with partial tiles; the last two run a chain of tiles over partial ones)
FORMS = [(40, 70, 200), (5, 100, 4100), (17, 24700, 200), (50, 24701, 270), (250, 2001, 300), (250, 8100, 130), (500, 8101, 300),
         (1000, 8100, 300), (6001, 8203, 300), (6000, 8200, 1025), (33000, 700, 250), (33000, 2100, 129),
         (500, 8101, 2500), (1000, 8101, 4100), (600, 2600, 4200), (16300, 4096, 300), (7001, 4100, 1100),
         # (rows of whole lines, which go past the caches)
         (250, 2048, 300), (250, 8192, 130), (500, 8192, 2500), (1000, 8192, 4100), (500, 8192, 300), (1000, 8192, 300), (136, 10944, 100),
         (50000, 4096, 300)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("m,n,k", FORMS)
def test_every_form_matches_float64(m, n, k, bias, dtype):
    x, xc, xs = _matrix(m, k, m + k, dtype)
    w, wc, ws = _matrix(n, k, n + k)
    b = torch.randn(n, device="cuda", generator=_gen(7)).to(dtype) if bias else None
    for out in (None, torch.full((m, n + 5), 3.0, device="cuda", dtype=dtype)):       # (rows on 16 bytes or not)
        y = ops.linear_int8(x, w, b, out=None if out is None else out[:, 2:n + 2])
        if out is not None:
            assert bool((out[:, :2] == 3.0).all()) and bool((out[:, n + 2:] == 3.0).all())
        for i in range(0, m, 4096):
            ref, off = _reference(xc[i:i + 4096], wc, xs[i:i + 4096], ws, b)
            got = y[i:i + 4096].double()
            assert bool(((got - ref).abs() <= off + HALF[dtype] * (ref.abs() + off)).all())
    first = ops.linear_int8(x, w, b)
    assert all(torch.equal(first, ops.linear_int8(x, w, b)) for _ in range(3))


def test_offsets_past_32_bits():
    # codes of 8.6 GB, and an output of 2.4e9 values
    n, k = 1 << 20, 8192
    codes = torch.randint(-127, 128, (n, k), device="cuda", generator=_gen(0), dtype=torch.int8)
    w = ops.Int8(codes, torch.full((n,), 0.01, device="cuda"), k)
    for m in (1, 40):
        x, xc, xs = _matrix(m, k, m)
        y = ops.linear_int8(x, w)
        for rows in (slice(0, 100), slice(n - 100, n)):
            ref, off = _reference(xc, codes[rows].double(), xs, w.scales[rows].double(), None)
            assert bool(((y[:, rows].double() - ref).abs() <= off + HALF[torch.float32] * ref.abs()).all())
    back = ops.dequantize_int8(w, torch.bfloat16)
    for rows in (slice(0, 5), slice(n - 5, n)):
        assert torch.equal(back[rows], (codes[rows].float() * w.scales[rows, None]).bfloat16())
    q = ops.quantize_int8(back)
    for rows in (slice(0, 5), slice(n - 5, n)):
        assert torch.equal(q.codes[rows].double(), _codes(back[rows].float())[0])
    del codes, w, back, q
    x, xc, xs = _matrix(40000, 128, 1)
    w, wc, ws = _matrix(60000, 128, 2)
    y = ops.linear_int8(x, w)
    for rows in (slice(0, 64), slice(39936, 40000)):
        ref, off = _reference(xc[rows], wc, xs[rows], ws, None)
        assert bool(((y[rows].double() - ref).abs() <= off + HALF[torch.float32] * ref.abs()).all())


# ------------------------------------------------------------------ one float row
ROW_SIZES = [(1, 1), (16, 128), (15, 127), (17, 129), (768, 1536), (1001, 777), (2048, 4096), (33, 4097), (100, 5121),
             (257, 8192), (8192, 2048), (16384, 64), (16385, 64), (40, 8193)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,k", ROW_SIZES)
def test_a_float_row_gives_the_bits_of_its_codes(n, k, dtype):
    w, _, _ = _matrix(n, k, n + k)
    bias = torch.randn(n, device="cuda", generator=_gen(7)).to(dtype)
    x = torch.randn(5, k, device="cuda", generator=_gen(n)).to(dtype)
    x[1] = 0.0
    x[2, k // 2], x[3, k - 1] = float("inf"), float("nan")
    x[4, 0] = 100.0
    for i in range(5):
        for b in (None, bias):
            want = ops.linear_int8(ops.quantize_int8(x[i]), w, b)
            assert want.shape == (n,) and want.dtype == dtype
            for row, shape in ((x[i], (n,)), (x[i:i + 1], (1, n)), (x[i].view(1, 1, k), (1, 1, n)),
                               (torch.stack([x[i], x[0]], 1)[:, 0], (n,))):
                y = ops.linear_int8(row, w, b)
                assert y.shape == shape and torch.equal(y.view(-1).isnan(), want.isnan())
                assert torch.equal(y.view(-1).nan_to_num(7.0), want.nan_to_num(7.0))
    # rows of x past 16 bytes' alignment, y too, and what lies beside it
    out = torch.full((n + 5,), 3.0, device="cuda", dtype=dtype)
    flat = torch.cat([x[4].new_zeros(3), x[4]])
    ops.linear_int8(flat[3:], w, bias, out=out[2:n + 2])
    assert torch.equal(out[2:n + 2], want) and bool((out[:2] == 3.0).all()) and bool((out[n + 2:] == 3.0).all())
    # more rows than one, from floats
    assert torch.equal(ops.linear_int8(x[3:], w, bias).isnan(), ops.linear_int8(ops.quantize_int8(x[3:]), w, bias).isnan())
    assert torch.equal(ops.linear_int8(x[3:], w, bias)[1], want)


@pytest.mark.parametrize("wt", DTYPES)
@pytest.mark.parametrize("n,k", [(16, 1), (15, 127), (17, 129), (100, 777), (768, 768), (2049, 2048), (33, 3333), (64, 4096)])
def test_a_float_row_with_its_norm(n, k, wt):
    g = _gen(n + k)
    x, y = (torch.randn(1, k, device="cuda", generator=g) * 3 for _ in range(2))
    nw = (1 + 0.3 * torch.randn(k, device="cuda", generator=g)).to(wt)
    w, _, _ = _matrix(n, k, 1)
    bias = torch.randn(n, device="cuda", generator=g).to(wt)
    for add in (None, y):
        h, keep = torch.full((1, k + 2), 7.0, device="cuda"), x.clone()
        want_h = torch.empty_like(x)
        q = ops.add_rmsnorm_int8(x, nw, 1e-5, y=add, x_out=want_h, dtype=wt)
        want = ops.linear_int8(q, w, bias)
        for f32 in (0, 1):
            want_y = want if wt == torch.float32 or not f32 else \
                ops.linear_int8(ops.Int8(q.codes, q.scales, k), w, bias.float())
            got = torch.full((n + 1,), 5.0, device="cuda", dtype=torch.float32 if f32 else wt)
            a = _lib.RowLinearInt8Args(x.data_ptr(), None if add is None else add.data_ptr(), h.data_ptr() + 4, nw.data_ptr(),
                                       w.codes.data_ptr(), w.scales.data_ptr(), bias.data_ptr(), got.data_ptr(), n, k, 1e-5,
                                       ops._ACT_DTYPES[wt], f32, 0)
            _lib.check(_lib.load().mtl_row_linear_int8(ctypes.byref(a), ops._stream(x)), "row_linear_int8")
            assert torch.equal(got[:n], want_y[0]) and float(got[n]) == 5.0
            assert torch.equal(h[0, 1:k + 1], want_h[0]) and float(h[0, 0]) == float(h[0, -1]) == 7.0
            assert torch.equal(x, keep)


def test_sums_are_exact_at_the_largest_codes():
    k = 131071
    for a, b in ((127, 127), (-127, 127), (-128, -128)):
        x = ops.pack_int8(torch.full((3, k), a, device="cuda", dtype=torch.int8), torch.ones(3, device="cuda"))
        w = ops.pack_int8(torch.full((70, k), b, device="cuda", dtype=torch.int8), torch.ones(70, device="cuda"))
        y = ops.linear_int8(x, w)
        assert bool((y == torch.tensor(float(a * b * k), device="cuda")).all())
    # small sums come out whole: the order of the sum does not show
    x, xc, _ = _matrix(200, 300, 1)
    w, wc, _ = _matrix(300, 300, 2)
    one = lambda q: ops.Int8(q.codes, torch.ones_like(q.scales), q.k)
    assert torch.equal(ops.linear_int8(one(x), one(w)).double(), xc @ wc.t().contiguous())


@pytest.mark.parametrize("m", [1, 7, 40, 300])
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_writes_its_rows_and_nothing_else(m, dtype):
    x, xc, xs = _matrix(m, 300, 1, dtype)
    w, wc, ws = _matrix(100, 300, 2)
    want = ops.linear_int8(x, w)
    for c0, width in ((7, 130), (8, 128), (0, 101)):
        room = torch.full((m + 2, width), 3.0, device="cuda", dtype=dtype)
        got = ops.linear_int8(x, w, out=room[1:m + 1, c0:c0 + 100])
        assert torch.equal(got, want)
        room[1:m + 1, c0:c0 + 100] = 3.0
        assert bool((room == 3.0).all())
        room = torch.full((m + 2, width + 210), 3.0, device="cuda", dtype=dtype)
        ops.dequantize_int8(x, dtype, out=room[1:m + 1, c0:c0 + 300])
        assert torch.equal(room[1:m + 1, c0:c0 + 300], ops.dequantize_int8(x, dtype))
        room[1:m + 1, c0:c0 + 300] = 3.0
        assert bool((room == 3.0).all())


def test_leading_dimensions_and_no_rows():
    x = torch.randn(2, 3, 40, device="cuda", generator=_gen(0))
    w, _, _ = _matrix(10, 40, 1)
    flat = ops.linear_int8(ops.quantize_int8(x.view(6, 40)), w)
    assert torch.equal(ops.linear_int8(ops.quantize_int8(x), w), flat.view(2, 3, 10))
    assert torch.equal(ops.linear_int8(ops.quantize_int8(x[0, 0]), w), flat[0])
    for lead in ((0,), (2, 0)):
        q = ops.quantize_int8(torch.empty(*lead, 40, device="cuda"))
        assert ops.linear_int8(q, w).shape == (*lead, 10) and ops.dequantize_int8(q).shape == (*lead, 40)
        assert ops.add_rmsnorm_int8(torch.empty(*lead, 40, device="cuda"), torch.ones(40, device="cuda"), 1e-5).shape == (*lead, 40)


@pytest.mark.parametrize("sx,sw", [(1e-30, 1e-6), (1e30, 1e-30), (1e-20, 1e20), (3e30, 1e2)])
def test_large_and_small_scales(sx, sw):
    x, xc, xs = _matrix(5, 300, 1)
    w, wc, ws = _matrix(70, 300, 2)
    x = ops.Int8(x.codes, x.scales * sx, 300)
    w = ops.Int8(w.codes, w.scales * sw, 300)
    ref, off = _reference(xc, wc, x.scales.double(), w.scales.double(), None)
    assert bool(((ops.linear_int8(x, w).double() - ref).abs() <= off + 2.0 ** -149).all())


# ------------------------------------------------------------------ streams and graphs
def _run(x, y, w, weights, bias):
    q = ops.add_rmsnorm_int8(x, weights, 1e-5, y=y)
    z = ops.linear_int8(q, w, bias)
    return z, ops.linear_int8(ops.quantize_int8(z), w.rows(0, 40)), ops.dequantize_int8(q)


def _operands(m, k, n, seed):
    g = _gen(seed)
    w, _, _ = _matrix(n, k, seed + 1)
    # (n = k: the second product's columns)
    return (torch.randn(m, k, device="cuda", generator=g), torch.randn(m, k, device="cuda", generator=g), w,
            torch.ones(k, device="cuda"), torch.randn(n, device="cuda", generator=g))


@pytest.mark.parametrize("m", [1, 40, 300])
def test_replays_equal_the_eager_calls(m):
    a = _operands(m, 640, 640, m)
    want = _run(*a)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        _run(*a)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _run(*a)
    for i in range(3):
        a[0].copy_(torch.randn(m, 640, device="cuda", generator=_gen(100 + i)))
        want = _run(*a)
        for t in got:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(u, v) for u, v in zip(got, want))


def test_two_streams_at_once():
    jobs = [_operands(m, 640, 640, m) for m in (1, 40, 300, 17)]
    want = [_run(*a) for a in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    got = []
    for _ in range(5):
        for s, a in zip(streams, jobs):
            with torch.cuda.stream(s):
                got.append(_run(*a))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert all(torch.equal(u, v) for u, v in zip(g, want[i % len(jobs)]))


@pytest.mark.parametrize("wt", DTYPES)
def test_a_float_row_takes_buffers_side_by_side(wt):
    # x, add, x_out and y follow each other without a gap
    n, k = 100, 300
    g = _gen(5)
    w, _, _ = _matrix(n, k, 1)
    nw = (1 + 0.3 * torch.randn(k, device="cuda", generator=g)).to(wt)
    room = torch.randn(3 * k + n, device="cuda", generator=g)
    x, add, h = room[:k].clone()[None], room[k:2 * k].clone()[None], torch.empty(1, k, device="cuda")
    want = ops.linear_int8(ops.add_rmsnorm_int8(x, nw, 1e-5, y=add, x_out=h, dtype=wt), w)
    at = lambda i: room.data_ptr() + 4 * i * k
    a = _lib.RowLinearInt8Args(at(0), at(1), at(2), nw.data_ptr(), w.codes.data_ptr(), w.scales.data_ptr(), None, at(3), n, k,
                               1e-5, ops._ACT_DTYPES[wt], 0, 0)
    _lib.check(_lib.load().mtl_row_linear_int8(ctypes.byref(a), ops._stream(x)), "row_linear_int8")
    assert torch.equal(room[:k], x[0]) and torch.equal(room[k:2 * k], add[0]) and torch.equal(room[2 * k:3 * k], h[0])
    assert torch.equal(room[3 * k:].view(wt)[:n], want[0])
