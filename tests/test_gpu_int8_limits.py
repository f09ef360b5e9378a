"""More rows than one launch has threads for, and the products whose stores or tiles depend on the size of y: quantize_int8,
add_rmsnorm_int8, dequantize_int8, linear_int8 and the product of one float row."""
import ctypes

import pytest
import torch

from mamba_lite import _lib, ops

pytestmark = pytest.mark.gpu

STEP = 1 << 24                                             # rows checked at a time


@pytest.fixture(autouse=True)
def _memory():
    torch.cuda.empty_cache()
    yield
    torch.cuda.empty_cache()


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _same_codes(q, t):
    """q's codes are those of the float32 rows that t(slice) gives, by the definition in 64 bits."""
    m, k = q.scales.numel(), q.k
    for i in range(0, m, STEP):
        rows = t(slice(i, min(i + STEP, m))).double()
        a = rows.abs().amax(-1, keepdim=True)
        if not torch.equal(q.codes[i:i + STEP, :k].double(), torch.where(a > 0, (rows * 127 / a).round(), 0.0)):
            return False
        if bool(q.codes[i:i + STEP, k:].any()):
            return False
    return True


def test_rows_into_codes_and_back():
    # 64 threads a row
    m, k = (1 << 26) + 5, 8
    x = torch.randn(m, k, device="cuda", generator=_gen(0), dtype=torch.bfloat16)
    q = ops.quantize_int8(x)
    assert _same_codes(q, lambda s: x[s].float())
    for dt in (torch.bfloat16, torch.float32):
        out = torch.full((m, k), 7.0, device="cuda", dtype=dt)
        ops.dequantize_int8(q, dt, out=out)
        room = torch.full((m, k + 1), 7.0, device="cuda", dtype=dt)          # (rows off 16 bytes)
        ops.dequantize_int8(q, dt, out=room[:, :k])
        for i in range(0, m, STEP):
            want = (q.codes[i:i + STEP, :k].float() * q.scales[i:i + STEP, None]).to(dt)
            assert torch.equal(out[i:i + STEP], want) and torch.equal(room[i:i + STEP, :k], want)
        assert bool((room[:, k] == 7.0).all())


def test_norm():
    m, k = (1 << 26) + 5, 8
    x = torch.randn(m, k, device="cuda", generator=_gen(1))
    y = torch.randn(m, k, device="cuda", generator=_gen(2), dtype=torch.bfloat16)
    w = 1 + 0.3 * torch.randn(k, device="cuda", generator=_gen(3))
    h = torch.full_like(x, 7.0)
    q = ops.add_rmsnorm_int8(x, w, 1e-5, y=y, x_out=h)
    for i in range(0, m, STEP):
        assert torch.equal(h[i:i + STEP], x[i:i + STEP] + y[i:i + STEP].float())
    assert _same_codes(q, lambda s: h[s] * w)
    for rows in (slice(0, 1000), slice(m - 1000, m)):
        t = h[rows].double() * w.double()
        want = t.abs().amax(-1) / 127 * (h[rows].double().pow(2).mean(-1) + 1e-5).rsqrt()
        # the sum of 8 squares, half of it in its root; the root, its product, the division and the row's own products
        assert bool(((q.scales[rows].double() - want).abs() <= 12 * 2.0 ** -24 * want).all())


def test_wide_rows_into_codes():
    # 192 threads a row; the rows are one row, which the library takes as rows 0 elements apart
    k, m = 1025, ((1 << 32) - 1) // 192 + 7
    x = torch.randn(k, device="cuda", generator=_gen(4))
    one = ops.quantize_int8(x)
    codes = torch.zeros(m, one.codes.numel(), device="cuda", dtype=torch.int8)
    scales = torch.zeros(m, device="cuda")
    _lib.check(_lib.load().mtl_quantize_int8(x.data_ptr(), 0, codes.data_ptr(), scales.data_ptr(), m, k, 0, ops._stream(x)),
               "quantize_int8")
    assert bool((scales == one.scales).all())
    want = one.codes.view(torch.int64)
    for i in range(0, m, 1 << 21):
        assert bool((codes[i:i + (1 << 21)].view(torch.int64) == want).all())


def test_product_of_more_rows_than_one_launch_takes():
    m, n, k = (1 << 29) + 5, 3, 100
    codes = torch.zeros(m, 128, device="cuda", dtype=torch.int8)
    some = [slice(0, 300), slice((1 << 29) - 300, (1 << 29) + 5)]
    for i, rows in enumerate(some):
        codes[rows, :k] = torch.randint(-127, 128, (rows.stop - rows.start, k), device="cuda", generator=_gen(i), dtype=torch.int8)
    x = ops.Int8(codes, torch.full((m,), 0.02, device="cuda"), k, torch.bfloat16)
    wc = torch.randint(-127, 128, (n, k), device="cuda", generator=_gen(9), dtype=torch.int8)
    w = ops.pack_int8(wc, torch.tensor([0.5, 1.0, 2.0], device="cuda"))
    out = torch.full((m, n), 7.0, device="cuda", dtype=torch.bfloat16)
    ops.linear_int8(x, w, out=out)
    for rows in some:
        ref = codes[rows, :k].double() @ wc.double().t().contiguous() * float(x.scales[0]) * w.scales.double()
        # the float of the sum, two products; and the output's rounding
        assert bool(((out[rows].double() - ref).abs() <= (3.01 * 2.0 ** -24 + 1.01 * 2.0 ** -8) * ref.abs()).all())
    for i in range(some[0].stop, some[1].start, 1 << 26):
        assert not bool(out[i:min(i + (1 << 26), some[1].start)].any())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_float_row_through_more_columns_than_one_launch_takes(dtype):
    n, k = 1 << 27, 8
    codes = torch.zeros(n, 128, device="cuda", dtype=torch.int8)
    some = [slice(0, 300), slice((1 << 26) - 300, (1 << 26) + 300), slice(n - 300, n)]
    for i, rows in enumerate(some):
        codes[rows, :k] = torch.randint(-127, 128, (rows.stop - rows.start, k), device="cuda", generator=_gen(i), dtype=torch.int8)
    w = ops.Int8(codes, torch.full((n,), 0.02, device="cuda"), k)
    bias = torch.randn(n, device="cuda", generator=_gen(7)).to(dtype)
    x, norm = torch.randn(1, k, device="cuda", generator=_gen(8)), torch.ones(k, device="cuda")
    for with_norm in (False, True):
        q = ops.add_rmsnorm_int8(x, norm, 1e-5, dtype=dtype) if with_norm else ops.quantize_int8(x.to(dtype))
        row = x if with_norm else x.to(dtype)
        nw, h = norm.to(dtype), torch.full_like(x, 7.0)
        y = torch.full((n,), 7.0, device="cuda", dtype=dtype)
        a = _lib.RowLinearInt8Args(row.data_ptr(), None, h.data_ptr() if with_norm else None, nw.data_ptr() if with_norm else None,
                                   w.codes.data_ptr(), w.scales.data_ptr(), bias.data_ptr(), y.data_ptr(), n, k, 1e-5,
                                   ops._ACT_DTYPES[dtype], 0, 0)
        _lib.check(_lib.load().mtl_row_linear_int8(ctypes.byref(a), ops._stream(x)), "row_linear_int8")
        assert torch.equal(y, ops.linear_int8(q, w, bias)[0])
        assert torch.equal(h, x) or not with_norm


# ------------------------------------------------------------------ the size of y, and chains of tiles
def _int8(rows, k, seed, dtype=torch.float32):
    g = _gen(seed)
    codes = torch.randint(-127, 128, (rows, k), device="cuda", generator=g, dtype=torch.int8)
    return ops.pack_int8(codes, (torch.rand(rows, device="cuda", generator=g) + 0.5) * 0.01, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
# (rows of whole lines: up to 28 MB in fp32 and in bf16, a row more, and a chain's around 384 MB)
@pytest.mark.parametrize("m,n,k", [(740, 8192, 4100), (768, 8192, 4100), (769, 8192, 4100), (1536, 8192, 2048), (1537, 8192, 2048),
                                   (40959, 2048, 390), (40960, 2048, 390), (40960, 4096, 390), (896, 8192, 4100), (897, 8192, 4100),
                                   (1792, 8192, 300), (1793, 8192, 300), (49151, 2048, 390), (49152, 2048, 390), (49152, 4096, 390)])
def test_product_at_the_sizes_of_y_where_its_stores_change(m, n, k, dtype):
    x, w = _int8(m, k, m, dtype), _int8(n, k, n)
    bias = torch.randn(n, device="cuda", generator=_gen(1)).to(dtype)
    out = torch.full((m, n), 7.0, device="cuda", dtype=dtype)
    ops.linear_int8(x, w, bias, out=out)
    half = 2.0 ** -24 if dtype == torch.float32 else 2.0 ** -8
    wc = w.codes[:, :k].double().t().contiguous()
    for i in range(0, m, 4096):
        p = x.codes[i:i + 4096, :k].double() @ wc * x.scales[i:i + 4096, None].double() * w.scales.double()
        ref = p + bias.double()
        # the sum as a float, times one scale, times the other and with the bias; the output's rounding
        off = 3.01 * 2.0 ** -24 * p.abs() + 2.0 ** -24 * ref.abs()
        assert bool(((out[i:i + 4096].double() - ref).abs() <= off + half * (ref.abs() + off)).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,k", [(1023, 1024), (1024, 1024), (2048, 1024), (4096, 1020), (4096, 1024), (4097, 1024), (8192, 1024), (8193, 1024),
                                 (32767, 1024), (32768, 1024), (65535, 1024), (65536, 1024), (65536, 1020)])
def test_values_at_the_sizes_where_their_stores_change(m, k, dtype):
    q = _int8(m, k, m, dtype)
    out = torch.full((m + 1, k), 7.0, device="cuda", dtype=dtype)
    ops.dequantize_int8(q, out=out[:m])
    assert torch.equal(out[:m], (q.codes[:, :k].float() * q.scales[:, None]).to(dtype)) and bool((out[m] == 7.0).all())


# (chains of tiles: partial ones and with a bias; whole lines past the caches; the smallest K)
CHAINS = [(3000, 8200, 400, True), (24000, 4096, 390, False), (6001, 8203, 1025, True)]


def _product(x, w, bias, out):
    return ops.linear_int8(x, w, bias, out=out)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,n,k,bias", CHAINS)
def test_chains_replay_what_they_compute_eagerly(m, n, k, bias, dtype):
    x, w = _int8(m, k, 1, dtype), _int8(n, k, 2)
    b = torch.randn(n, device="cuda", generator=_gen(3)).to(dtype) if bias else None
    out = torch.empty(m, n, device="cuda", dtype=dtype)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        _product(x, w, b, out)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _product(x, w, b, out)
    for i in range(3):
        x.codes[:, :k].copy_(torch.randint(-127, 128, (m, k), device="cuda", generator=_gen(10 + i), dtype=torch.int8))
        want = ops.linear_int8(x, w, b)
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_chains_on_streams_side_by_side(dtype):
    jobs = []
    for i, (m, n, k, bias) in enumerate(CHAINS + [(300, 640, 640, True)]):
        b = torch.randn(n, device="cuda", generator=_gen(i)).to(dtype) if bias else None
        jobs.append((_int8(m, k, i, dtype), _int8(n, k, 20 + i), b))
    want = [ops.linear_int8(*a) for a in jobs]
    outs = [[torch.full_like(t, 7.0) for t in want] for _ in range(3)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    for row in outs:
        for s, a, out in zip(streams, jobs, row):
            with torch.cuda.stream(s):
                _product(*a, out)
    torch.cuda.synchronize()
    assert all(torch.equal(t, w) for row in outs for t, w in zip(row, want))
