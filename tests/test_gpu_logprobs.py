"""token_logprobs against float64: sizes from one logit to more than a segment's, masks, ties, strides."""
import pytest
import torch

from mamba_lite import ops

pytestmark = pytest.mark.gpu

INF = float("inf")


def _reference(x, tokens, top):
    """By the definition, in float64, row by row over the last dimension."""
    v = x.shape[-1]
    p = x.reshape(-1, v).double()
    c = tokens.reshape(-1)
    m = p.amax(-1, keepdim=True)                  # (taken off first: ln V is lost beside float32's lowest value)
    empty = m == -INF
    d = p - torch.where(empty, 0.0, m)
    lnp = torch.where(empty, -INF, d - torch.log(d.exp().sum(-1, keepdim=True)))
    h = -(lnp.exp() * torch.where(lnp == -INF, 0.0, lnp)).sum(-1)
    lp = lnp.gather(1, c.clamp(0, v - 1)[:, None])[:, 0]
    lp = torch.where(c < 0, 0.0, torch.where(c >= v, torch.nan, lp))
    order = torch.sort(-p, dim=-1, stable=True)[1][:, :top]
    a = lnp.gather(1, order)
    lead = x.shape[:-1]
    return (lp.view(lead), h.view(lead), a.view(*lead, top),
            torch.where(p.gather(1, order) == -INF, -1, order).view(*lead, top))


def _check(x, tokens, top):
    got, ref = ops.token_logprobs(x, tokens, top=top), _reference(x, tokens, top)
    for g, r in zip(got, ref):
        assert g.shape == r.shape
    assert torch.equal(got.top_token, ref[3])
    for g, r in zip(got[:3], ref[:3]):
        g = g.double()
        assert torch.equal(torch.isnan(g), torch.isnan(r)) and torch.equal(g == -INF, r == -INF)
        ok = torch.isfinite(r)
        # x - m and ln s round once each (2^-24 of |ln p| + ln s, ln s < 20); a term's exponential is off by
        # 2^-24 (|d| + 2) with e^-d |d| < 0.4, and a sum's tree of V terms adds 2^-24 (a thread's share + 20) at most:
        # 2^-24 x 64 of s over a share of a few hundred terms of one sign walks ~sqrt(share)
        e = (g - r).abs()[ok]
        assert bool((e <= 2.0 ** -24 * (2 * r[ok].abs() + 100)).all()), float(e.max())
    return got


def _logits(rows, v, dtype, seed, spread=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(rows, v, device="cuda", generator=g) * spread).to(dtype)
    return x, torch.randint(0, v, (rows,), device="cuda", generator=g)


DTYPES = pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])


@DTYPES
@pytest.mark.parametrize("rows,v", [(1, 1), (3, 2), (2, 63), (5, 64), (1, 65), (7, 257), (2, 1023), (3, 4099), (1, 50280),
                                    (33, 50277), (2, 131073), (300, 1000), (700, 5003), (4100, 257), (1, 400003)])
def test_matches_float64(rows, v, dtype):
    x, c = _logits(rows, v, dtype, rows + v)
    for top in sorted({0, 1, min(5, v), min(64, v)}):
        got = _check(x, c, top)
        again = ops.token_logprobs(x, c, top=top)
        assert all(torch.equal(a, b) for a, b in zip(got, again))


@DTYPES
@pytest.mark.parametrize("rows", [1, 40, 5000])
def test_ties_go_to_the_lowest_index(rows, dtype):
    v = 2000
    x = torch.zeros(rows, v, device="cuda", dtype=dtype)                       # every logit alike
    c = torch.full((rows,), v - 1, device="cuda")
    got = _check(x, c, 64)
    assert torch.equal(got.top_token, torch.arange(64, device="cuda").expand(rows, 64))
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randint(-3, 3, (rows, v), device="cuda", generator=g).to(dtype)   # few values
    _check(x, c, 20)
    x[:, ::2] = -0.0
    x[:, 1::2] = 0.0                                                            # equal, whatever their sign
    assert torch.equal(_check(x, c, 7).top_token[0], torch.arange(7, device="cuda"))


@DTYPES
@pytest.mark.parametrize("rows", [1, 40, 4200])
def test_sorted_rows(rows, dtype):
    v = 3000
    for step in (0.5, -0.5):                                                    # every later logit larger, or smaller
        x = (torch.arange(v, device="cuda") * step).expand(rows, v).to(dtype)
        _check(x, torch.arange(rows, device="cuda") % v, 33)


# one wavefront and several, with one tile each and more, few alternatives a wavefront and many
@DTYPES
@pytest.mark.parametrize("rows,v,top", [(1, 64, 8), (1, 1000, 64), (2, 2049, 33), (3, 9000, 64), (40, 5000, 20), (2, 20011, 64),
                                        (300, 2100, 64), (1100, 20011, 20), (1100, 9000, 64), (1, 131075, 9)])
def test_the_order_of_alternatives(rows, v, top, dtype):
    torch.manual_seed(rows + v)
    x = torch.randn(rows, v, device="cuda") * 3
    lowest = torch.finfo(dtype).min
    some = torch.rand(rows, v, device="cuda")
    for kind in (x, x.sort(-1)[0], x.sort(-1, descending=True)[0], x.round(), torch.full_like(x, 1.5),
                 torch.where(some < 0.95, lowest, x), torch.where(some < 0.95, -INF, x)):
        kind = kind.to(dtype)
        got = ops.token_logprobs(kind, torch.zeros(rows, dtype=torch.int64, device="cuda"), top=top)
        value, order = torch.sort(kind.float(), dim=-1, descending=True, stable=True)
        value, order = value[:, :top], order[:, :top]
        assert torch.equal(got.top_token, torch.where(value == -INF, -1, order))
        assert bool((got.top_logprob[:, 1:] <= got.top_logprob[:, :-1]).all())


@DTYPES
@pytest.mark.parametrize("rows,v", [(1, 7), (1, 50280), (9, 3001), (4200, 300)])
def test_masks(rows, v, dtype):
    x, c = _logits(rows, v, dtype, 5)
    low = torch.finfo(dtype).min
    for fill in (-INF, low):
        for keep in (0, 1, 3):
            y = torch.full_like(x, fill)
            y[:, v - keep:] = x[:, v - keep:]
            got = _check(y, c, min(7, v))
            _check(y, torch.full_like(c, v - 1), 2)
            if fill == -INF and keep == 0:
                assert bool((got.logprob == -INF).all() and (got.entropy == 0).all() and (got.top_token == -1).all()
                            and (got.top_logprob == -INF).all())
    _check(x, torch.full_like(c, -100), 3)                                      # padding
    _check(x, torch.full_like(c, v), 3)                                         # past the vocabulary
    assert bool((ops.token_logprobs(x, torch.full_like(c, -1)).logprob == 0).all())


@DTYPES
@pytest.mark.parametrize("rows,v,at", [(1, 9, 0), (6, 50280, 50279), (4200, 301, 17)])
def test_rows_with_nan_or_infinity(rows, v, at, dtype):
    x, c = _logits(rows, v, dtype, 6)
    bad = rows // 2
    for value in (float("nan"), INF):
        y = x.clone()
        y[bad, at] = value
        got = ops.token_logprobs(y, c, top=3)
        assert bool(torch.isnan(got.logprob[bad]) and torch.isnan(got.entropy[bad])
                    and torch.isnan(got.top_logprob[bad]).all() and (got.top_token[bad] == -1).all())
        rest = [i for i in range(rows) if i != bad]
        if rest:
            want = ops.token_logprobs(x, c, top=3)
            assert all(torch.equal(g[rest], w[rest]) for g, w in zip(got, want))
    y[bad] = -INF
    y[bad, at] = INF
    assert bool(torch.isnan(ops.token_logprobs(y, c).entropy[bad]))
    c[bad] = -100
    assert float(ops.token_logprobs(y, c).logprob[bad]) == 0.0


@DTYPES
def test_large_and_close_values(dtype):
    x, c = _logits(20, 1000, dtype, 7)
    _check((x.float() * 1e4).to(dtype), c, 5)
    _check((x.float() + 3e4).to(dtype), c, 5)
    _check((x.float() * 1e-3).to(dtype), c, 5)
    x[:, 17] = 80.0                                                             # one certain token
    got = _check(x, torch.full_like(c, 17), 5)
    assert bool((got.entropy >= 0).all() and (got.logprob <= 0).all())


@DTYPES
def test_strides_and_shapes(dtype):
    x, _ = _logits(6 * 5, 703, dtype, 8)
    x = x.view(6, 5, 703)
    c = torch.randint(0, 600, (6, 5), device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    _check(x[:, :-1], c[:, 1:], 4)                           # every token but a prompt's first, given the ones before
    _check(x[..., 1:], c, 4)                                 # rows that start off a 16-byte boundary
    _check(x[..., 3:700], c, 64)
    _check(x.transpose(0, 1), c.t(), 4)
    _check(x[:, ::2, ::2], c[:, ::2] // 2, 4)
    _check(x[0, 0], c[0, 0], 4)
    _check(x.view(2, 3, 5, 703)[:, 1:, ::2], c.view(2, 3, 5)[:, 1:, ::2], 4)
    _check(x[:1, 0].expand(4, 703), c[:4, 0], 4)
    e = x.view(2, 3, 5, 703)[:, :, :0]
    assert ops.token_logprobs(e, c.view(2, 3, 5)[:, :, :0], top=2).top_logprob.shape == (2, 3, 0, 2)
    r = ops.token_logprobs(x[:0], c[:0], top=3)
    assert r.logprob.shape == (0, 5) and r.top_token.shape == (0, 5, 3)


def test_streams_and_graph_replays():
    x, c = _logits(3, 50280, torch.float32, 9)
    want = ops.token_logprobs(x, c, top=5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.token_logprobs(x, c, top=5)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    sx, sc = x.clone(), c.clone()
    graphs = []
    for _ in range(2):                                       # two graphs of one pool, replayed in turn
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=graphs[0][0].pool() if graphs else None):
            out = ops.token_logprobs(sx, sc, top=5)
        graphs.append((g, out))
    for i in range(4):
        sx.copy_(x.roll(i + 1, 1))
        sc.copy_((c + 7 * i) % 50280)
        eager = ops.token_logprobs(sx, sc, top=5)
        for g, out in graphs:
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, eager))


def test_refusals_on_the_gpu():
    x, c = _logits(3, 100, torch.float32, 10)
    with pytest.raises(RuntimeError, match="operands"):
        ops.token_logprobs(x, c.cpu())
    with pytest.raises(RuntimeError, match="backward"):
        ops.token_logprobs(x.requires_grad_(), c)
    with torch.no_grad():
        ops.token_logprobs(x, c)


def test_four_bit_head_then_log_probabilities():
    """The two as a step of serving uses them: a 4-bit lm_head, then the token's log probability and alternatives."""
    g = torch.Generator(device="cuda").manual_seed(11)
    W = torch.randn(5003, 256, device="cuda", generator=g) * 0.1
    w4 = ops.quantize_w4(W, 64)
    h = torch.randn(4, 256, device="cuda", generator=g)
    logits = ops.linear_w4(h, w4)
    ref = h.double() @ ops.dequantize_w4(w4).double().t().contiguous()
    got = _check(logits, ref.argmax(-1), 5)
    want = _reference(ref, ref.argmax(-1), 5)
    # logits of norm ~1.6 with 2^-24 x (16 + 6 x 8 + 4) of it, as in the product's own test
    assert float((got.top_logprob.double() - want[2]).abs().max()) < 2.0 ** -24 * (100 + 10 * 68)
    # rounding to 4 bits with one scale for 64 weights (7 steps to the largest of about 2.4 sigma): an eighth of a
    # sigma in each weight at most by the uniform error of a step, 2.6 / 7 / sqrt(12) = 0.107
    full = h.double() @ W.double().t().contiguous()
    assert float((ref - full).norm() / full.norm()) < 0.13
