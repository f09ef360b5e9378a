"""LinearW4, a model whose projections and lm_head are in 4-bit codes, and log probabilities through the model: each
against the same computation on the matrices that the codes stand for."""
import copy

import pytest
import torch
import torch.nn.functional as F

from mamba_lite import ops
from mamba_lite.cuda_graph import GraphedPrefill, GraphedStepper
from mamba_lite.model import LinearW4, MambaCache, MambaConfig, MambaLM

pytestmark = pytest.mark.gpu

# The two sides differ in how fp32 sums of at most 2048 products are ordered, 2^-24 sqrt(2048) of each product's norm, as
# tests of the per-op and one-call paths against each other do (1e-5 there for two layers)
TOL = 1e-5


def _rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


def _model(d_model=256, n_layer=2, dtype=torch.float32, **kw):
    torch.manual_seed(d_model + n_layer)
    m = MambaLM(MambaConfig(d_model=d_model, n_layer=n_layer, vocab_size=1003, **kw)).cuda().eval()
    with torch.no_grad():
        for blk in m.layers:                        # small steps, as a trained model takes them
            blk.mixer.dt_proj.bias.uniform_(-4.0, -2.0)
    return m.to(dtype)


def _on_matrices(q):
    """A model of plain projections that hold the quantized ones' matrices."""
    m = copy.deepcopy(q)
    for blk in m.layers:
        for name in ("in_proj", "out_proj"):
            w = getattr(blk.mixer, name)
            lin = torch.nn.Linear(w.in_features, w.out_features, bias=w.bias is not None).cuda().to(q.embedding.weight.dtype)
            with torch.no_grad():
                lin.weight.copy_(ops.dequantize_w4(w.w4(), lin.weight.dtype))
                if w.bias is not None:
                    lin.bias.copy_(w.bias)
            setattr(blk.mixer, name, lin)
    m._modules.pop("head_w4", None)
    return m


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("zero_points,bias", [(False, True), (True, False)])
def test_linear_w4_module(zero_points, bias, dtype):
    torch.manual_seed(0)
    lin = torch.nn.Linear(300, 200, bias=bias).cuda().to(dtype)
    q = LinearW4.from_linear(lin, 32, zero_points)
    w = ops.dequantize_w4(q.w4(), torch.float32).double()
    step = q.scales.max().item() * (1.5 if zero_points else 1.0)       # half a step, and the end of the range
    assert float((w - lin.weight.detach().double()).abs().max()) <= step
    tol = TOL if dtype == torch.float32 else 2.0 ** -7                 # the output's and (many rows) the matrix's rounding
    with torch.no_grad():
        for shape in ((300,), (1, 300), (4, 5, 300), (64, 300), (65, 300), (3, 40, 300), (1500, 300)):
            x = torch.randn(shape, device="cuda").to(dtype)
            ref = x.double() @ w.t().contiguous() + (lin.bias.double() if bias else 0)
            y = q(x)
            assert y.dtype == dtype and y.shape == ref.shape and _rel(y, ref) < tol
        again = copy.deepcopy(q)
        again.load_state_dict(q.state_dict())
        assert torch.equal(again(x[:3]), q(x[:3]))
    x = torch.randn(5, 300, device="cuda", dtype=dtype, requires_grad=True)   # the matrix's product, with x's gradient
    g = torch.randn(5, 200, device="cuda").to(dtype)
    q(x).backward(g)
    assert _rel(x.grad, g.double() @ w) < tol and q.weight.grad is None


@pytest.mark.parametrize("kw", [dict(), dict(zero_points=True, group=128, scale_dtype=torch.float32)])
@pytest.mark.parametrize("b,l", [(1, 5), (3, 30), (2, 200)])
def test_prefill_and_steps_are_those_of_the_matrices(b, l, kw):
    q = _model(bias=True).quantize_w4(lm_head=False, **kw)
    ref = _on_matrices(q)
    ids = torch.randint(0, 1003, (b, l + 4), device="cuda")
    with torch.no_grad():
        got, cq = q.prefill(ids[:, :l])
        want, cr = ref.prefill(ids[:, :l])
        assert _rel(got, want) < TOL
        for t in range(l, l + 4):
            got, want = q.step(ids[:, t:t + 1], cq), ref.step(ids[:, t:t + 1], cr)
            assert _rel(got, want) < TOL
        for a, c in zip(cq.layers, cr.layers):
            assert _rel(a.ssm_state, c.ssm_state) < TOL and _rel(a.conv_state, c.conv_state) < TOL


def test_bf16_model():
    q = _model(d_model=512, dtype=torch.bfloat16).quantize_w4()
    ref = _on_matrices(q)
    ids = torch.randint(0, 1003, (2, 20), device="cuda")
    with torch.no_grad():
        head = ops.dequantize_w4(q.head_w4.w4(), torch.bfloat16)
        got, cq = q.prefill(ids[:, :19])
        xf, cr = ref._prefill_hidden(ids[:, :19])
        # activations rounded to bf16 between a dozen operations: 2^-8 each, a walk of them
        assert _rel(got, F.linear(xf, head)) < 2.0 ** -8 * 6
        assert q.step(ids[:, 19:], cq).shape == (2, 1, q.cfg.vocab_size)


def test_the_head_and_the_one_call_plans():
    m = _model()
    ids = torch.randint(0, 1003, (2, 40), device="cuda")
    with torch.no_grad():
        before, cache = m.prefill(ids)                     # makes the plain model's call plans
        m.step(ids[:, :1], cache)
        plain = copy.deepcopy(m)
        q = m.quantize_w4(group=32)
        assert q is m
        got, _ = q.prefill(ids)
        ref = _on_matrices(q)
        xf, _ = ref._prefill_hidden(ids)
        w = ops.dequantize_w4(q.head_w4.w4())
        assert _rel(got, F.linear(xf, w)) < TOL
        # 16 values for 32 weights: a step of about a seventh of 2.2 sigma, an error of 0.09 sigma in each of the three
        # products of a layer and in the head
        assert _rel(got, before) < 0.5
        assert _rel(plain.prefill(ids)[0], before) == 0.0
    with pytest.raises(TypeError, match="plain nn.Linear"):
        q.quantize_w4()
    state = q.state_dict()
    other = _model().quantize_w4(group=32)
    with torch.no_grad():
        for p in other.parameters():
            p.zero_()
    other.load_state_dict(state)
    with torch.no_grad():
        assert torch.equal(other.prefill(ids)[0], got)


@pytest.mark.parametrize("b", [1, 3])
def test_captured_prefill_and_steps(b):
    q = _model().quantize_w4()
    ids = torch.randint(0, 1003, (b, 24), device="cuda")
    with torch.no_grad():
        cache = MambaCache.allocate(q.cfg, b, "cuda", torch.float32)
        pre = GraphedPrefill(q, cache, b, 16, "cuda")
        pre.capture()
        step = GraphedStepper(q, cache, b, "cuda")
        step.capture()
        for turn in range(2):
            prompt = ids.roll(turn, 1)
            logits = pre.replay(prompt[:, :16])
            want, c2 = q.prefill(prompt[:, :16])
            torch.cuda.synchronize()
            assert torch.equal(logits, want)
            for t in range(16, 20):
                got, want = step.replay(prompt[:, t:t + 1]), q.step(prompt[:, t:t + 1], c2)
                torch.cuda.synchronize()
                assert torch.equal(got, want)


def _reference(logits, given, top):
    lnp = torch.log_softmax(logits.double(), -1)
    a, i = torch.sort(lnp, dim=-1, descending=True, stable=True)
    return (lnp.gather(-1, given[..., None])[..., 0], -(lnp.exp() * lnp).sum(-1), a[..., :top], i[..., :top])


@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("b,l", [(1, 1), (1, 2), (3, 37), (2, 300)])
def test_score(b, l, quantized):
    m = _model()
    if quantized:
        m.quantize_w4()
    ids = torch.randint(0, 1003, (b, l), device="cuda")
    r = m.score(ids, top=3)
    assert r.logprob.shape == r.entropy.shape == (b, l - 1) and r.top_token.shape == r.top_logprob.shape == (b, l - 1, 3)
    if l == 1:
        return
    with torch.no_grad():
        logits, _ = m.prefill(ids)
    want = _reference(logits[:, :-1], ids[:, 1:], 3)
    # the head's product runs over other rows here: TOL of a logit's size, and token_logprobs' own rounding
    tol = 4 * TOL * float(logits.abs().max()) + 2.0 ** -24 * 120
    assert all(float((g - w).abs().max()) < tol for g, w in zip(r[:3], want[:3]))
    gap = (want[2][..., :-1] - want[2][..., 1:]).min(-1)[0] > tol      # where the order is not a matter of rounding
    assert torch.equal(r.top_token[..., 0][gap], want[3][..., 0][gap])
    whole = m._SCORE_LOGITS
    try:
        m._SCORE_LOGITS = 1008 * 7                                     # 7 rows at a time
        parts = m.score(ids, top=3)
    finally:
        m._SCORE_LOGITS = whole
    assert float((parts.logprob - r.logprob).abs().max()) < tol and parts.top_token.shape == r.top_token.shape


@pytest.mark.parametrize("b", [1, 4])
def test_generate_with_log_probabilities(b):
    m = _model().quantize_w4()
    ids = torch.randint(0, 1003, (b, 9), device="cuda")
    tokens = m.generate(ids, 6)
    again, r = m.generate(ids, 6, return_logprobs=True, top=4)
    assert torch.equal(tokens, again) and tokens.shape == (b, 15)
    assert r.logprob.shape == (b, 6) and r.top_token.shape == (b, 6, 4)
    assert torch.equal(r.top_token[..., 0], tokens[:, 9:])             # greedy: the most probable one was taken
    assert torch.equal(r.top_logprob[..., 0], r.logprob)
    s = m.score(tokens, top=1)
    tol = 64 * TOL                                                     # a prompt's logits against the steps'
    assert float((s.logprob[:, 8:] - r.logprob).abs().max()) < tol
    with pytest.raises(ValueError, match="return_logprobs"):
        m.generate(ids, 2, top=3)


SHAPES = [(256, 2, 1, 4, dict()), (320, 2, 3, 2, dict(zero_points=True, group=32)), (512, 2, 17, 3, dict(group=128)),
          (2048, 2, 32, 4, dict(scale_dtype=torch.float32)), (768, 2, 2, 4, dict(zero_points=True))]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dm,expand,b,d_conv,kw", SHAPES)
def test_the_one_call_step(dm, expand, b, d_conv, kw, dtype, monkeypatch):
    """mtl_decode_step_w4 against the steps op by op (fp32: the same launches, the same bits; bf16: as near to the fp32
    step on the same weights), eager and captured."""
    import mamba_lite.model as mm
    q = _model(dm, 2, dtype, expand=expand, d_conv=d_conv, bias=dm == 320).quantize_w4(**kw)
    cache = MambaCache.allocate(q.cfg, b, "cuda", dtype)
    for lc in cache.layers:
        lc.conv_state.normal_(0, 0.6)
        lc.ssm_state.normal_(0, 0.1)
    clone = lambda t=dtype: MambaCache([type(lc)(lc.conv_state.to(t, copy=True), lc.ssm_state.clone())
                                        for lc in cache.layers])
    ids = torch.randint(0, 1003, (b, 2), device="cuda")
    calls = []
    real = ops.decode_step_w4
    monkeypatch.setattr(ops, "decode_step_w4", lambda *a, **k: (calls.append(1), real(*a, **k))[1])
    run = lambda m, c: [m.step(ids[:, t:t + 1], c) for t in range(2)]
    with torch.no_grad():
        c1, c2 = clone(), clone()
        one = run(q, c1)
        assert len(calls) == 2
        monkeypatch.setattr(mm, "BATCHED_STEP_NATIVE", False)
        old = run(q, c2)
        assert len(calls) == 2
        if dtype == torch.float32:
            assert all(torch.equal(x, y) for x, y in zip(one, old))
            assert all(torch.equal(x.ssm_state, y.ssm_state) and torch.equal(x.conv_state, y.conv_state)
                       for x, y in zip(c1.layers, c2.layers))
        else:
            wide = copy.deepcopy(q).float()                    # the same weights, activations in fp32
            c3 = clone(torch.float32)
            ref = run(wide, c3)
            for x, y, r in zip(one, old, ref):
                # a dozen roundings of 2^-8 in a walk; and no further off than op by op, where out_proj's sum is rounded once
                # more.  Both norms hold the n logits' own roundings, independent ones: a root of a sum of n squares
                # spreads by 1 / sqrt(n) of itself at most (uniform errors: 0.45 / sqrt(n)), six of those allowed
                assert _rel(x, r) < 2.0 ** -8 * 6 and _rel(x, r) <= (1 + 6 / r.numel() ** 0.5) * _rel(y, r)
            for x, r in zip(c1.layers, c3.layers):
                assert _rel(x.ssm_state, r.ssm_state) < 2.0 ** -8 * 6
        monkeypatch.setattr(mm, "BATCHED_STEP_NATIVE", True)
        st = GraphedStepper(q, clone(), b, "cuda")
        st.capture()
        for t in range(2):
            got = st.replay(ids[:, t:t + 1])
            torch.cuda.synchronize()
            assert torch.equal(got, one[t])


def test_what_keeps_the_step_op_by_op():
    q = _model(512).quantize_w4()
    cache = MambaCache.allocate(q.cfg, 2, "cuda", torch.float32)
    x = torch.zeros(2, 512, device="cuda")
    with torch.no_grad():
        took = lambda: q._w4_step_layers(x, cache, q._layer_tensors()) is not None
        assert took()
        handle = q.layers[1].mixer.in_proj.register_forward_hook(lambda *_: None)
        assert not took()
        handle.remove()
        assert took() and q._w4_step_layers(torch.zeros(33, 512, device="cuda"), cache, q._layer_tensors()) is None
        q.norm_f.double()
        assert not took()
        q.norm_f.float()
        q.layers[1].mixer.out_proj = torch.nn.Linear(1024, 512, bias=False).cuda()
        assert not took()
        before = q.step(torch.zeros(2, 1, dtype=torch.long, device="cuda"), cache)
        assert bool(torch.isfinite(before).all())
    # weights changed after a step: the next one reads them
    q = _model(512).quantize_w4()
    ids = torch.randint(0, 1003, (2, 1), device="cuda")
    fresh = lambda: MambaCache.allocate(q.cfg, 2, "cuda", torch.float32)
    with torch.no_grad():
        q.step(ids, fresh())
        q.layers[0].mixer.x_proj.weight.mul_(-1.5)
        q.layers[1].mixer.in_proj.scales.mul_(0.5)
        got = q.step(ids, fresh())
        want = copy.deepcopy(q).step(ids, fresh())
        assert torch.equal(got, want)


def test_a_graph_of_replaced_weights_is_refused():
    m = _model()
    cache = MambaCache.allocate(m.cfg, 1, "cuda", torch.float32)
    step, pre = GraphedStepper(m, cache, 1, "cuda"), GraphedPrefill(m, cache, 1, 8, "cuda")
    with torch.no_grad():
        step.capture()
        pre.capture()
        held = [m.layers[0].mixer.in_proj.weight]          # (kept alive here: only the refusal is looked at)
        ids = torch.zeros(1, 8, dtype=torch.long, device="cuda")
        pre.replay(ids)
        step.replay(ids[:, :1])
        m.quantize_w4()
        for call in (lambda: pre.replay(ids), lambda: step.replay(ids[:, :1])):
            with pytest.raises(RuntimeError, match="capture again"):
                call()
        step.capture()
        assert held and bool(torch.isfinite(step.replay(ids[:, :1])).all())


def test_a_long_batch_of_prompts():
    """From 16384 tokens on a plain mixer splits its in_proj; a 4-bit one is called whole."""
    q = _model(64, 1).quantize_w4()
    ref = _on_matrices(q)
    ids = torch.randint(0, 1003, (4, 4100), device="cuda")
    with torch.no_grad():
        got, want = q._prefill_hidden(ids)[0], ref._prefill_hidden(ids)[0]
    assert _rel(got, want) < TOL


def test_a_mixer_by_itself():
    q = _model(256, 1).quantize_w4()
    mx, ref = q.layers[0].mixer, _on_matrices(q).layers[0].mixer
    x = torch.randn(2, 9, 256, device="cuda")
    from mamba_lite.model import LayerCache
    with torch.no_grad():
        y, cs, hs = mx.prefill(x)
        yr, csr, hsr = ref.prefill(x)
        assert _rel(y, yr) < TOL and _rel(hs, hsr) < TOL
        a, b = LayerCache(cs, hs), LayerCache(csr, hsr)
        assert _rel(mx.step(x[:, 0], a), ref.step(x[:, 0], b)) < TOL and _rel(a.ssm_state, b.ssm_state) < TOL


@pytest.mark.parametrize("zero_points", [False, True])
def test_linear_w4_module_under_transforms(zero_points):
    """What torch does around a module it does around this one: few rows (from the codes otherwise) as many."""
    torch.manual_seed(1)
    lin = torch.nn.Linear(300, 200).cuda()
    q = LinearW4.from_linear(lin, 64, zero_points)
    w = ops.dequantize_w4(q.w4(), torch.float32)
    assert torch.equal(ops.w4_matrix(q.w4()), w) and torch.equal(ops.w4_matrix(q.w4(), torch.bfloat16), w.bfloat16())
    for rows in (5, 65):
        x, v = torch.randn(rows, 300, device="cuda"), torch.randn(rows, 300, device="cuda")
        with torch.no_grad():
            want = q(x)
            # forward mode, plain and through functorch
            with torch.autograd.forward_ad.dual_level():
                y, dy = torch.autograd.forward_ad.unpack_dual(q(torch.autograd.forward_ad.make_dual(x, v)))
            assert dy is not None and _rel(y, want) < TOL and _rel(dy, v.double() @ w.double().t().contiguous()) < TOL
            y, dy = torch.func.jvp(q, (x,), (v,))
            assert _rel(y, want) < TOL and _rel(dy, v.double() @ w.double().t().contiguous()) < TOL
            assert _rel(torch.func.vmap(q)(x), want) < TOL
            traced = torch.jit.trace(q, (x,), check_trace=False)
            assert _rel(traced(v), q(v)) < TOL
            seen = []

            class Mode(torch.overrides.TorchFunctionMode):
                def __torch_function__(self, func, types, args=(), kwargs=None):
                    seen.append(func)
                    return func(*args, **(kwargs or {}))

            with Mode():
                q(x)
            assert F.linear in seen
        g = torch.func.grad(lambda x: q(x).square().sum())(x)
        assert _rel(g, 2 * want.double() @ w.double()) < TOL
        bias = q.bias.requires_grad_()                             # a bias that learns
        q(x).sum().backward()
        assert torch.equal(bias.grad, torch.full_like(bias, rows))
        bias.grad = None
        bias.requires_grad_(False)


@pytest.mark.parametrize("l", [20, 100, 700])
def test_prompts_and_steps_under_autocast(l):
    """The layers keep the embedding's type, as a step from the codes does."""
    q = _model(256).quantize_w4()
    ids = torch.randint(0, 1003, (3, l + 1), device="cuda")
    clone = lambda c: MambaCache([type(lc)(lc.conv_state.clone(), lc.ssm_state.clone()) for lc in c.layers])
    with torch.no_grad():
        want, cache = q.prefill(ids[:, :l])
        hidden, _ = q._prefill_hidden(ids[:, :l])
        c1, c2 = clone(cache), clone(cache)
        step = q.step(ids[:, l:], c1)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            assert torch.equal(q._prefill_hidden(ids[:, :l])[0], hidden)
            got, c3 = q.prefill(ids[:, :l])
            assert _rel(got, want) < 2.0 ** -8 * 2                    # the head's operands and logits in bf16
            assert _rel(q.step(ids[:, l:], c2), step) < TOL
        for a, b, c in zip(c1.layers, c2.layers, c3.layers):
            assert _rel(b.ssm_state, a.ssm_state) < TOL and _rel(b.conv_state, a.conv_state) < TOL
            assert c.conv_state.dtype == torch.float32
    lin = torch.nn.Linear(128, 40).cuda()
    m = LinearW4.from_linear(lin)
    x = torch.randn(5, 128, device="cuda", dtype=torch.bfloat16)
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):       # a bias of the module's type, x of autocast's
        ref = x.double() @ ops.dequantize_w4(m.w4()).double().t().contiguous() + lin.bias.double()
        assert m(x).dtype == torch.bfloat16 and _rel(m(x), ref) < 2.0 ** -7   # x's products and the matrix: a rounding each


def test_a_projection_of_another_form_at_the_same_addresses():
    """Groups of 64 with bf16 scales and of 128 with fp32 ones take as many bytes: the step after a swap reads the new ones."""
    m = _model(256)
    other = copy.deepcopy(m)
    q = m.quantize_w4(group=64, scale_dtype=torch.bfloat16)
    other.quantize_w4(group=128, scale_dtype=torch.float32)
    ids = torch.randint(0, 1003, (2, 1), device="cuda")
    fresh = lambda: MambaCache.allocate(q.cfg, 2, "cuda", torch.float32)
    with torch.no_grad():
        q.step(ids, fresh())                                              # the plan is made
        for a, b in zip(q.layers, other.layers):
            for name in ("in_proj", "out_proj"):
                old, new = getattr(a.mixer, name), getattr(b.mixer, name)
                # the new module's values in the old one's memory, as an allocator may place them
                assert old.scales.numel() * 2 == new.scales.numel() * 4
                old.weight.copy_(new.weight)
                scales = old.scales.data.view(-1).view(torch.float32).view(new.scales.shape)
                scales.copy_(new.scales)
                w4 = ops.W4(old.weight.data, scales, None, new.out_features, new.in_features, 128)
                assert w4.scales.data_ptr() == old.scales.data_ptr()
                setattr(a.mixer, name, LinearW4(w4, new.bias))
        q.head_w4 = other.head_w4
        assert torch.equal(q.step(ids, fresh()), other.step(ids, fresh()))


@pytest.mark.parametrize("b", [1, 3])
def test_a_4_bit_head_on_plain_projections(b):
    """Projections put back as matrices, the head left in 4 bits: steps answer through it as prompts do."""
    q = _model(256).quantize_w4()
    m = _on_matrices(q)
    m.head_w4 = q.head_w4
    ids = torch.randint(0, 1003, (b, 6), device="cuda")
    with torch.no_grad():
        _, c1 = q.prefill(ids[:, :5])
        _, c2 = m.prefill(ids[:, :5])
        assert _rel(m.step(ids[:, 5:], c2), q.step(ids[:, 5:], c1)) < TOL


def test_score_takes_what_prefill_takes():
    m = _model()
    ids = torch.randint(0, 1003, (2, 9), device="cuda")
    for a, b in zip(m.score(ids.int(), top=2), m.score(ids, top=2)):
        assert torch.equal(a, b)
    for bad in (ids[:, :0], ids[0]):
        with pytest.raises(ValueError, match="input_ids"):
            m.score(bad)
