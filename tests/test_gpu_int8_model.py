"""LinearInt8 and a model whose projections and lm_head run in 8-bit integers, against the same computation in torch."""
import copy

import pytest
import torch

from mamba_lite import model as mm
from mamba_lite import ops
from mamba_lite.cuda_graph import GraphedPrefill, GraphedStepper
from mamba_lite.model import LinearInt8, MambaCache, MambaConfig, MambaLM

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16]
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
# Two computations whose float roundings differ put a value next to a border into neighbouring codes now and then: its row of
# k values moves by one step, a / 127, of sqrt(k) times its root mean square, a / 4 or more.  Taken for every row, at
# k = 256: 4 / 127 / 16 = 2e-3 a product, and five products follow each other in two layers and a head.
TOL = {torch.float32: 1e-2, torch.bfloat16: 1e-2 + 5 * 2.0 ** -8}


def _rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


def _model(d_model=256, n_layer=2, dtype=torch.float32, **kw):
    torch.manual_seed(d_model + n_layer)
    m = MambaLM(MambaConfig(d_model=d_model, n_layer=n_layer, vocab_size=1003, **kw)).cuda().eval()
    with torch.no_grad():
        for blk in m.layers:                        # small steps, as a trained model takes them
            blk.mixer.dt_proj.bias.uniform_(-4.0, -2.0)
    return m.to(dtype)


def _codes(t):
    a = t.double().abs().amax(-1, keepdim=True)
    return torch.where(a > 0, (t.double() * 127 / a).round(), 0.0), a


class _Plain(torch.nn.Module):
    """A LinearInt8 by its definition, on float rows."""

    def __init__(self, q):
        super().__init__()
        self.q = [q]
        self.register_parameter("weight", torch.nn.Parameter(q.scales.double()[:, None], requires_grad=False))
        self.register_parameter("bias", None)

    def forward(self, x):
        q = self.q[0]
        c, a = _codes(x.float())
        y = (c * a / 127) @ (q.weight[:, :q.in_features].double() * q.scales.double()[:, None]).t().contiguous()
        return (y if q.bias is None else y + q.bias.double()).to(x.dtype)


def _by_definition(q):
    m = copy.deepcopy(q)
    for blk, of in zip(m.layers, q.layers):
        blk.mixer.in_proj, blk.mixer.out_proj = _Plain(of.mixer.in_proj), _Plain(of.mixer.out_proj)
    if "head_int8" in m._modules:
        m._modules.pop("head_int8")
        m._modules["head_w4"] = _Plain(q.head_int8)
    return m


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bias", [False, True])
def test_linear_int8_module(bias, dtype):
    torch.manual_seed(0)
    lin = torch.nn.Linear(300, 200, bias=bias).cuda().to(dtype)
    q = LinearInt8.from_linear(lin)
    c, a = _codes(lin.weight.float())
    assert torch.equal(q.weight[:, :300].double(), c) and not q.weight.requires_grad
    with torch.no_grad():
        for shape in ((300,), (1, 300), (4, 5, 300), (64, 300), (3, 40, 300), (1500, 300), (0, 300)):
            x = torch.randn(shape, device="cuda").to(dtype)
            xc, xa = _codes(x.float())
            # (the sum of whole numbers first: of scaled ones, in 64 bits, a sum that is 0 comes out as 1e-16)
            p = (xc @ c.t().contiguous()) * (xa / 127) * (a / 127)[:, 0]
            ref = p + (lin.bias.double() if bias else 0)
            y = q(x)
            # the scales' rounding (two halves) and the product's (linear_int8)
            off = 5.1 * 2.0 ** -24 * p.abs() + 2.0 ** -24 * ref.abs()
            assert y.dtype == dtype and y.shape == ref.shape
            assert bool(((y.double() - ref).abs() <= off + HALF[dtype] * (ref.abs() + off)).all())
            assert torch.equal(q(ops.quantize_int8(x)), y)
            assert torch.equal(torch.cat((q.rows(x, 0, 70), q.rows(x, 70, 200)), -1), y)
        x = torch.randn(3, 300, device="cuda", dtype=dtype)
        again = copy.deepcopy(q)
        again.load_state_dict(q.state_dict())
        assert torch.equal(again(x), q(x))
        with torch.autocast("cuda", torch.float16):
            y = q(x)
        assert y.dtype == dtype and torch.equal(y, q(x))


def test_linear_int8_module_refuses_what_it_would_lose():
    q = LinearInt8.from_linear(torch.nn.Linear(64, 32).cuda())
    x = torch.randn(5, 64, device="cuda")
    with pytest.raises(RuntimeError, match="backward"):
        q(x.clone().requires_grad_())
    with pytest.raises(RuntimeError, match="transform"):
        torch.func.vmap(q)(x)
    with pytest.raises(RuntimeError):
        torch.func.jvp(q, (x,), (x,))
    with pytest.raises(RuntimeError, match="trace"):
        torch.jit.trace(q, x)
    with pytest.raises(TypeError):
        LinearInt8.from_linear(q)
    bad = torch.nn.Linear(64, 32).cuda()
    with torch.no_grad():
        bad.weight[3, 5] = float("inf")
    with pytest.raises(ValueError, match="infinities"):
        LinearInt8.from_linear(bad)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,l", [(1, 5), (3, 30), (2, 200)])
def test_prefill_and_steps_are_those_of_the_definition(b, l, dtype):
    q = _model(bias=True, dtype=dtype).quantize_int8()
    ref = _by_definition(q)
    ids = torch.randint(0, 1003, (b, l + 4), device="cuda")
    with torch.no_grad():
        got, cache = q.prefill(ids[:, :l])
        want, ref_cache = ref.prefill(ids[:, :l])
        assert got.dtype == dtype and _rel(got, want) < TOL[dtype]
        for a, r in zip(cache.layers, ref_cache.layers):
            assert _rel(a.ssm_state, r.ssm_state) < TOL[dtype] and _rel(a.conv_state, r.conv_state) < TOL[dtype]
        for i in range(l, l + 4):
            got, want = q.step(ids[:, i:i + 1], cache), ref.step(ids[:, i:i + 1], ref_cache)
            assert got.dtype == dtype and _rel(got, want) < 2 * TOL[dtype]      # (the caches differ too)


def test_it_stays_near_the_float_model():
    m = _model(d_model=512)
    ids = torch.randint(0, 1003, (2, 64), device="cuda")
    with torch.no_grad():
        want, _ = m.prefill(ids)
        got, _ = m.quantize_int8().prefill(ids)
    # a step of a row is a / 127, its values off by up to half of one, evenly: 1 / sqrt(12) of a / 127 against a
    # root mean square of a / 4 or more is 1% for each operand, 1.3% a product; five follow each other
    assert _rel(got, want) < 5 * 4 / 127 / 12 ** 0.5 * 2 ** 0.5


@pytest.mark.parametrize("rows", [1, 2, 5, 40])
def test_a_prompt_equals_its_steps(rows):
    q = _model(dtype=torch.float32).quantize_int8()
    ids = torch.randint(0, 1003, (rows, 12), device="cuda")
    with torch.no_grad():
        want, _ = q.prefill(ids)
        cache = MambaCache.allocate(q.cfg, rows, "cuda", torch.float32)
        got = torch.cat([q.step(ids[:, i:i + 1], cache) for i in range(12)], 1)
    assert _rel(got, want) < TOL[torch.float32]


@pytest.mark.parametrize("dtype", DTYPES)
def test_halves_of_in_proj_in_a_large_prompt(monkeypatch, dtype):
    q = _model(dtype=dtype, bias=True).quantize_int8()
    ids = torch.randint(0, 1003, (2, 100), device="cuda")
    with torch.no_grad():
        want, c0 = q.prefill(ids)
        monkeypatch.setattr(mm, "SPLIT_PROJ_MIN_TOKENS", 150)
        got, c1 = q.prefill(ids)
    # (the scan reads the same values through other strides)
    assert _rel(got, want) < TOL[dtype] and _rel(c1.layers[1].ssm_state, c0.layers[1].ssm_state) < TOL[dtype]
    assert torch.equal(c1.layers[0].conv_state, c0.layers[0].conv_state)


@pytest.mark.parametrize("dtype", DTYPES)
def test_captured_steps_and_prompts_replay_the_eager_ones(dtype):
    q = _model(dtype=dtype).quantize_int8()
    ids = torch.randint(0, 1003, (2, 20), device="cuda")
    cache = MambaCache.allocate(q.cfg, 2, "cuda", dtype)
    prefill = GraphedPrefill(q, cache, 2, 16, "cuda")
    prefill.capture()
    stepper = GraphedStepper(q, cache, 2, "cuda")
    stepper.capture()
    with torch.no_grad():
        for shift in range(3):
            x = ids.roll(shift, 1)
            want, c = q.prefill(x[:, :16])
            assert torch.equal(prefill.replay(x[:, :16]), want)
            for i in range(16, 20):
                want = q.step(x[:, i:i + 1], c)
                assert torch.equal(stepper.replay(x[:, i:i + 1]), want)
            torch.cuda.synchronize()


def test_graphs_of_the_old_weights_refuse_to_replay():
    m = _model()
    cache = MambaCache.allocate(m.cfg, 1, "cuda", torch.float32)
    stepper = GraphedStepper(m, cache, 1, "cuda")
    stepper.capture()
    m.quantize_int8()
    with pytest.raises(RuntimeError, match="captur"):
        stepper.replay(torch.zeros(1, 1, device="cuda", dtype=torch.long))


def test_generate_and_score():
    q = _model().quantize_int8()
    ids = torch.randint(0, 1003, (2, 9), device="cuda")
    tokens, lp = q.generate(ids, 5, return_logprobs=True, top=3)
    assert tokens.shape == (2, 14) and lp.logprob.shape == (2, 5)
    assert torch.equal(lp.top_token[..., 0], tokens[:, 9:])
    s = q.score(tokens)
    assert s.logprob.shape == (2, 13) and bool((s.logprob[:, 8:] - lp.logprob).abs().max() < 0.1)


def test_lm_head_may_stay():
    m = _model()
    q = copy.deepcopy(m).quantize_int8(lm_head=False)
    assert "head_int8" not in q._modules
    ids = torch.randint(0, 1003, (1, 9), device="cuda")
    with torch.no_grad():
        want, c = q.prefill(ids)
        got = q.step(ids[:, :1], c)
    assert want.shape == (1, 9, q.cfg.vocab_size) and got.shape == (1, 1, q.cfg.vocab_size)


def test_hooks_on_a_projection_see_its_rows():
    q = _model().quantize_int8()
    ids = torch.randint(0, 1003, (1, 9), device="cuda")
    seen = []
    with torch.no_grad():
        want, _ = q.prefill(ids)
        handle = q.layers[0].mixer.in_proj.register_forward_pre_hook(lambda mod, args: seen.append(args[0]))
        got, _ = q.prefill(ids)
        handle.remove()
    assert len(seen) == 1 and isinstance(seen[0], torch.Tensor) and seen[0].shape == (1, 9, 256)
    assert _rel(got, want) < TOL[torch.float32]


def test_a_mixer_takes_float_rows():
    q = _model().quantize_int8()
    x = torch.randn(2, 7, 256, device="cuda")
    mixer = q.layers[0].mixer
    with torch.no_grad():
        y, conv, ssm = mixer.prefill(x)
        z, conv8, ssm8 = mixer.prefill(ops.quantize_int8(x))
        assert y.shape == x.shape and torch.equal(y, z) and torch.equal(conv, conv8) and torch.equal(ssm, ssm8)
        with torch.autocast("cuda", torch.bfloat16):
            z, _, _ = mixer.prefill(x)
        assert z.dtype == torch.float32 and torch.equal(y, z)


def test_outside_no_grad_the_model_runs_as_inside():
    q = _model().quantize_int8()
    ids = torch.randint(0, 1003, (1, 9), device="cuda")
    with torch.no_grad():
        want, c = q.prefill(ids)
        step = q.step(ids[:, :1], c)
    got, c = q.prefill(ids)
    assert torch.equal(got, want) and torch.equal(q.step(ids[:, :1], c), step)


def test_quantize_int8_changes_all_or_nothing():
    m = _model()
    with torch.no_grad():
        m.layers[1].mixer.out_proj.weight[0, 0] = float("nan")
    with pytest.raises(ValueError, match="infinities"):
        m.quantize_int8()
    assert all(type(b.mixer.in_proj) is torch.nn.Linear and type(b.mixer.out_proj) is torch.nn.Linear for b in m.layers)
    assert getattr(m, "weight_set", 0) == 0
    q = _model().quantize_int8()
    with pytest.raises(TypeError, match="quantize_int8"):
        q.quantize_int8()
    with pytest.raises(TypeError, match="quantize_w4"):
        q.quantize_w4()


def test_casts_keep_the_scales():
    q = _model(dtype=torch.float32).quantize_int8()
    s = q.layers[0].mixer.in_proj.scales.detach().clone()
    ids = torch.randint(0, 1003, (1, 9), device="cuda")
    q.bfloat16()
    assert torch.equal(q.layers[0].mixer.in_proj.scales, s)
    with torch.no_grad():
        got, _ = q.prefill(ids)
    assert got.dtype == torch.bfloat16 and bool(got.isfinite().all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 2, 5, 32])
def test_steps_in_one_call_are_those_op_by_op(rows, dtype, monkeypatch):
    q = _model(d_model=512, n_layer=3, dtype=dtype, bias=True).quantize_int8()
    ids = torch.randint(0, 1003, (rows, 12), device="cuda")
    calls = []
    real = ops.decode_step_int8
    monkeypatch.setattr(ops, "decode_step_int8", lambda *a, **k: (calls.append(1), real(*a, **k))[1])
    with torch.no_grad():
        _, cache = q.prefill(ids[:, :8])
        other = copy.deepcopy(cache)
        got = [q.step(ids[:, i:i + 1], cache) for i in range(8, 12)]
        assert len(calls) == 4
        monkeypatch.setattr(mm, "BATCHED_STEP_NATIVE", False)
        want = [q.step(ids[:, i:i + 1], other) for i in range(8, 12)]
        assert len(calls) == 4
    # float32: the same launches with the same arguments, but for the SSM update's parameters (the same values) and the sums
    # of the residual; bfloat16: op by op rounds each out_proj's output once more
    for a, r in zip(got, want):
        assert a.dtype == dtype and a.shape == r.shape
        assert _rel(a, r) < TOL[dtype]
    if dtype == torch.float32:
        assert all(torch.equal(a, r) for a, r in zip(got, want))
        for a, r in zip(cache.layers, other.layers):
            assert torch.equal(a.ssm_state, r.ssm_state) and torch.equal(a.conv_state, r.conv_state)


def test_the_one_call_step_leaves_other_stacks_alone():
    q = _model(d_model=512).quantize_int8()
    cache = MambaCache.allocate(q.cfg, 2, "cuda", torch.float32)
    x = torch.zeros(2, 512, device="cuda")
    took = lambda: q._quant_step_layers(x, cache, q._layer_tensors(), LinearInt8) is not None
    assert took()
    handle = q.layers[0].mixer.out_proj.register_forward_hook(lambda *a: None)
    assert not took()
    handle.remove()
    assert took()
    big = MambaCache.allocate(q.cfg, 33, "cuda", torch.float32)
    assert q._quant_step_layers(torch.zeros(33, 512, device="cuda"), big, q._layer_tensors(), LinearInt8) is None
    ids = torch.zeros(2, 1, device="cuda", dtype=torch.long)
    with torch.no_grad():
        before = q.step(ids, copy.deepcopy(cache))
        # another projection in its place, of other sizes' addresses: the plan follows
        lin = torch.nn.Linear(512, 2048, bias=False).cuda()
        q.layers[0].mixer.in_proj = LinearInt8.from_linear(lin)
        after = q.step(ids, copy.deepcopy(cache))
        assert not torch.equal(before, after)
        q.layers[0].mixer.in_proj = lin                      # (a plain one: op by op)
        assert not took() and q.step(ids, copy.deepcopy(cache)).shape == before.shape


@pytest.mark.parametrize("b,l", [(1, 1), (1, 64), (2, 65), (3, 130)])
def test_prompts_in_one_call_are_those_op_by_op(b, l, monkeypatch):
    q = _model(d_model=256, n_layer=3, bias=True).quantize_int8()
    ids = torch.randint(0, 1003, (b, 2 * l), device="cuda")
    calls = []
    real = ops.prefill_long
    monkeypatch.setattr(ops, "prefill_long", lambda *a, **k: (calls.append(k["matrices"]), real(*a, **k))[1])
    with torch.no_grad():
        got, cache = q.prefill(ids[:, :l])
        got2, _ = q.prefill(ids[:, l:], cache, out_cache=cache)          # the next part of the prompt, in place
        assert len(calls) == 2 and all(m is not None for m in calls)
        monkeypatch.setattr(mm, "LONG_PREFILL_NATIVE", False)
        want, other = q.prefill(ids[:, :l])
        want2, other = q.prefill(ids[:, l:], other)
        assert len(calls) == 2
    # (x_proj's and dt_proj's library products differ in the order of their sums)
    assert _rel(got, want) < TOL[torch.float32] and _rel(got2, want2) < TOL[torch.float32]
    for a, r in zip(cache.layers, other.layers):
        assert _rel(a.ssm_state, r.ssm_state) < TOL[torch.float32] and _rel(a.conv_state, r.conv_state) < TOL[torch.float32]


def test_the_one_call_prompt_follows_its_weights():
    q = _model().quantize_int8()
    ids = torch.randint(0, 1003, (1, 30), device="cuda")
    with torch.no_grad():
        before, _ = q.prefill(ids)
        q.layers[1].mixer.out_proj = LinearInt8.from_linear(torch.nn.Linear(512, 256, bias=False).cuda())
        after, _ = q.prefill(ids)
        assert not torch.equal(before, after)
        seen = []
        handle = q.layers[0].mixer.out_proj.register_forward_hook(lambda m, a, o: seen.append(o))
        q.prefill(ids)
        handle.remove()
        assert len(seen) == 1 and seen[0].shape == (1, 30, 256)
        q.layers[0].mixer.in_proj = torch.nn.Linear(256, 1024, bias=False).cuda()       # a mixed stack: op by op
        assert q.prefill(ids)[0].shape == before.shape and q.step(ids[:, :1], q.prefill(ids)[1]).shape[0] == 1


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kw", [dict(d_model=4352, expand=1, dt_rank=16), dict(d_model=4096), dict(d_model=4480, dt_rank=32),
                                dict(d_model=96, expand=3)])
def test_a_step_of_one_row_in_every_mix_of_launches(kw, dtype, monkeypatch):
    # (rows past mtl_row_linear_int8's widths before in_proj, none, and before both)
    if dtype == torch.bfloat16 and kw["d_model"] == 96:
        kw = dict(kw, expand=4)                              # (channels in 64s)
    q = _model(n_layer=3, dtype=dtype, **kw).quantize_int8()
    ids = torch.randint(0, 1003, (1, 8), device="cuda")
    calls = []
    real = ops.decode_step_int8
    monkeypatch.setattr(ops, "decode_step_int8", lambda *a, **k: (calls.append(1), real(*a, **k))[1])
    with torch.no_grad():
        _, cache = q.prefill(ids[:, :4])
        other = copy.deepcopy(cache)
        got = [q.step(ids[:, i:i + 1], cache) for i in range(4, 8)]
        # (in bf16 the one call takes dt_rank + 2 d_state in fours)
        assert len(calls) == (0 if dtype == torch.bfloat16 and (q.cfg.dt_rank + 2 * q.cfg.d_state) % 4 else 4)
        monkeypatch.setattr(mm, "BATCHED_STEP_NATIVE", False)
        want = [q.step(ids[:, i:i + 1], other) for i in range(4, 8)]
    for a, r in zip(got, want):
        assert torch.equal(a, r) if dtype == torch.float32 else _rel(a, r) < TOL[dtype]


@pytest.mark.parametrize("kind", [torch.float16, torch.float64])
def test_a_mixers_output_of_another_float_type_is_added(kind):
    q = _model(n_layer=3).quantize_int8()
    ids = torch.randint(0, 1003, (2, 9), device="cuda")

    def run(hook):
        handle = q.layers[0].mixer.out_proj.register_forward_hook(hook)
        logits, cache = q.prefill(ids)
        step = q.step(ids[:, :1], cache)
        handle.remove()
        return logits, step

    with torch.no_grad():
        # (the value is converted to float32 where the float norm converts it)
        want = run(lambda m, a, o: o.to(kind).float())
        got = run(lambda m, a, o: o.to(kind))
    assert all(torch.equal(u, v) for u, v in zip(got, want))


def _row_rel(a, b):
    """The largest relative distance of a row (equal rows, of zeros too: 0)."""
    a, b = (t.double().reshape(-1, t.shape[-1]) for t in (a, b))
    off = (a - b).norm(dim=-1)
    return float(torch.where(off == 0, 0.0, off / b.norm(dim=-1)).max())


# As TOL, which counts one value of each row and product on the other side of a border, for seven products (three layers and a
# head): 7 * 4 / 127 / 16 = 1.4e-2, and as much again for what earlier tokens' states bring.
ROW_TOL = 2 * 7 * 4 / 127 / 16


@pytest.mark.parametrize("b,l", [(1, 1), (1, 64), (2, 65), (3, 130), (1, 700)])
def test_prompts_in_one_call_are_those_op_by_op_row_by_row(b, l, monkeypatch):
    q = _model(d_model=256, n_layer=3, bias=True).quantize_int8()
    ids = torch.randint(0, 1003, (b, 2 * l), device="cuda")
    calls = []
    real = ops.prefill_long
    monkeypatch.setattr(ops, "prefill_long", lambda *a, **k: (calls.append(k["matrices"]), real(*a, **k))[1])
    runs = []
    with torch.no_grad():
        for native in (True, False):
            monkeypatch.setattr(mm, "LONG_PREFILL_NATIVE", native)
            first, cache = q.prefill(ids[:, :l])
            kept = copy.deepcopy(cache)
            second, cache = q.prefill(ids[:, l:], cache)
            runs.append((first, second, kept, cache))
    assert len(calls) == 2 and all(m is not None for m in calls)
    (a0, a1, ka, ca), (r0, r1, kr, cr) = runs
    assert _row_rel(a0, r0) < ROW_TOL and _row_rel(a1, r1) < ROW_TOL
    for mine, theirs in ((ka, kr), (ca, cr)):
        # the first layer's history is what the norm and in_proj give: no library product before it
        assert torch.equal(mine.layers[0].conv_state, theirs.layers[0].conv_state)
        for u, v in zip(mine.layers, theirs.layers):
            # (rows of a state: all channels of a place)
            assert _row_rel(u.conv_state.transpose(1, 2), v.conv_state.transpose(1, 2)) < ROW_TOL
            assert _row_rel(u.ssm_state.transpose(1, 2), v.ssm_state.transpose(1, 2)) < ROW_TOL


def _by_definition_of(q):
    """_by_definition() of a stack in which some projections are plain."""
    m = copy.deepcopy(q)
    for blk, of in zip(m.layers, q.layers):
        for name in ("in_proj", "out_proj"):
            p = getattr(of.mixer, name)
            if type(p) is LinearInt8:
                setattr(blk.mixer, name, _Plain(p))
    if "head_int8" in m._modules:
        m._modules.pop("head_int8")
        m._modules["head_w4"] = _Plain(q.head_int8)
    return m


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,l", [(1, 9), (2, 70)])
@pytest.mark.parametrize("which", ["no head", "plain in_proj first", "plain in_proj last", "plain out_proj first"])
def test_stacks_of_both_kinds_are_those_of_the_definition(which, b, l, dtype):
    m = _model(n_layer=3, dtype=dtype)
    q = copy.deepcopy(m).quantize_int8(lm_head=which != "no head")
    if which != "no head":
        i, name = (2 if "last" in which else 0), "out_proj" if "out" in which else "in_proj"
        setattr(q.layers[i].mixer, name, getattr(m.layers[i].mixer, name))
    ref = _by_definition_of(q)
    ids = torch.randint(0, 1003, (b, l + 3), device="cuda")
    # as ROW_TOL, with seven roundings of each value to bf16
    tol = ROW_TOL + (7 * 2.0 ** -8 if dtype == torch.bfloat16 else 0.0)
    with torch.no_grad():
        got, cache = q.prefill(ids[:, :l])
        want, ref_cache = ref.prefill(ids[:, :l])
        assert got.dtype == dtype and _row_rel(got, want) < tol
        for i in range(l, l + 3):
            got, want = q.step(ids[:, i:i + 1], cache), ref.step(ids[:, i:i + 1], ref_cache)
            assert got.dtype == dtype and got.shape == (b, 1, q.cfg.vocab_size) and _row_rel(got, want) < 2 * tol


@pytest.mark.parametrize("dtype", DTYPES)
def test_what_a_model_records_outside_no_grad(dtype):
    m = _model(dtype=dtype)
    ids = torch.randint(0, 1003, (1, 9), device="cuda")
    for lm_head in (True, False):
        q = copy.deepcopy(m).quantize_int8(lm_head=lm_head)
        logits, cache = q.prefill(ids)
        # the layers nothing; an lm_head that stays its own product, as in an unquantized model
        assert logits.requires_grad == (not lm_head)
        if not lm_head:
            logits.float().sum().backward()
            assert q.embedding.weight.grad is not None
        assert all(p.grad is None for name, p in q.named_parameters() if name != "embedding.weight")
        assert not any(t.requires_grad for c in cache.layers for t in (c.conv_state, c.ssm_state))
