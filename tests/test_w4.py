"""4-bit weights on the host: the layout word by word, the choice of codes, and what the entry points refuse."""
import copy
import ctypes

import pytest
import torch

from mamba_lite import _lib, ops


def _random(n, k, group, zeros, seed=0):
    g = torch.Generator().manual_seed(seed)
    ng = -(-k // group)
    return (torch.randint(0, 16, (n, k), generator=g, dtype=torch.uint8), torch.rand(n, ng, generator=g) + 0.5,
            torch.randint(0, 16, (n, ng), generator=g, dtype=torch.uint8) if zeros else None)


@pytest.mark.parametrize("n,k,group,zeros", [(1, 1, 32, True), (16, 128, 128, False), (17, 129, 64, True),
                                             (40, 300, 32, True), (33, 256, 128, True)])
def test_layout_is_the_documented_one(n, k, group, zeros):
    codes, scales, z = _random(n, k, group, zeros)
    w4 = ops.pack_w4(codes, scales, z, group)
    nt, kb = -(-n // 16), -(-k // 128)
    assert tuple(w4.codes.shape) == (nt, kb, 64, 16)
    words = w4.codes.view(torch.int32)                      # [nt, kb, 64, 4]
    for t in range(nt):
        for b in range(kb):
            for l in range(64):
                r, j = l % 16, l // 16
                for i in range(4):
                    for e in range(8):
                        row, col = 16 * t + r, 128 * b + 32 * i + 8 * j + e
                        got = (int(words[t, b, l, i]) >> (16 * (e & 1) + 4 * (e // 2))) & 15
                        inside = row < n and col < k
                        assert got == (int(codes[row, col]) if inside else 0)
                        s = float(w4.scales[t, b, r, (col % 128) // group])
                        # past N or in a group past K: scale 0; columns past K in K's last group carry code 0
                        assert s == (float(scales[row, col // group]) if row < n and col // group < scales.shape[1]
                                     else 0.0)
                        if zeros and inside:
                            assert int(w4.zeros[t, b, r, (col % 128) // group]) == int(z[row, col // group])


@pytest.mark.parametrize("scale_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("zero_points", [False, True])
@pytest.mark.parametrize("n,k,group", [(5, 64, 32), (3, 200, 128), (20, 77, 64)])
def test_quantize_rounds_to_the_nearest_value(n, k, group, zero_points, scale_dtype):
    g = torch.Generator().manual_seed(1)
    W = torch.randn(n, k, generator=g) + (0.7 if zero_points else 0.0)
    W[0, :group] = 0.0                                       # a group of zeros
    W[1, 0] = 9.0                                            # an outlier
    w4 = ops.quantize_w4(W, group, zero_points, scale_dtype)
    assert w4.scales.dtype == scale_dtype and (w4.zeros is not None) == zero_points
    per = 128 // group
    scales = w4.scales.transpose(1, 2).reshape(-1, w4.codes.shape[1] * per)[:n].double()
    words = w4.codes.view(torch.int32).view(w4.codes.shape[0], w4.codes.shape[1], 4, 16, 4)
    codes = torch.stack([(words >> (16 * (e & 1) + 4 * (e // 2))) & 15 for e in range(8)], -1)   # [nt,kb,j,r,i,e]
    codes = codes.permute(0, 3, 1, 4, 2, 5).reshape(w4.codes.shape[0] * 16, -1)[:n, :k].double()
    col = torch.arange(k) // group
    z = 8.0 if w4.zeros is None else \
        w4.zeros.transpose(1, 2).reshape(-1, w4.codes.shape[1] * per)[:n].double()[:, col]
    s = scales[:, col]
    back = (codes - z) * s
    # half a step, and what rounding a scale down (bf16: by 2^-8) cuts off the end of the range, at most 15 steps; with
    # zero points the zero's own rounding may cut off another half step
    step = s * (0.5 + (0.5 if zero_points else 0.0) + 15 * (2.0 ** -8 if scale_dtype == torch.bfloat16 else 2.0 ** -23))
    assert bool(((back - W.double()).abs() <= step + 1e-12).all())
    assert bool((back[0, :group] == 0).all())


@pytest.mark.parametrize("change,error", [
    (dict(codes=torch.zeros(4, 8)), "uint8"),
    (dict(codes=torch.zeros(4, 8, 1, dtype=torch.uint8)), "uint8"),
    (dict(codes=torch.full((4, 64), 16, dtype=torch.uint8)), "0..15"),
    (dict(zeros=torch.full((4, 1), 16, dtype=torch.uint8)), "0..15"),
    (dict(zeros=torch.zeros(4, 2, dtype=torch.uint8)), "zeros"),
    (dict(scales=torch.ones(4, 2)), "scales"),
    (dict(scales=torch.ones(4, 1, dtype=torch.float16)), "scales"),
    (dict(group=48), "group"),
    (dict(codes=torch.zeros(0, 64, dtype=torch.uint8)), "rows"),
])
def test_pack_refuses(change, error):
    a = dict(codes=torch.zeros(4, 64, dtype=torch.uint8), scales=torch.ones(4, 1), zeros=None, group=64)
    a.update(change)
    with pytest.raises(ValueError, match=error):
        ops.pack_w4(**a)


@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_pack_refuses_scales_that_are_not_finite(bad, dtype):
    scales = torch.ones(4, 2, dtype=dtype)
    scales[3, 1] = bad
    with pytest.raises(ValueError, match="infinities or NaN"):
        ops.pack_w4(torch.zeros(4, 128, dtype=torch.uint8), scales)
    # a finite matrix whose float32 form is not
    if dtype == torch.float32 and bad > 0:
        with pytest.raises(ValueError, match="infinities or NaN"):
            ops.quantize_w4(torch.full((2, 64), 1e300, dtype=torch.float64))


def test_quantize_refuses():
    for bad in (torch.zeros(3), torch.zeros(3, 4, dtype=torch.int32), torch.zeros(0, 4),
                torch.tensor([[1.0, float("inf")]]), torch.tensor([[float("nan"), 1.0]])):
        with pytest.raises(ValueError):
            ops.quantize_w4(bad)
    with pytest.raises(ValueError, match="group"):
        ops.quantize_w4(torch.zeros(2, 64), group=16)
    with pytest.raises(TypeError, match="scale_dtype"):
        ops.quantize_w4(torch.zeros(2, 64), scale_dtype=torch.float16)


def test_a_made_up_layout_is_refused():
    w = ops.pack_w4(*_random(20, 200, 64, True), group=64)
    ops.W4(w.codes, w.scales, w.zeros, 20, 200, 64)
    for a in ((w.codes[:1], w.scales, w.zeros, 20, 200, 64), (w.codes, w.scales[:1], w.zeros, 20, 200, 64),
              (w.codes, w.scales, w.zeros[:1], 20, 200, 64), (w.codes, w.scales, w.zeros, 40, 200, 64),
              (w.codes, w.scales, w.zeros, 20, 300, 64), (w.codes, w.scales, w.zeros, 20, 200, 32),
              (w.codes, w.scales, w.zeros, 0, 200, 64), (w.codes, w.scales.half(), None, 20, 200, 64)):
        with pytest.raises(ValueError):
            ops.W4(*a)


def test_a_matrix_is_fixed_and_can_be_copied():
    w = ops.pack_w4(*_random(20, 200, 64, True), group=64)
    with pytest.raises(AttributeError):
        w.zeros = None
    c = copy.deepcopy(w)
    assert c.codes is not w.codes and torch.equal(c.codes, w.codes) and torch.equal(c.scales, w.scales) and c.n == 20


def test_calls_are_refused_on_the_host():
    w4 = ops.pack_w4(*_random(20, 200, 64, True), group=64)
    x = torch.zeros(2, 200)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.linear_w4(x, w4)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.dequantize_w4(w4)
    for bad in (dict(x=torch.zeros(2, 199)), dict(x=torch.zeros(65, 200)), dict(bias=torch.zeros(19)),
                dict(out=torch.zeros(2, 19)), dict(out=torch.zeros(2, 40)[:, ::2])):
        with pytest.raises(ValueError):
            ops.linear_w4(**{**dict(x=x, w4=w4), **bad})
    shared = torch.zeros(4000)
    with pytest.raises(ValueError, match="overlap"):
        ops.linear_w4(shared[:400].view(2, 200), w4, out=shared[390:430].view(2, 20))
    with pytest.raises(TypeError, match="W4"):
        ops.linear_w4(x, torch.zeros(20, 200))
    with pytest.raises(TypeError):
        ops.linear_w4(x.half(), w4)
    with pytest.raises(TypeError):
        ops.linear_w4(x, w4, bias=torch.zeros(20, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="backward"):
        ops.linear_w4(torch.zeros(2, 200, requires_grad=True), w4)
    with pytest.raises(TypeError):
        ops.dequantize_w4(w4, torch.float16)
    with pytest.raises(ValueError):
        ops.dequantize_w4(w4, out=torch.zeros(20, 199))


def _args(**change):
    buf = 0x1000
    a = dict(x=buf, codes=buf, scales=buf, zeros=None, bias=None, y=buf, ldx=200, ldy=20, M=2, N=20, K=200, group=64,
             dtype=0, scale_dtype=0, y_f32=0)
    a.update(change)
    return _lib.LinearW4Args(**a)


@pytest.mark.parametrize("change,error", [
    (dict(group=16), b"group"), (dict(M=65), b"M must"), (dict(M=-1), b"M must"), (dict(N=0), b"N must"),
    (dict(K=0), b"K in"), (dict(K=(1 << 20) + 1), b"K in"), (dict(dtype=2), b"dtype"), (dict(scale_dtype=2), b"dtype"),
    (dict(x=None), b"null"), (dict(codes=None), b"null"), (dict(y=None), b"null"), (dict(codes=0x1004), b"aligned"),
    (dict(scales=0x1008), b"aligned"), (dict(zeros=0x1001), b"aligned"), (dict(ldx=199), b"overlap"),
    (dict(ldy=19), b"overlap"),
])
def test_the_library_refuses(change, error):
    lib = _lib.load()
    assert lib.mtl_linear_w4(ctypes.byref(_args(**change)), None) == 1
    assert error in lib.mtl_last_error()


def test_the_library_refuses_a_matrix():
    lib = _lib.load()
    p = 0x1000
    assert lib.mtl_linear_w4(None, None) == 1
    assert lib.mtl_linear_w4(ctypes.byref(_args(M=0)), None) == 0            # nothing to do, nothing launched
    for bad in ((p, p, None, None, 200, 20, 200, 64, 0, 0), (p, p, None, p, 199, 20, 200, 64, 0, 0),
                (p, p, p + 1, p, 200, 20, 200, 64, 0, 0), (p, p, None, p, 200, 20, 200, 65, 0, 0),
                (p, p, None, p, 200, 0, 200, 64, 0, 0)):
        assert lib.mtl_dequantize_w4(*bad, None) == 1


def _step_args(**change):
    p = 0x1000
    a = _lib.DecodeStepBatchedArgs()
    for n in ("h", "norm_f", "inp", "xc", "z", "y", "xpart", "x_dbl", "parts", "normed_out"):
        setattr(a, n, p)
    a.h, a.normed_out, a.n_layers, a.batch = 0x2000, 0x3000, 1, 2
    a.d_model, a.d_inner, a.d_state, a.dt_rank, a.d_conv = 256, 512, 16, 16, 4
    L = (_lib.DecodeLayer * 1)()
    for n in ("norm_w", "conv_w", "W_xT", "W_x", "W_dt", "dt_bias", "A_log", "conv_state", "ssm_state"):
        setattr(L[0], n, p)
    m = (_lib.W4Matrix * 2)()
    for x in m:
        x.codes, x.scales, x.group = p, p, 64
    dtype = change.pop("dtype", 0)
    for n, v in change.items():
        if n.startswith("L_"):
            setattr(L[0], n[2:], v)
        elif n.startswith("m_"):
            setattr(m[1], n[2:], v)
        else:
            setattr(a, n, v)
    return ctypes.byref(a), L, m, dtype, None


@pytest.mark.parametrize("change,error", [
    (dict(batch=33), b"batch"), (dict(batch=0), b"batch"), (dict(n_layers=0), b"n_layers"), (dict(d_model=0), b"d_model"),
    (dict(d_state=17), b"d_state"), (dict(dt_rank=257), b"dt_rank"), (dict(d_conv=5), b"d_conv"), (dict(fold=1), b"folded"),
    (dict(dtype=2), b"dtype"), (dict(dtype=1, d_inner=200), b"multiple of 64"), (dict(dtype=1, dt_rank=17), b"of 4"),
    (dict(parts=None), b"null"), (dict(h=0x1000), b"alias"), (dict(L_W_xT=None), b"null"), (dict(L_ssm_state=None), b"null"),
    (dict(dtype=1, L_W_x=0x1008), b"aligned"), (dict(m_codes=None), b"codes"), (dict(m_scales=0x1008), b"aligned"),
    (dict(m_group=48), b"group"), (dict(m_scale_dtype=2), b"scale_dtype"), (dict(xc=0x1004), b"aligned"),
])
def test_the_library_refuses_a_step(change, error):
    lib = _lib.load()
    assert lib.mtl_decode_step_w4(*_step_args(**change)) == 1
    assert error in lib.mtl_last_error()


def test_struct_layouts_match_the_header():
    # six pointers, five int64, four int32; six pointers, five int64, two int32; three pointers, two int32
    assert ctypes.sizeof(_lib.LinearW4Args) == 6 * 8 + 5 * 8 + 4 * 4 and _lib.LinearW4Args.group.offset == 88
    assert ctypes.sizeof(_lib.TokenLogprobsArgs) == 6 * 8 + 5 * 8 + 2 * 4 and _lib.TokenLogprobsArgs.top.offset == 88
    assert ctypes.sizeof(_lib.W4Matrix) == 3 * 8 + 2 * 4


def test_a_weight_that_cannot_be_quantized_leaves_the_model_alone():
    from mamba_lite.model import LinearW4, MambaConfig, MambaLM
    m = MambaLM(MambaConfig(d_model=64, n_layer=2, vocab_size=40))
    with torch.no_grad():
        m.layers[1].mixer.out_proj.weight[3, 5] = float("nan")
    with pytest.raises(ValueError, match="NaN"):
        m.quantize_w4()
    assert all(type(getattr(b.mixer, n)) is torch.nn.Linear for b in m.layers for n in ("in_proj", "out_proj"))
    with torch.no_grad():
        m.layers[1].mixer.out_proj.weight[3, 5] = 0.0
    keys = set(m.state_dict())
    assert all(type(getattr(b.mixer, n)) is LinearW4 for b in m.quantize_w4().layers for n in ("in_proj", "out_proj"))
    new = set(m.state_dict()) - keys
    assert new == {f"layers.{i}.mixer.{n}.scales" for i in range(2) for n in ("in_proj", "out_proj")} | \
        {"head_w4.weight", "head_w4.scales"}


@pytest.mark.parametrize("n,k,group,zeros", [(1, 1, 32, True), (40, 300, 32, True), (33, 256, 128, False), (17, 129, 64, True)])
def test_the_matrix_as_torch_operations(n, k, group, zeros):
    codes, scales, z = _random(n, k, group, zeros)
    col = torch.arange(k) // group
    w = (codes.double() - (z.double()[:, col] if zeros else 8.0)) * scales.double()[:, col]
    w4 = ops.pack_w4(codes, scales, z, group)
    assert torch.equal(ops.w4_matrix(w4), w.float()) and torch.equal(ops.w4_matrix(w4, torch.bfloat16), w.float().bfloat16())


def test_forward_mode_and_tracing_are_refused():
    """A raw launch would come back without its tangent, or with a trace of memory that nothing fills."""
    w4 = ops.pack_w4(*_random(20, 200, 64, True), group=64)
    x, tokens = torch.zeros(2, 200), torch.zeros(2, dtype=torch.int64)
    with torch.autograd.forward_ad.dual_level(), torch.no_grad():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(RuntimeError, match="forward-mode"):
            ops.linear_w4(dual, w4)
        with pytest.raises(RuntimeError, match="forward-mode"):
            ops.linear_w4(x, w4, torch.autograd.forward_ad.make_dual(torch.zeros(20), torch.ones(20)))
        with pytest.raises(RuntimeError, match="forward-mode"):
            ops.token_logprobs(dual, tokens)
        with pytest.raises(RuntimeError, match="GPU"):             # a primal by itself is an ordinary operand
            ops.linear_w4(x, w4)
    for call in (lambda x: ops.linear_w4(x, w4), lambda x: ops.token_logprobs(x, tokens).logprob,
                 lambda x: x @ ops.dequantize_w4(w4).t()):
        with pytest.raises(RuntimeError, match="trace"):
            torch.jit.trace(call, (x,), check_trace=False)


@pytest.mark.parametrize("lm_head", [False, True])
def test_codes_are_not_sharded(lm_head):
    from mamba_lite import tp_utils
    from mamba_lite.model import MambaConfig, MambaLM
    from mamba_lite.tp_model import LocalTPLM
    m = MambaLM(MambaConfig(d_model=64, n_layer=1, vocab_size=40))
    LocalTPLM.from_dense(m)
    m.quantize_w4(lm_head=lm_head)
    with pytest.raises(TypeError, match="quantize_w4"):
        LocalTPLM.from_dense(m)
    for shard in (tp_utils.shard_mixer_params, tp_utils.naive_shard_mixer_params):
        with pytest.raises(TypeError, match="quantize_w4"):
            shard(m.layers[0].mixer, 0, 2)
