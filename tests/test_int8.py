"""Rows in 8-bit integers on the host: the layout, and what the entry points refuse."""
import copy
import ctypes
import pickle

import pytest
import torch

from mamba_lite import _lib, ops


def _q(*lead, k=40, dtype=torch.float32):
    g = torch.Generator().manual_seed(0)
    return ops.pack_int8(torch.randint(-127, 128, (*lead, k), generator=g, dtype=torch.int8),
                         torch.rand(lead, generator=g) + 0.5, dtype)


@pytest.mark.parametrize("lead,k", [((), 1), ((1,), 128), ((3,), 129), ((2, 5), 40), ((0,), 7), ((4,), 777)])
def test_layout_is_the_documented_one(lead, k):
    g = torch.Generator().manual_seed(1)
    codes = torch.randint(-128, 128, (*lead, k), generator=g, dtype=torch.int8)
    scales = torch.rand(lead, generator=g)
    q = ops.pack_int8(codes, scales, torch.bfloat16)
    kp = -(-k // 128) * 128
    assert tuple(q.codes.shape) == (*lead, kp) and q.codes.is_contiguous()
    assert torch.equal(q.codes[..., :k], codes) and not bool(q.codes[..., k:].any())
    assert torch.equal(q.scales, scales) and q.scales.data_ptr() != scales.data_ptr() or scales.numel() == 0
    assert tuple(q.shape) == (*lead, k) and q.dtype == torch.bfloat16 and q.k == k


def test_pack_takes_strided_operands():
    codes = torch.arange(60, dtype=torch.int8).view(6, 10)
    scales = torch.arange(12, dtype=torch.float32)
    q = ops.pack_int8(codes[::2, 1::3], scales[::4])
    assert torch.equal(q.codes[:, :3], codes[::2, 1::3]) and torch.equal(q.scales, scales[::4])


def test_rows_share_memory_and_parts_are_fixed():
    q = _q(6)
    r = q.rows(2, 5)
    assert tuple(r.shape) == (3, 40) and r.codes.data_ptr() == q.codes[2:].data_ptr()
    for name in ("codes", "scales", "k", "dtype"):
        with pytest.raises(AttributeError, match="fixed"):
            setattr(q, name, getattr(q, name))
    for c in (copy.deepcopy(q), pickle.loads(pickle.dumps(q))):
        assert torch.equal(c.codes, q.codes) and torch.equal(c.scales, q.scales) and c.k == q.k and c.dtype == q.dtype


@pytest.mark.parametrize("change,error", [
    (dict(codes=torch.zeros(4, 40)), "int8"),
    (dict(codes=torch.zeros(4, 40, dtype=torch.uint8)), "int8"),
    (dict(codes=torch.zeros((), dtype=torch.int8), scales=torch.ones(())), "int8"),
    (dict(codes=torch.zeros(4, 0, dtype=torch.int8)), "columns"),
    (dict(codes=torch.zeros(1, 1 << 17, dtype=torch.int8), scales=torch.ones(1)), "columns"),
    (dict(scales=torch.ones(5)), "scales"),
    (dict(scales=torch.ones(4, 1)), "scales"),
    (dict(scales=torch.ones(4, dtype=torch.bfloat16)), "scales"),
    (dict(scales=torch.tensor([1.0, float("inf"), 1.0, 1.0])), "infinities"),
    (dict(scales=torch.tensor([1.0, float("nan"), 1.0, 1.0])), "infinities"),
])
def test_pack_refuses(change, error):
    a = dict(codes=torch.zeros(4, 40, dtype=torch.int8), scales=torch.ones(4))
    a.update(change)
    with pytest.raises(ValueError, match=error):
        ops.pack_int8(**a)


def test_a_made_up_layout_is_refused():
    q = _q(6)
    ops.Int8(q.codes, q.scales, 128)
    for a in ((q.codes[:5], q.scales, 40), (q.codes, q.scales[:5], 40), (q.codes, q.scales, 129), (q.codes, q.scales, 0),
              (q.codes.float(), q.scales, 40), (q.codes, q.scales.double(), 40), (q.codes.t(), q.scales, 40),
              (q.codes[:, :40], q.scales, 40), (torch.zeros(6 * 128 + 1, dtype=torch.int8)[1:].view(6, 128), q.scales, 40)):
        with pytest.raises(ValueError):
            ops.Int8(*a)
    with pytest.raises(TypeError, match="dtype"):
        ops.Int8(q.codes, q.scales, 40, torch.float16)


def test_kernels_need_gpu_tensors():
    x = torch.zeros(3, 40)
    for call in (lambda: ops.quantize_int8(x), lambda: ops.add_rmsnorm_int8(x, torch.ones(40), 1e-5),
                 lambda: ops.linear_int8(_q(3), _q(6)), lambda: ops.dequantize_int8(_q(3))):
        with pytest.raises(RuntimeError, match="GPU tensors"):
            call()


class _Sub(torch.Tensor):
    pass


def test_quantize_refuses():
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        ops.quantize_int8(torch.zeros(3, 4, dtype=torch.float16))
    for bad in (torch.zeros(()), torch.zeros(3, 0), torch.zeros(1, 1 << 17)):
        with pytest.raises(ValueError, match="x must be"):
            ops.quantize_int8(bad)
    with pytest.raises(RuntimeError, match="backward"):
        ops.quantize_int8(torch.zeros(3, 4, requires_grad=True))
    with pytest.raises(TypeError, match="plain"):
        ops.quantize_int8(torch.zeros(3, 4).as_subclass(_Sub))


@pytest.mark.parametrize("change,error", [
    (dict(x=torch.zeros(3, 8, dtype=torch.bfloat16)), "x must be"),
    (dict(x=torch.zeros(8, 3).t()), "x must be"),
    (dict(x=torch.zeros(3, 0), weight=torch.zeros(0)), "x must be"),
    (dict(weight=torch.ones(7)), "weight"),
    (dict(weight=torch.ones(8, dtype=torch.float16)), "weight"),
    (dict(weight=torch.ones(16)[::2]), "weight"),
    (dict(y=torch.zeros(3, 7)), "y must be"),
    (dict(y=torch.zeros(3, 8, dtype=torch.float16)), "y must be"),
    (dict(y=torch.zeros(8, 3).t()), "y must be"),
    (dict(x_out=torch.zeros(3, 8, dtype=torch.bfloat16)), "x_out"),
    (dict(x_out=torch.zeros(2, 8)), "x_out"),
])
def test_norm_refuses(change, error):
    a = dict(x=torch.zeros(3, 8), weight=torch.ones(8), eps=1e-5)
    a.update(change)
    with pytest.raises(ValueError, match=error):
        ops.add_rmsnorm_int8(**a)


def test_norm_refuses_outputs_over_operands_and_gradients():
    room = torch.zeros(64)
    x = room[:24].view(3, 8)
    with pytest.raises(ValueError, match="overlap"):
        ops.add_rmsnorm_int8(x, torch.ones(8), 1e-5, x_out=room[8:32].view(3, 8))
    with pytest.raises(ValueError, match="overlap"):
        ops.add_rmsnorm_int8(x, room[40:48], 1e-5, x_out=room[40:].view(3, 8))
    yb = torch.zeros(48, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="overlap"):
        ops.add_rmsnorm_int8(x, torch.ones(8), 1e-5, y=yb[:24].view(3, 8), x_out=yb.view(torch.float32).view(3, 8))
    with pytest.raises(TypeError, match="dtype"):
        ops.add_rmsnorm_int8(x, torch.ones(8), 1e-5, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="backward"):
        ops.add_rmsnorm_int8(x, torch.ones(8, requires_grad=True), 1e-5)


def test_linear_and_dequantize_refuse():
    x, w = _q(3), _q(6)
    for a, kind, error in (
            (([1.0], w), TypeError, "x must be an Int8"), ((x, torch.zeros(6, 40)), TypeError, "w must be"),
            ((torch.zeros(3, 40).half(), w), TypeError, "float32 or bfloat16"),
            ((torch.zeros(1, 40).half(), w), TypeError, "float32 or bfloat16"),
            ((torch.zeros(1, 40, requires_grad=True), w), RuntimeError, "backward"),
            ((torch.zeros(1, 40), w, torch.zeros(6, dtype=torch.bfloat16)), TypeError, "bias"),
            ((torch.zeros(1, 40), w, None, torch.zeros(6)), ValueError, "out"),
            ((torch.zeros(1, 40), w), RuntimeError, "GPU"), ((torch.zeros(3, 40), w), RuntimeError, "GPU"),
            ((x, _q(6, k=41)), ValueError, r"w must be \[n, 40\]"), ((x, _q(2, 6)), ValueError, "w must be"),
            ((x, _q(0)), ValueError, "no rows"), ((x, w, torch.zeros(6, dtype=torch.bfloat16)), TypeError, "bias"),
            ((x, w, torch.zeros(5)), ValueError, "bias"), ((x, w, torch.zeros(12)[::2]), ValueError, "bias"),
            ((x, w, torch.zeros(6, requires_grad=True)), RuntimeError, "backward"),
            ((x, w, None, torch.zeros(3, 6, dtype=torch.bfloat16)), TypeError, "out"),
            ((x, w, None, torch.zeros(3, 5)), ValueError, "out"), ((x, w, None, torch.zeros(6, 3).t()), ValueError, "out"),
            ((x, w, None, x.scales.expand(6, 3).t()), ValueError, "out")):
        with pytest.raises(kind, match=error):
            ops.linear_int8(*a)
    with pytest.raises(TypeError, match="q must be an Int8"):
        ops.dequantize_int8(torch.zeros(3, 4))
    with pytest.raises(TypeError, match="dtype"):
        ops.dequantize_int8(x, torch.float16)
    for out in (torch.zeros(3, 41), torch.zeros(3, 40, dtype=torch.bfloat16), torch.zeros(40, 3).t()):
        with pytest.raises(ValueError, match="out"):
            ops.dequantize_int8(x, out=out)


def test_library_refuses_before_any_launch():
    lib = _lib.load()
    some = ctypes.cast(ctypes.create_string_buffer(64), ctypes.c_void_p).value // 16 * 16 + 16
    refused = lambda rc, text: rc == 1 and text in lib.mtl_last_error()
    assert refused(lib.mtl_quantize_int8(some, 8, some, some, 1, 0, 0, None), b"K must be")
    assert refused(lib.mtl_quantize_int8(some, 8, some, some, 1, 1 << 17, 0, None), b"K must be")
    assert refused(lib.mtl_quantize_int8(some, 8, some, some, -1, 8, 0, None), b"rows must be")
    assert refused(lib.mtl_quantize_int8(some, 8, some, some, 1, 8, 2, None), b"dtype")
    assert refused(lib.mtl_quantize_int8(None, 8, some, some, 1, 8, 0, None), b"null")
    assert refused(lib.mtl_quantize_int8(some, 8, some + 8, some, 1, 8, 0, None), b"aligned")
    assert refused(lib.mtl_dequantize_int8(some, some, some, 7, 1, 8, 0, None), b"overlap")
    assert refused(lib.mtl_dequantize_int8(some, None, some, 8, 1, 8, 0, None), b"null")
    assert lib.mtl_quantize_int8(None, 8, None, None, 0, 8, 0, None) == 0          # no rows: nothing to do
    assert lib.mtl_dequantize_int8(None, None, None, 8, 0, 8, 0, None) == 0
    n = _lib.AddRmsnormInt8Args(some, None, None, some, some, some, 1, 8, 1e-5, 0, 0, 0)
    for name, value, text in (("K", 0, b"K must be"), ("y_dtype", 2, b"y_dtype"), ("w_dtype", 3, b"w_dtype"),
                              ("w", None, b"null"), ("codes", some + 4, b"aligned"), ("M", 1 << 31, b"rows must be")):
        bad = _lib.AddRmsnormInt8Args.from_buffer_copy(n)
        setattr(bad, name, value)
        assert refused(lib.mtl_add_rmsnorm_int8(ctypes.byref(bad), None), text), name
    p = _lib.LinearInt8Args(some, some, some, some, None, some, 4, 1, 4, 8, 0, 0)
    for name, value, text in (("K", 1 << 17, b"K must be"), ("N", 0, b"N must be"), ("N", (1 << 27) + 1, b"N must be"),
                              ("ldy", 3, b"overlap"), ("dtype", 5, b"dtype"), ("w_scales", None, b"null"),
                              ("x", some + 8, b"aligned")):
        bad = _lib.LinearInt8Args.from_buffer_copy(p)
        setattr(bad, name, value)
        assert refused(lib.mtl_linear_int8(ctypes.byref(bad), None), text), name
    r = _lib.RowLinearInt8Args(some, None, None, None, some, some, None, some, 4, 8, 1e-5, 0, 0, 0)
    for change, text in (({"K": 0}, b"K must be"), ({"K": 8193}, b"K must be"), ({"K": 4097, "norm_w": some}, b"K must be"),
                         ({"N": 0}, b"N must be"), ({"dtype": 2}, b"dtype"), ({"x": None}, b"null"), ({"y": None}, b"null"),
                         ({"add": some}, b"need a norm"), ({"x_out": some}, b"need a norm"), ({"w": some + 8}, b"aligned"),
                         ({"norm_w": some, "x_out": some}, b"x_out"),
                         ({"norm_w": some, "add": some + 64, "x_out": some + 64}, b"x_out")):
        bad = _lib.RowLinearInt8Args.from_buffer_copy(r)
        for name, value in change.items():
            setattr(bad, name, value)
        assert refused(lib.mtl_row_linear_int8(ctypes.byref(bad), None), text), change
    for f in (lib.mtl_linear_int8, lib.mtl_add_rmsnorm_int8, lib.mtl_row_linear_int8):
        assert refused(f(None, None), b"null")
    assert lib.mtl_quantize_int8(None, 8, None, None, 0, 8, 0, None) == 0 and lib.mtl_last_error() == b""


def test_linear_int8_module_on_the_host():
    from mamba_lite.model import LinearInt8

    q = LinearInt8(_q(6), torch.zeros(6))
    assert (q.in_features, q.out_features) == (40, 6) and "in_features=40" in repr(q)
    s = q.scales.detach().clone()
    for cast in (lambda m: m.bfloat16(), lambda m: m.half(), lambda m: m.double(), lambda m: m.to("cpu", torch.float32)):
        cast(q)
        assert q.scales.dtype == torch.float32 and torch.equal(q.scales, s) and q.weight.dtype == torch.int8
        assert isinstance(q.scales, torch.nn.Parameter) and set(q.state_dict()) == {"weight", "scales", "bias"}
    p = LinearInt8(_q(6), torch.ones(6))
    p.load_state_dict(q.state_dict())
    assert torch.equal(p.bias, q.bias)
    assert torch.equal(q.int8(2, 5).codes, q.weight[2:5]) and tuple(q.int8().shape) == (6, 40)
    with pytest.raises(ValueError, match="matrix"):
        LinearInt8(_q(2, 3))


def test_shards_of_an_int8_model_are_refused():
    from mamba_lite import tp_utils
    from mamba_lite.model import LinearInt8, MambaConfig, MambaLM
    from mamba_lite.tp_model import LocalTPLM

    m = MambaLM(MambaConfig(d_model=32, n_layer=1, vocab_size=40))
    mx = m.layers[0].mixer
    mx.in_proj, mx.out_proj = LinearInt8(_q(128, k=32)), LinearInt8(_q(32, k=64))
    with pytest.raises(TypeError, match="quantize_int8"):
        tp_utils.shard_mixer_tensors({k: v.detach() for k, v in mx.state_dict().items()}, 64, 0, 2)
    m.head_int8 = LinearInt8(_q(40, k=32))
    with pytest.raises(TypeError, match="quantize_int8"):
        LocalTPLM.from_dense(m)


def test_a_checkpoint_of_floats_does_not_turn_into_codes():
    from mamba_lite.model import LinearInt8

    codes = torch.ones(6, 128, dtype=torch.int8)                # (as wide as its codes: nothing else would notice)
    for strict in (True, False):
        q = LinearInt8(ops.pack_int8(codes, torch.ones(6)), torch.zeros(6))
        with pytest.raises(RuntimeError, match="8-bit codes"):
            q.load_state_dict(torch.nn.Linear(128, 6).state_dict(), strict=strict)
        assert torch.equal(q.weight, codes) and not bool(q.bias.any())
    with pytest.raises(RuntimeError, match="float32"):
        q.load_state_dict({k: v.bfloat16() if k == "scales" else v for k, v in q.state_dict().items()})
    q.load_state_dict({k: v for k, v in q.state_dict().items() if k == "bias"}, strict=False)


def test_scales_that_record_a_gradient_are_refused():
    from mamba_lite.model import LinearInt8

    codes, s = torch.zeros(6, 128, dtype=torch.int8), torch.ones(6, requires_grad=True)
    w, x = ops.Int8(codes, s, 40), _q(2)
    for call in (lambda: ops.linear_int8(x, w), lambda: ops.linear_int8(ops.Int8(codes, s, 40), _q(3)),
                 lambda: ops.dequantize_int8(w)):
        with pytest.raises(RuntimeError, match="backward"):
            call()
    lin = LinearInt8(_q(6))
    lin.scales.requires_grad_()
    for call in (lambda: lin(x), lambda: lin.rows(x, 0, 3)):
        with pytest.raises(RuntimeError, match="backward"):
            call()


def test_linear_takes_as_many_rows_as_the_others():
    # (a check behind that of the rows)
    a = _lib.LinearInt8Args(None, None, None, None, None, None, 4, (1 << 31) - 1, 4, 8, 0, 0)
    lib = _lib.load()
    assert lib.mtl_linear_int8(ctypes.byref(a), None) == 1 and b"null" in lib.mtl_last_error()
    a.M = 1 << 31
    assert lib.mtl_linear_int8(ctypes.byref(a), None) == 1 and b"rows must be" in lib.mtl_last_error()


def test_a_float_row_is_refused_outputs_over_what_other_workgroups_read():
    # (addresses that nothing reads: every call here is refused)
    lib, at = _lib.load(), lambda i: (1 << 24) + (i << 16)
    n, k = 100, 300
    for dtype, f32 in ((0, 0), (1, 0), (1, 1)):
        es, ys = 2 if dtype else 4, 2 if dtype and not f32 else 4
        size = dict(x=4 * k, add=4 * k, norm_w=es * k, w=384 * n, w_scales=4 * n, bias=es * n, x_out=4 * k, y=ys * n)
        a = dict(x=at(0), add=at(1), x_out=at(2), norm_w=at(3), w=at(4), w_scales=at(5), bias=at(6), y=at(7))
        for out in ("x_out", "y"):
            for over in set(a) - {out}:
                # (the codes are moved in whole 16 bytes)
                for d in {0, 4, 16, size[over] - 4, 4 - size[out]} if over != "w" else {0, 16, size[over] - 4}:
                    p = _lib.RowLinearInt8Args(N=n, K=k, eps=1e-5, dtype=dtype, y_f32=f32, **dict(a, **{out: a[over] + d}))
                    assert lib.mtl_row_linear_int8(ctypes.byref(p), None) == 1, (out, over, d)
                    assert b"overlap" in lib.mtl_last_error(), (out, over, d)
        # without a norm the row is of dtype
        b = dict(a, add=None, x_out=None, norm_w=None)
        for d in (0, es * k - 2, 2 - ys * n):
            p = _lib.RowLinearInt8Args(N=n, K=k, dtype=dtype, y_f32=f32, **dict(b, y=a["x"] + d))
            assert lib.mtl_row_linear_int8(ctypes.byref(p), None) == 1 and b"overlap" in lib.mtl_last_error()


def test_the_norms_sum_is_refused_over_another_place_of_its_operands():
    # (addresses that nothing reads: every call here is refused)
    lib, at = _lib.load(), lambda i: (1 << 24) + (i << 16)
    m, k = 5, 300
    for y_dtype, w_dtype in ((0, 0), (1, 0), (0, 1), (1, 1)):
        size = dict(x=4 * m * k, y=(2 if y_dtype else 4) * m * k, w=(2 if w_dtype else 4) * k)
        a = dict(x=at(0), y=at(1), x_out=at(2), w=at(3), codes=at(4), scales=at(5))
        for over in size:
            for d in {0, 4, k, size[over] - 4, 4 - 4 * m * k, -4}:
                if d == 0 and (over == "x" or (over == "y" and not y_dtype)):
                    continue                                     # (in place)
                p = _lib.AddRmsnormInt8Args(M=m, K=k, eps=1e-5, y_dtype=y_dtype, w_dtype=w_dtype, **dict(a, x_out=a[over] + d))
                assert lib.mtl_add_rmsnorm_int8(ctypes.byref(p), None) == 1, (over, d)
                assert b"x_out" in lib.mtl_last_error(), (over, d)


def test_one_rule_says_where_a_float_row_is_put_into_codes_within_its_product():
    pays = _lib.load().mtl_row_linear_int8_pays
    # (n, k, norm): one launch measured faster, two
    for n, k, norm in ((768, 1536, 0), (8192, 64, 0), (12288, 512, 0), (24576, 1024, 0), (24576, 2048, 0), (50280, 2048, 0),
                       (65536, 4096, 0), (16384, 2560, 0), (16384, 7168, 0), (8192, 256, 1), (8192, 2048, 1), (16384, 4096, 1)):
        assert pays(n, k, norm) == 1, (n, k, norm)
    for n, k, norm in ((16384, 64, 0), (20480, 512, 0), (24576, 768, 0), (50280, 768, 0), (32768, 1024, 0), (24576, 2560, 0),
                       (20480, 7168, 0), (12288, 256, 1), (16384, 768, 1), (24576, 2560, 1), (50280, 2048, 1)):
        assert pays(n, k, norm) == 0, (n, k, norm)
    # what the launch does not take
    for n, k, norm in ((16, 8193, 0), (16, 4097, 1), (0, 64, 0), (16, 0, 0), (1 << 40, 2048, 0)):
        assert pays(n, k, norm) == 0, (n, k, norm)
    for n, k in ((768, 1536), (50280, 2048), (50280, 768), (16, 8193)):
        assert ops.row_linear_int8_pays(n, k) == bool(pays(n, k, 0))


@pytest.mark.parametrize("shape", [(40,), (1, 40), (1, 1, 40), (5, 40)])
def test_a_trace_is_refused_by_name_for_any_number_of_rows(shape):
    from mamba_lite.model import LinearInt8

    q = LinearInt8(_q(6))
    with pytest.raises(RuntimeError, match="trace"):
        torch.jit.trace(q, torch.zeros(shape))
    with pytest.raises(RuntimeError, match="trace"):
        torch.jit.trace(lambda x: ops.linear_int8(x, _q(6)), torch.zeros(shape))
