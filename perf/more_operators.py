"""Performance cases of the 8-bit integer serving operators on one GPU: rows quantized to int8 with a scale each, the
residual add and RMSNorm with such an output, the product of two such matrices, and their values read back.

listed()   the cases by name;  draw(rng)  one more case of the same ranges
prepare / run / work / exact: the inputs of a case, one pass, the bytes and operations it cannot do without, and the
           64-bit values.  With `own` false, run() computes the operators in elementary torch operations; with `own`
           true it calls this framework's.

An int8 row stands for code * scale, its codes in -127..127.  A row t of float32 values is put into codes by its largest
magnitude a: code = the whole number nearest to 127 t / a (halves to the even one), scale = a / 127; a row of zeros has
codes and scale 0.

Kinds:
  linear      y = X W^T (+ bias) for X [m, k] and W [n, k] in int8, one scale per row of each: the projections and the
              lm_head of a decode step (few rows) and of prompts (many)
  norm        h = x + y in float32, and w rmsnorm(h) in int8: what stands between two blocks.  The codes are those of
              the float32 row t = h w, since the norm's factor r = 1 / sqrt(mean(h^2) + eps) belongs to the row's
              scale, a r / 127
  quantize    rows of floats in int8: the input of out_proj
  dequantize  the floats that such rows stand for

What is held in 8 bits is returned as the values it stands for: norm and quantize read their rows back.
"""
import os
import sys

import torch

own = False

DEV = "cuda"
VOCAB = 50280
EPS = 1e-5


def _ops():
    """This framework's operators (only where `own` is true)."""
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mamba-tp-lite_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from mamba_lite import ops

    return ops


# ------------------------------------------------------------------ the cases
def listed():
    lin, norm, quant, deq = (dict(kind=k) for k in ("linear", "norm", "quantize", "dequantize"))
    return [
        # one token of one stream through the out_proj of a 768-wide model: the smallest product
        dict(lin, name="linear_fp32_m1_768x1536", dtype="fp32", m=1, n=768, k=1536, bias=False),
        # a batch of 16 streams through the lm_head of a 2048-wide model
        dict(lin, name="linear_bf16_m16_50280x2048", dtype="bf16", m=16, n=VOCAB, k=2048, bias=False),
        # widths that are no tile's multiple, a batch past two matrix tiles, a bias
        dict(lin, name="linear_bf16_m33_1001x777_bias", dtype="bf16", m=33, n=1001, k=777, bias=True),
        # a short prompt through the out_proj of the 2048-wide model
        dict(lin, name="linear_fp32_m256_2048x4096", dtype="fp32", m=256, n=2048, k=4096, bias=False),
        # a prompt of 1024 tokens through its in_proj
        dict(lin, name="linear_fp32_m1024_8192x2048", dtype="fp32", m=1024, n=8192, k=2048, bias=False),
        # 32 prompts of 1024 tokens through it: the largest
        dict(lin, name="linear_bf16_m32768_8192x2048", dtype="bf16", m=32768, n=8192, k=2048, bias=False),
        # one token between two blocks of the 768-wide model
        dict(norm, name="norm_fp32_m1_768", dtype="fp32", m=1, k=768, y="fp32"),
        # 32 prompts of 1024 tokens between two blocks of a bf16 model
        dict(norm, name="norm_bf16_m32768_2048", dtype="bf16", m=32768, k=2048, y="bf16"),
        # the out_proj's input in a step of 8 streams, and in 32 prompts of 1024 tokens of the 768-wide model
        dict(quant, name="quantize_bf16_m8_4096", dtype="bf16", m=8, k=4096),
        dict(quant, name="quantize_fp32_m32768_1536", dtype="fp32", m=32768, k=1536),
        # an in_proj's matrix read back in bf16, and one of odd sizes in fp32
        dict(deq, name="dequantize_bf16_8192x2048", dtype="bf16", m=8192, k=2048),
        dict(deq, name="dequantize_fp32_1001x777", dtype="fp32", m=1001, k=777),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear", "norm", "norm", "quantize", "dequantize"])
    even = rng.random() < 0.5                              # whole tiles, as most models have
    if kind == "linear":
        n = _log(rng, 48, VOCAB)
        k = _log(rng, 64, 8192)
        if even:
            n, k = max(64, n // 64 * 64), max(128, k // 128 * 128)
        most = min(32768, 32768 * 8192 * 2048 // (n * k), 32768 * 8192 // n)
        return dict(kind=kind, dtype=rng.choice(["fp32", "bf16"]), m=_log(rng, 1, max(1, most)), n=n, k=k,
                    bias=rng.random() < 0.3)
    k = _log(rng, 64, 8192)
    if even:
        k = max(128, k // 128 * 128)
    q = dict(kind=kind, dtype=rng.choice(["fp32", "bf16"]), m=_log(rng, 1, 32768 * 2048 // max(k, 2048)), k=k)
    return dict(q, y=rng.choice(["fp32", "bf16", "none"])) if kind == "norm" else q


# ------------------------------------------------------------------ inputs
def _type(name):
    return torch.bfloat16 if name == "bf16" else torch.float32


def _size(name):
    return 2 if name == "bf16" else 4


def _rows(m, k, g):
    """Activations: some channels far larger than the others, and rows of different sizes."""
    x = torch.randn(m, k, device=DEV, generator=g)
    x *= 1.0 + 7.0 * (torch.rand(k, device=DEV, generator=g) < 0.01)
    x *= 0.5 + torch.rand(m, 1, device=DEV, generator=g)
    return x


def _codes(t):
    """(codes, the rows' largest magnitudes a): 127 t / a to the nearest whole number.  The quotient is taken in 64 bits,
    where 127 t is exact and no value next to a border crosses it."""
    a = t.abs().amax(-1, keepdim=True)
    q = t.double().mul_(127.0).div_(torch.where(a > 0, a, 1.0).double())
    return q.round_().to(torch.int8), a


def _held(t):
    """Rows as checkpoints and caches hold them: codes int8 [m, k], scales [m]."""
    codes, a = _codes(t)
    return codes, (a / 127.0)[..., 0]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    kind, k = case["kind"], case["k"]
    st = dict(kind=kind, dtype=_type(case["dtype"]))
    if kind == "linear":
        x = _held(_rows(case["m"], k, g))
        w = _held(torch.randn(case["n"], k, device=DEV, generator=g) * k ** -0.5)
        st["bias"] = torch.randn(case["n"], device=DEV, generator=g).mul_(0.1).to(st["dtype"]) if case["bias"] else None
        if own:                                             # laid out once, kept with the model
            x, w = (_ops().pack_int8(*t, dtype=st["dtype"]) for t in (x, w))
        st["x"], st["w"] = x, w
    elif kind == "dequantize":
        q = _held(torch.randn(case["m"], k, device=DEV, generator=g) * k ** -0.5)
        st["q"] = _ops().pack_int8(*q, dtype=st["dtype"]) if own else q
    elif kind == "quantize":
        st["x"] = _activations(case, g)
    else:
        st["x"], st["y"], st["w"] = _residual(case, g)
        st["h"] = torch.empty_like(st["x"])
    return st


def _activations(case, g):
    x = _rows(case["m"], case["k"], g)
    x[torch.rand(case["m"], device=DEV, generator=g) < 0.01] = 0.0          # padding rows
    return x.to(_type(case["dtype"]))


def _residual(case, g):
    m, k = case["m"], case["k"]
    x = _rows(m, k, g) * 3.0                               # the residual stream is float32 in both models
    y = None if case["y"] == "none" else _rows(m, k, g).to(_type(case["y"]))
    w = (1.0 + 0.3 * torch.randn(k, device=DEV, generator=g)).to(_type(case["dtype"]))
    return x, y, w


# ------------------------------------------------------------------ one pass
@torch.no_grad()
def run(st):
    if not own:
        return _plain(st)
    ops, kind = _ops(), st["kind"]
    if kind == "linear":
        return ops.linear_int8(st["x"], st["w"], st["bias"])
    if kind == "dequantize":
        return ops.dequantize_int8(st["q"])
    if kind == "quantize":
        q = ops.quantize_int8(st["x"])
        return ops.dequantize_int8(q), q.scales
    q = ops.add_rmsnorm_int8(st["x"], st["w"], EPS, y=st["y"], x_out=None if st["y"] is None else st["h"],
                             dtype=st["dtype"])
    values = ops.dequantize_int8(q)
    return (values, q.scales) if st["y"] is None else (st["h"], values, q.scales)


def _plain(st):
    kind, dtype = st["kind"], st["dtype"]
    if kind == "linear":
        (xc, xs), (wc, ws) = st["x"], st["w"]
        y = (xc.float() @ wc.float().t()) * xs[:, None] * ws
        return (y if st["bias"] is None else y + st["bias"].float()).to(dtype)
    if kind == "dequantize":
        codes, scales = st["q"]
        return (codes.float() * scales[:, None]).to(dtype)
    if kind == "quantize":
        codes, scales = _held(st["x"].float())
        return (codes.float() * scales[:, None]).to(dtype), scales
    h = st["x"] if st["y"] is None else st["x"] + st["y"].float()
    codes, a = _codes(h * st["w"].float())
    scales = a * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS) / 127.0
    values = (codes.float() * scales).to(dtype)
    return (values, scales[:, 0]) if st["y"] is None else (h, values, scales[:, 0])


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    e, kind, m, k = _size(case["dtype"]), case["kind"], case["m"], case["k"]
    if kind == "linear":
        n = case["n"]
        return {"bytes": m * k + n * k + 4 * (m + n) + m * n * e + (n * e if case["bias"] else 0), "flops": 2 * m * n * k}
    held = m * k + 4 * m                                   # codes and scales
    if kind == "dequantize":
        return {"bytes": held + m * k * e, "flops": m * k}
    # the rows in int8 are written and, read back, written as floats
    if kind == "quantize":
        return {"bytes": m * k * e + 2 * held + m * k * e, "flops": 4 * m * k}
    y = {"none": 0, "bf16": 2, "fp32": 4}[case["y"]]
    return {"bytes": m * k * (4 + y + (4 if y else 0)) + k * e + 2 * held + m * k * e, "flops": 8 * m * k}


# ------------------------------------------------------------------ the same in 64 bits
@torch.no_grad()
def exact(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    kind, m, k = case["kind"], case["m"], case["k"]
    if kind == "linear":
        xc, xs = _held(_rows(m, k, g))
        wc, ws = _held(torch.randn(case["n"], k, device=DEV, generator=g) * k ** -0.5)
        b = torch.randn(case["n"], device=DEV, generator=g).mul_(0.1).to(_type(case["dtype"])).double() if case["bias"] else 0.0
        w = (wc.double() * ws.double()[:, None]).t().contiguous()
        rows = max(1, (1 << 27) // case["n"])
        return torch.cat([(xc[i:i + rows].double() * xs[i:i + rows].double()[:, None]) @ w + b for i in range(0, m, rows)])
    if kind == "dequantize":
        codes, scales = _held(torch.randn(m, k, device=DEV, generator=g) * k ** -0.5)
        return codes.double() * scales.double()[:, None]
    h = None
    if kind == "quantize":
        t = _activations(case, g).double()
        r = 1.0
    else:
        x, y, w = _residual(case, g)
        h = x.double() if y is None else (x.double() + y.double()).float().double()     # the stored rows
        r = (h.pow(2).sum(-1, keepdim=True) / k + EPS).pow(-0.5)
        t = (h * w.double()).float().double()               # the float32 row
    most = t.abs().max(-1, keepdim=True).values
    codes = torch.where(most > 0, (127.0 * t / most).round(), 0.0)
    values, scales = codes * (most / 127.0) * r, (most / 127.0 * r)[:, 0]
    return (values, scales) if h is None or case["y"] == "none" else (h, values, scales)
