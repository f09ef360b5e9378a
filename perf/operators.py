"""Performance cases of the 4-bit serving operators on one GPU: products with 4-bit weights, those weights as a matrix,
and log probabilities of tokens with entropy and top alternatives.

listed()   the cases by name;  draw(rng)  one more case of the same ranges
prepare / run / work / exact: the inputs of a case, one pass, the bytes and operations it cannot do without, and the
           64-bit values.  With `own` false, run() computes the operators in elementary torch operations; with `own`
           true it calls this framework's.

Kinds:
  linear   y = x W^T (+ bias) for 1 to 64 rows of x, W [n, k] in 4-bit codes: w = scale (code - zero), one scale (and
           zero, or 8) for each group of g columns of a row: a decode step's projections and lm_head
  matrix   W itself, in fp32 or bf16: what a prompt's product reads
  logprob  for rows of logits: ln p of a given token, the row's entropy, and its `top` most probable tokens
"""
import os
import sys

import torch

own = False

DEV = "cuda"
VOCAB = 50280


def _ops():
    """This framework's operators (only where `own` is true)."""
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mamba-tp-lite_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from mamba_lite import ops

    return ops


# ------------------------------------------------------------------ the cases
def listed():
    lin, mat, lp = dict(kind="linear"), dict(kind="matrix"), dict(kind="logprob", masked=False)
    return [
        # one token of one stream through the out_proj of a 768-wide model: the smallest work per call
        dict(lin, name="linear_bf16_m1_768x1536_g64", dtype="bf16", m=1, n=768, k=1536, g=64, zeros=False,
             scale="bf16", bias=False),
        # one token through the in_proj of a 2048-wide fp32 model
        dict(lin, name="linear_fp32_m1_8192x2048_g128", dtype="fp32", m=1, n=8192, k=2048, g=128, zeros=False,
             scale="bf16", bias=False),
        # a server of few streams, the out_proj of the same model, codes with zero points and fp32 scales
        dict(lin, name="linear_fp32_m5_2048x4096_g64_z", dtype="fp32", m=5, n=2048, k=4096, g=64, zeros=True,
             scale="fp32", bias=False),
        # the lm_head of a 2048-wide model for a batch of 16 streams
        dict(lin, name="linear_bf16_m16_50280x2048_g128", dtype="bf16", m=16, n=VOCAB, k=2048, g=128, zeros=False,
             scale="bf16", bias=False),
        # widths that are no tile's multiple, a batch past one matrix tile, small groups, a bias
        dict(lin, name="linear_bf16_m33_1001x777_g32_z", dtype="bf16", m=33, n=1001, k=777, g=32, zeros=True,
             scale="bf16", bias=True),
        # a prompt's in_proj matrix of the 2048-wide model in bf16, and an out_proj of the 768-wide one in fp32
        dict(mat, name="matrix_bf16_8192x2048_g128", dtype="bf16", n=8192, k=2048, g=128, zeros=False, scale="bf16"),
        dict(mat, name="matrix_fp32_768x1536_g64_z", dtype="fp32", n=768, k=1536, g=64, zeros=True, scale="bf16"),
        # one decoded token with its five best alternatives
        dict(lp, name="logprob_fp32_1x50280_top5", dtype="fp32", b=1, l=1, v=VOCAB, top=5),
        # a step of 32 streams, twenty alternatives each
        dict(lp, name="logprob_fp32_32x50280_top20", dtype="fp32", b=32, l=1, v=VOCAB, top=20),
        # scoring eight prompts of 1024 tokens: each token given the ones before it (the rows are a view that leaves out
        # every prompt's last position)
        dict(lp, name="logprob_fp32_8x1023x50280", dtype="fp32", b=8, l=1023, v=VOCAB, top=0),
        # scoring in bf16 with alternatives: equal logits are common there
        dict(lp, name="logprob_bf16_2x511x50280_top5", dtype="bf16", b=2, l=511, v=VOCAB, top=5),
        # a vocabulary of odd size under constraint masks, some of which leave nothing, and padding tokens
        dict(lp, name="logprob_fp32_37x10007_top64_masked", dtype="fp32", b=37, l=1, v=10007, top=64, masked=True),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear", "matrix", "logprob", "logprob", "logprob"])
    if kind == "logprob":
        v = _log(rng, 1000, 131072)
        l = rng.choice([1, 1, _log(rng, 2, 1023)])
        b = _log(rng, 1, max(1, min(64 if l == 1 else 8, 8 * 1023 * VOCAB // (v * l))))
        return dict(kind=kind, dtype=rng.choice(["fp32", "fp32", "bf16"]), b=b, l=l, v=v,
                    top=rng.choice([0, 1, 5, 20, 64]) if b * l <= 2048 else rng.choice([0, 5]),
                    masked=rng.random() < 0.3)
    n = _log(rng, 48, VOCAB)
    k = _log(rng, 64, min(8192, VOCAB * 2048 // n))
    if rng.random() < 0.5:
        n, k = max(64, n // 64 * 64), max(64, k // 64 * 64)
    q = dict(kind=kind, dtype=rng.choice(["fp32", "bf16"]), n=n, k=k, g=rng.choice([32, 64, 128]),
             zeros=rng.random() < 0.5, scale=rng.choice(["bf16", "bf16", "fp32"]))
    if kind == "matrix":
        return q
    most = max(1, 16 * VOCAB * 2048 // (n * k))
    return dict(q, m=_log(rng, 1, min(64, most)), bias=rng.random() < 0.3)


# ------------------------------------------------------------------ inputs
def _type(name):
    return torch.bfloat16 if name == "bf16" else torch.float32


def _size(name):
    return 2 if name == "bf16" else 4


def _weights(case, g):
    """A matrix of 4-bit codes as checkpoints hold it: codes [n, k] of about normal weights, scales and zeros for
    groups of columns (w ~ N(0, 1/k))."""
    n, k, ng = case["n"], case["k"], -(-case["k"] // case["g"])
    mid = 8.0
    zeros = None
    if case["zeros"]:
        zeros = torch.randint(5, 11, (n, ng), device=DEV, generator=g, dtype=torch.uint8)
    codes = torch.empty(n, k, device=DEV, dtype=torch.uint8)
    rows = max(1, (1 << 24) // k)
    for r in range(0, n, rows):
        t = torch.randn(min(rows, n - r), k, device=DEV, generator=g).mul_(2.7).add_(mid)
        codes[r:r + rows] = t.round_().clamp_(0, 15).to(torch.uint8)
    scales = (torch.rand(n, ng, device=DEV, generator=g) * 0.6 + 0.7) / (2.7 * k ** 0.5)
    return codes, scales.to(_type(case["scale"])), zeros


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    if case["kind"] == "logprob":
        return _prepare_logits(case, g)
    codes, scales, zeros = _weights(case, g)
    st = dict(kind=case["kind"], dtype=_type(case["dtype"]), n=case["n"], k=case["k"], g=case["g"], scales=scales,
              zeros=zeros)
    if own:
        st["w4"] = _ops().pack_w4(codes, scales, zeros, group=case["g"])      # laid out once, kept with the model
    else:
        if case["k"] % 2:
            codes = torch.nn.functional.pad(codes, (0, 1))
        st["packed"] = codes[:, 0::2] | (codes[:, 1::2] << 4)                 # two codes a byte
    if case["kind"] == "linear":
        st["x"] = torch.randn(case["m"], case["k"], device=DEV, generator=g).to(st["dtype"])
        st["bias"] = torch.randn(case["n"], device=DEV, generator=g).mul_(0.1).to(st["dtype"]) if case["bias"] else None
    return st


def _prepare_logits(case, g):
    b, l, v, t = case["b"], case["l"], case["v"], _type(case["dtype"])
    n = l + 1 if l > 1 else 1                              # a prompt's last position is not scored
    x = torch.empty(b, n, v, device=DEV, dtype=t)
    tokens = torch.randint(0, v, (b, l), device=DEV, generator=g)
    for i in range(b):
        xi = torch.randn(n, v, device=DEV, generator=g).mul_(2.2)
        likely = torch.randint(0, v // 24, (n, 24), device=DEV, generator=g)
        likely += torch.arange(24, device=DEV) * (v // 24)      # no token twice
        likely = likely.gather(1, torch.rand(n, 24, device=DEV, generator=g).argsort(dim=1, stable=True))
        xi.scatter_(1, likely, torch.randn(n, 24, device=DEV, generator=g).mul_(2.5).add_(9.0))
        x[i] = xi.to(t)
        pick = torch.rand(l, device=DEV, generator=g) < 0.7      # most tokens of a text are likely ones
        tokens[i] = torch.where(pick, likely[:l, 0], tokens[i])
    if case["masked"]:
        for r in range(b):
            allowed = torch.rand(v, device=DEV, generator=g) < 0.02
            allowed[tokens[r, 0]] = True
            if r % 7 == 1:
                x[r].masked_fill_(~allowed, float("-inf"))              # a constraint on the next token
            elif r % 7 == 2:
                x[r].masked_fill_(~allowed, torch.finfo(t).min)         # the same with the type's lowest value
            elif r % 7 == 3:
                x[r, ..., 3:] = float("-inf")                           # fewer tokens than alternatives
            elif r % 7 == 4:
                x[r] = float("-inf")                                    # nothing is allowed
            elif r % 7 == 5:
                tokens[r] = -100                                        # padding
    return dict(kind="logprob", logits=x[:, :l], tokens=tokens, top=case["top"])


# ------------------------------------------------------------------ one pass
@torch.no_grad()
def run(st):
    if st["kind"] == "linear":
        return _ops().linear_w4(st["x"], st["w4"], st["bias"]) if own else _plain_linear(st)
    if st["kind"] == "matrix":
        return _ops().dequantize_w4(st["w4"], st["dtype"]) if own else _plain_matrix(st).to(st["dtype"])
    if not own:
        return _plain_logprobs(st["logits"], st["tokens"], st["top"])
    r = _ops().token_logprobs(st["logits"], st["tokens"], top=st["top"])
    return (r.logprob, r.entropy, r.top_logprob, r.top_token) if st["top"] else (r.logprob, r.entropy)


def _plain_matrix(st):
    n, k, g = st["n"], st["k"], st["g"]
    q = torch.stack((st["packed"] & 15, st["packed"] >> 4), -1).view(n, -1)[:, :k].float()
    z = 8.0 if st["zeros"] is None else st["zeros"].float().repeat_interleave(g, 1)[:, :k]
    return (q - z) * st["scales"].float().repeat_interleave(g, 1)[:, :k]


def _plain_linear(st):
    y = st["x"].float() @ _plain_matrix(st).t()
    return (y if st["bias"] is None else y + st["bias"].float()).to(st["dtype"])


def _plain_logprobs(logits, tokens, top):
    x = logits.float()
    m = x.amax(-1, keepdim=True)
    none = m == float("-inf")                                   # a row with no token left
    m = torch.where(none, 0.0, m)
    d = x - m
    e = torch.exp(d)
    s = e.sum(-1, keepdim=True)
    ls = torch.log(s)
    inside = tokens.clamp_min(0)[..., None]
    lp = torch.where(none, float("-inf"), d.gather(-1, inside) - ls)[..., 0]
    lp = torch.where(tokens < 0, 0.0, lp)
    h = torch.where(none, 0.0, ls - torch.where(e > 0, d * e, 0.0).sum(-1, keepdim=True) / s)[..., 0]
    if not top:
        return lp, h
    v, i = torch.sort(x, dim=-1, descending=True, stable=True)  # equal logits: the lower index first
    v, i = v[..., :top], i[..., :top]
    gone = v == float("-inf")
    return lp, h, torch.where(gone, v, v - m - ls), torch.where(gone, -1, i)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    e = _size(case["dtype"])
    if case["kind"] == "logprob":
        rows, v, top = case["b"] * case["l"], case["v"], case["top"]
        # a difference, an exponential, a sum, a product and its sum, a maximum for every logit
        return {"bytes": rows * (v * e + 8 + 8 + 12 * top), "flops": 6 * rows * v}
    n, k, ng = case["n"], case["k"], -(-case["k"] // case["g"])
    weights = (n * k + 1) // 2 + n * ng * (_size(case["scale"]) + (1 if case["zeros"] else 0))
    if case["kind"] == "matrix":
        return {"bytes": weights + n * k * e, "flops": 2 * n * k}
    m = case["m"]
    return {"bytes": weights + m * k * e + m * n * e + (n * e if case["bias"] else 0), "flops": 2 * m * n * k}


# ------------------------------------------------------------------ the same in 64 bits
@torch.no_grad()
def exact(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    if case["kind"] == "logprob":
        return _exact_logprobs(_prepare_logits(case, g))
    codes, scales, zeros = _weights(case, g)
    n, k = case["n"], case["k"]
    col = torch.arange(k, device=DEV) // case["g"]
    x = bias = None
    if case["kind"] == "linear":
        t = _type(case["dtype"])
        x = torch.randn(case["m"], k, device=DEV, generator=g).to(t).double()
        bias = torch.randn(n, device=DEV, generator=g).mul_(0.1).to(t).double() if case["bias"] else 0.0
    out = []
    rows = max(1, (1 << 25) // k)
    for r in range(0, n, rows):
        w = codes[r:r + rows].double()
        w -= 8.0 if zeros is None else zeros[r:r + rows].double()[:, col]
        w *= scales[r:r + rows].double()[:, col]
        out.append(w if x is None else x @ w.t().contiguous())
    return torch.cat(out, 0) if x is None else torch.cat(out, 1) + bias


def _exact_logprobs(st):
    x, tokens, top = st["logits"], st["tokens"], st["top"]
    v = x.shape[-1]
    parts = []
    for i in range(x.shape[0]):                          # one prompt at a time
        p = x[i].double()
        z = torch.logsumexp(p, -1)
        lnp = p - z[:, None]
        empty = torch.isinf(z)
        lnp[empty] = float("-inf")
        h = -(lnp.exp() * torch.where(torch.isinf(lnp), 0.0, lnp)).sum(-1)
        c = tokens[i]
        lp = lnp[torch.arange(len(c), device=DEV), c.clamp(0, v - 1)]
        lp[c < 0] = 0.0
        got = [lp, h]
        if top:
            # (-value, index) in order: equal values by index
            order = torch.argsort(-p, dim=-1, stable=True)[:, :top]
            a = lnp.gather(1, order)
            order[a == float("-inf")] = -1
            got += [a, order]
        parts.append(got)
    return tuple(torch.stack(t) for t in zip(*parts))
