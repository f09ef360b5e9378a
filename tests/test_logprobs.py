"""What token_logprobs and its entry point refuse, on the host."""
import ctypes

import pytest
import torch

from mamba_lite import _lib, ops


def test_calls_are_refused_on_the_host():
    x, t = torch.zeros(3, 50), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.token_logprobs(x, t)
    for bad in (dict(tokens=t[:2]), dict(tokens=t.int()), dict(top=51), dict(top=-1), dict(logits=torch.zeros(3, 0)),
                dict(logits=torch.zeros(3, 100), top=65)):
        with pytest.raises(ValueError):
            ops.token_logprobs(**{**dict(logits=x, tokens=t), **bad})
    with pytest.raises(TypeError):
        ops.token_logprobs(x.half(), t)
    with pytest.raises(TypeError):
        ops.token_logprobs(x.long(), t)
    with pytest.raises(RuntimeError, match="backward"):
        ops.token_logprobs(x.requires_grad_(), t)


@pytest.mark.parametrize("change,error", [
    (dict(dtype=2), b"dtype"), (dict(vocab=0), b"vocab"), (dict(vocab=1 << 31), b"vocab"), (dict(top=65), b"top"),
    (dict(top=-1), b"top"), (dict(vocab=4), b"top"), (dict(outer=-1), b"rows"), (dict(outer=1 << 20, inner=1 << 20), b"rows"),
    (dict(logits=None), b"null"), (dict(tokens=None), b"null"), (dict(logprob=None), b"null"),
    (dict(entropy=None), b"null"), (dict(top_logprob=None), b"null"), (dict(top_token=None), b"null"),
])
def test_the_library_refuses(change, error):
    a = dict(logits=0x1000, tokens=0x1000, logprob=0x1000, entropy=0x1000, top_logprob=0x1000, top_token=0x1000,
             outer=2, inner=3, stride_outer=300, stride_inner=100, vocab=100, top=5, dtype=0)
    lib = _lib.load()
    assert lib.mtl_token_logprobs(ctypes.byref(_lib.TokenLogprobsArgs(**{**a, **change})), None) == 1
    assert error in lib.mtl_last_error()
    assert lib.mtl_token_logprobs(ctypes.byref(_lib.TokenLogprobsArgs(**{**a, "outer": 0})), None) == 0
    assert lib.mtl_token_logprobs(None, None) == 1
