"""Refusals of bna_token_logprobs before it touches a device, and of its wrapper for CPU tensors."""
import pytest
import torch

import butterfly_b200 as bb
from butterfly_b200 import _lib

P = 1 << 20  # an aligned stand-in pointer: never dereferenced by a rejected call


def _call(**kw):
    a = dict(x=P, ld=100, ld_outer=0, rows=4, inner=4, vocab=100, dt=_lib.BF16, tok=P, tok64=1, lp=P, ent=P, ids=P, top=P, k=5, stream=None)
    a.update(kw)
    return _lib.lib().bna_token_logprobs(*a.values())


def test_refusals():
    assert _call(rows=0) == _lib.OK
    assert _call(dt=3) == _lib.BAD_DTYPE and _call(dt=-1) == _lib.BAD_DTYPE
    for bad in (dict(rows=-1), dict(vocab=0), dict(vocab=2 ** 31), dict(k=-1), dict(k=65), dict(k=11, vocab=10), dict(inner=0), dict(x=None),
                dict(ent=None), dict(tok=None), dict(lp=None), dict(ids=None), dict(top=None)):
        assert _call(**bad) == _lib.BAD_SHAPE, bad
    for bad in (dict(x=P + 1), dict(x=P + 2, dt=2), dict(tok=P + 4), dict(tok=P + 2, tok64=0), dict(lp=P + 2), dict(ent=P + 1), dict(ids=P + 4),
                dict(top=P + 2)):
        assert _call(**bad) == _lib.BAD_STRIDE, bad


def test_wrapper_refuses_cpu_tensors():
    with pytest.raises(ValueError, match="CUDA"):
        bb.token_logprobs(torch.zeros(2, 10), torch.zeros(2, dtype=torch.long))
    with pytest.raises(TypeError):
        bb.token_logprobs(None)
