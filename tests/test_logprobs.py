"""Refusals of token_logprobs: argument checks come before any CUDA call (CPU-only host)."""

import pytest
import torch

from exl3_b200 import _lib
from exl3_b200 import logprobs as LP

P = 4096  # never dereferenced


def call(**kw):
    a = dict(logits=P, stride=1000, rows=2, vocab=1000, dtype=_lib.DTYPE_BF16, tokens=P, top=5, lp=P, ent=P, tlp=P,
             ids=P, stream=None)
    a.update(kw)
    return _lib.lib().exl3b200_token_logprobs(*a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(logits=None), _lib.ENULL), (dict(tokens=None), _lib.ENULL), (dict(lp=None), _lib.ENULL),
    (dict(ent=None), _lib.ENULL), (dict(tlp=None), _lib.ENULL), (dict(ids=None), _lib.ENULL),
    (dict(rows=0), _lib.EBADSHAPE), (dict(vocab=0), _lib.EBADSHAPE),
    (dict(top=33), _lib.EBADSHAPE), (dict(top=-1), _lib.EBADSHAPE), (dict(vocab=4, stride=4), _lib.EBADSHAPE),
    (dict(stride=999), _lib.EBADSHAPE), (dict(vocab=2 ** 30 + 1, stride=2 ** 31), _lib.EBADSHAPE),
    (dict(dtype=_lib.DTYPE_E4M3), _lib.EBADARG), (dict(logits=P + 1), _lib.EUNALIGNED),
    (dict(logits=P + 2, dtype=_lib.DTYPE_F32), _lib.EUNALIGNED)])
def test_refusals(kw, code):
    assert call(**kw) == code


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="no CPU path"):
        LP.token_logprobs(torch.zeros(2, 10), torch.zeros(2, dtype=torch.int64), 3)
