"""Refusals of the paged-cache operators at the edges (CPU-only host: the argument checks come
before any CUDA call; a call that passes them ends as a failed launch)."""

import pytest

from exl3_b200 import _lib
from test_paged import append, attend, cache


@pytest.mark.parametrize("kw", [
    dict(out_stride=0), dict(out_head_stride=0), dict(out_stride=0, out_head_stride=0),
    dict(out_stride=512), dict(out_head_stride=64), dict(out_stride=128, out_head_stride=128),
    dict(out_stride=128, out_head_stride=128 * 2 - 8), dict(rows_per_seq=3, seqs=1, out_stride=0),
    dict(seqs=1, out_head_stride=0)])
def test_attention_refuses_overlapping_outputs(kw):
    assert attend(**kw) == _lib.EBADSHAPE


@pytest.mark.parametrize("kw", [
    dict(q_out_stride=0), dict(q_out_head_stride=0), dict(q_out_stride=0, q_out_head_stride=0),
    dict(q_out_stride=512), dict(q_out_head_stride=64), dict(q_out_stride=128, q_out_head_stride=128),
    dict(tokens=1, q_out_head_stride=0), dict(q_heads=1, q_out_stride=64)])
def test_append_refuses_overlapping_outputs(kw):
    assert append(**kw) == _lib.EBADSHAPE


@pytest.mark.parametrize("call,kw", [
    (attend, dict()), (attend, dict(seqs=1, out_stride=0)), (attend, dict(out_stride=128, out_head_stride=256)),
    (attend, dict(q_heads=2, out_head_stride=128 * 2, out_stride=128)), (attend, dict(out_head_stride=136, out_stride=8 * 136)),
    (attend, dict(q_stride=0, q_head_stride=0)),  # an input may be an expanded view
    (append, dict()), (append, dict(tokens=1, q_out_stride=0)), (append, dict(q_out_stride=128, q_out_head_stride=3 * 128)),
    (append, dict(c=cache(kv_heads=1), q_heads=1, q_out_head_stride=0)), (append, dict(q_stride=0, k_stride=0, v_head_stride=0))])
def test_outputs_apart_are_taken(call, kw):
    import torch

    if torch.cuda.is_available():
        pytest.skip("the addresses are not real ones")
    assert call(**kw) == _lib.ELAUNCH


def test_rows_of_one_token_or_one_head():
    """The stride of a dimension of one does not decide whether rows are aligned (a helper of the
    wrappers; no device needed)."""
    import torch

    from exl3_b200 import paged

    base = torch.zeros(4096, dtype=torch.bfloat16)
    for shape, strides, ok in (((1, 4, 64), (259, 64, 1), True), ((3, 1, 64), (256, 67, 1), True), ((1, 1, 64), (3, 5, 1), True),
                               ((2, 4, 64), (259, 64, 1), False), ((3, 2, 64), (256, 67, 1), False), ((1, 4, 64), (256, 60, 1), False)):
        t = base.as_strided(shape, strides)
        got = paged._rows(t, copy=False)
        assert (got is not None) == ok
        if ok:
            assert got[0] is t and got[2] % 8 == 0 and got[3] % 8 == 0
        copied = paged._rows(t)
        assert (copied[0] is t) == ok and copied[2] % 8 == 0 and copied[3] % 8 == 0
