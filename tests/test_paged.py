"""Refusals of the paged-cache operators: argument checks come before any CUDA call, so they
run on a CPU-only host (the pointers below are never dereferenced)."""

import ctypes

import pytest
import torch

from exl3_b200 import _lib, paged

P = 4096  # a 16-byte aligned, never dereferenced address


def cache(**kw):
    a = dict(k=P, v=P, dtype=_lib.DTYPE_BF16, pages=4, page_size=16, kv_heads=2, head_dim=128,
             page_stride=16 * 2 * 128, pos_stride=2 * 128, head_stride=128, k_scale=None, v_scale=None)
    a.update(kw)
    return _lib.PagedCache(*a.values())


def append(c=None, **kw):
    a = dict(cache=c or cache(), q=P, k=P, v=P, q_out=P, positions=P, slots=P, inv_freq=P, q_stride=1024,
             q_head_stride=128, k_stride=256, k_head_stride=128, v_stride=256, v_head_stride=128, q_out_stride=1024,
             q_out_head_stride=128, tokens=3, q_heads=8, rotary=128, interleaved=0, in_dtype=_lib.DTYPE_F16,
             q_out_dtype=_lib.DTYPE_BF16)
    a.update(kw)
    return _lib.lib().exl3b200_rope_append(ctypes.byref(_lib.RopeAppendArgs(*a.values())), None)


def attend(c=None, scratch=4096, nbytes=1 << 40, **kw):
    a = dict(cache=c or cache(), q=P, out=P, lse=None, block_table=P, seq_lens=P, q_stride=1024, q_head_stride=128,
             out_stride=1024, out_head_stride=128, table_stride=4, seqs=2, rows_per_seq=1, q_heads=8, max_pages=4,
             window=0, dtype=_lib.DTYPE_BF16, scale=0.1, softcap=0.0)
    a.update(kw)
    return _lib.lib().exl3b200_paged_attention(ctypes.byref(_lib.PagedAttentionArgs(*a.values())), scratch, nbytes, None)


@pytest.mark.parametrize("call", [append, attend])
@pytest.mark.parametrize("kw,code", [
    (dict(k=None), _lib.ENULL), (dict(v=None), _lib.ENULL), (dict(pages=0), _lib.EBADSHAPE),
    (dict(page_size=0), _lib.EBADSHAPE), (dict(kv_heads=0), _lib.EBADSHAPE), (dict(head_dim=96), _lib.EBADSHAPE),
    (dict(head_dim=256), _lib.EBADSHAPE), (dict(page_stride=-4096), _lib.EBADSHAPE),
    (dict(dtype=_lib.DTYPE_F32), _lib.EBADARG), (dict(dtype=_lib.DTYPE_F16), _lib.EBADARG),
    (dict(dtype=9), _lib.EBADARG), (dict(k=P + 8), _lib.EUNALIGNED), (dict(v=P + 2), _lib.EUNALIGNED),
    (dict(pos_stride=260), _lib.EUNALIGNED), (dict(head_stride=132), _lib.EUNALIGNED),
    (dict(page_stride=4097), _lib.EUNALIGNED)])
def test_cache_refusals(call, kw, code):
    assert call(cache(**kw)) == code


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), _lib.ENULL), (dict(slots=None), _lib.ENULL), (dict(positions=None), _lib.ENULL),
    (dict(inv_freq=None), _lib.ENULL), (dict(q_out=None), _lib.ENULL), (dict(tokens=0), _lib.EBADSHAPE),
    (dict(q_heads=0), _lib.EBADSHAPE), (dict(rotary=130), _lib.EBADSHAPE), (dict(rotary=24), _lib.EBADSHAPE),
    (dict(rotary=144), _lib.EBADSHAPE), (dict(rotary=-16), _lib.EBADSHAPE), (dict(interleaved=2), _lib.EBADARG),
    (dict(in_dtype=_lib.DTYPE_E4M3), _lib.EBADARG), (dict(q_out_dtype=_lib.DTYPE_F32), _lib.EBADARG),
    (dict(q_out_dtype=_lib.DTYPE_F16), _lib.EBADARG), (dict(q=P + 4), _lib.EUNALIGNED),
    (dict(k_stride=257), _lib.EUNALIGNED), (dict(v_head_stride=4), _lib.EUNALIGNED),
    (dict(q_out_stride=1028), _lib.EUNALIGNED)])
def test_append_refusals(kw, code):
    assert append(**kw) == code


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), _lib.ENULL), (dict(block_table=None), _lib.ENULL), (dict(seq_lens=None), _lib.ENULL),
    (dict(scratch=None), _lib.ENULL), (dict(seqs=0), _lib.EBADSHAPE), (dict(max_pages=0), _lib.EBADSHAPE),
    (dict(table_stride=3), _lib.EBADSHAPE), (dict(window=-1), _lib.EBADSHAPE), (dict(q_heads=7), _lib.EBADSHAPE),
    (dict(q_heads=1), _lib.EBADSHAPE), (dict(rows_per_seq=0), _lib.EBADSHAPE),
    (dict(rows_per_seq=257), _lib.EBADSHAPE), (dict(dtype=_lib.DTYPE_F32), _lib.EBADARG),
    (dict(softcap=-1.0), _lib.EBADARG), (dict(softcap=float("nan")), _lib.EBADARG), (dict(softcap=1e-9), _lib.EBADARG),
    (dict(scale=float("inf")), _lib.EBADARG), (dict(scale=0.0), _lib.EBADARG), (dict(scale=-0.1), _lib.EBADARG), (dict(nbytes=4096), _lib.EWORKSPACE),
    (dict(scratch=4096 + 16), _lib.EUNALIGNED), (dict(q=P + 8), _lib.EUNALIGNED),
    (dict(q_stride=1023), _lib.EUNALIGNED), (dict(out_head_stride=130), _lib.EUNALIGNED),
    (dict(seqs=2 ** 30, max_pages=2 ** 30, table_stride=2 ** 30), _lib.EBADSHAPE)])
def test_attention_refusals(kw, code):
    assert attend(**kw) == code


def test_scratch_size():
    size = _lib.lib().exl3b200_paged_attention_scratch_size
    assert size(1, 64, 8, 128) > 0 and size(5, 32, 4, 128) > size(1, 32, 4, 128)
    for bad in ((0, 64, 8, 128), (1, 63, 8, 128), (1, 64, 0, 128), (1, 64, 8, 80), (1025, 1, 1, 64)):
        assert size(*bad) == 0
    assert attend(nbytes=size(1, 8, 2, 128) - 1) == _lib.EWORKSPACE


def test_null_arguments():
    L = _lib.lib()
    assert L.exl3b200_rope_append(None, None) == _lib.ENULL
    assert L.exl3b200_paged_attention(None, P, 1 << 30, None) == _lib.ENULL


def test_cpu_tensors_are_refused():
    kc = torch.zeros(2, 16, 2, 128, dtype=torch.bfloat16)
    x = torch.zeros(1, 2, 128, dtype=torch.bfloat16)
    one = torch.zeros(1, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="no CPU path"):
        paged.rope_append(x, x, x, kc, kc, one, one, torch.zeros(64))
    with pytest.raises(RuntimeError, match="no CPU path"):
        paged.attention(x, kc, kc, torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))


def test_packed_arguments_have_the_structs_layout():
    def fields(st):
        out = []
        for name, t in st._fields_:
            v = getattr(st, name)
            out += fields(v) if isinstance(v, ctypes.Structure) else [v or 0]
        return out

    for cls, pack in ((_lib.RopeAppendArgs, _lib.pack_rope_append), (_lib.PagedAttentionArgs, _lib.pack_paged_attention)):
        raw = bytes((37 * i + 1) % 120 for i in range(ctypes.sizeof(cls)))
        st = cls.from_buffer_copy(raw)
        again = cls.from_buffer_copy(pack(*fields(st)))
        assert len(pack(*fields(st))) == ctypes.sizeof(cls) and fields(again) == fields(st)
