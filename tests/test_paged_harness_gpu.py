"""The paged decode step and the reported log-probabilities, as a serving loop runs them:
EXL3 q/k/v -> rope_append -> attention over the pages -> EXL3 o ... lm_head -> token_logprobs.

The paged and the dense unfused step share weights and matmul kernels; the dense one rounds
its attention output to bf16 as the paged one does, so the residual streams agree to the 1e-2
(max abs difference over max abs value) that the fused step is held to, the appended keys to
2e-2 (bf16 rounding of slightly different fp32 values)."""

import pytest
import torch

from exl3_b200 import _lib, ops
from exl3_b200.harness import DecodeModel, DecoderConfig
from exl3_b200.verify import VerifyConfig, VerifyModel

pytestmark = pytest.mark.gpu

CFG = DecoderConfig(layers=2, hidden=512, heads=16, kv_heads=4, head_dim=128, inter=1024, vocab=1024, K=4, cb=0)


def _tame(m):
    for L in m.layers:
        for lin in L["qkv"] + [L["o"]] + L["gu"] + [L["down"]]:
            lin[2].mul_(float(lin[0].size(0) * 16) ** -0.5)
    return m


def _rel(a, b):
    return ((a.float() - b.float()).abs().max() / b.float().abs().max()).item()


def _paged(batch, max_ctx, dev, **kw):
    return _tame(DecodeModel(CFG, batch=batch, max_ctx=max_ctx, device=dev, paged=True, **kw))


def _copy_cache(dst, src, lens):
    """Dense [layer, B, heads, ctx, dim] caches into a paged model's pages."""
    ps = dst.page_size
    for d, s in ((dst.k_cache, src.k_cache), (dst.v_cache, src.v_cache)):
        for b, n in enumerate(lens):
            for p in range(n):
                d[:, int(dst.block_table[b, p // ps]), p % ps] = s[:, b, :, p].to(d.dtype)


@pytest.mark.parametrize("batch,ctx,page_size", [(1, 0, 16), (3, 70, 16), (2, 127, 24), (20, 65, 64)])
def test_paged_step_matches_dense(cuda_device, batch, ctx, page_size):
    tokens = torch.arange(batch, device=cuda_device) * 7 + 3
    ref = _tame(DecodeModel(CFG, batch=batch, max_ctx=160, device=cuda_device, fused=False))
    ref.fill_random_kv(ctx)
    m = _paged(batch, 160, cuda_device, page_size=page_size)
    _copy_cache(m, ref, [ctx] * batch)
    m.pos.fill_(ctx)
    for x in (ref, m):
        x.tokens.copy_(tokens)
        x.step()
    assert _rel(m.h, ref.h) < 1e-2
    for li in range(CFG.layers):
        page, off = m.block_table[:, ctx // page_size].long(), ctx % page_size
        assert _rel(m.k_cache[li, page, off], ref.k_cache[li, :, :, ctx]) < 2e-2
        assert _rel(m.v_cache[li, page, off], ref.v_cache[li, :, :, ctx]) < 2e-2
    assert m.pos.tolist() == [ctx + 1] * batch and ops.device_status(cuda_device) == 0


@pytest.mark.parametrize("kv_dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_ragged_batch_matches_single_sequences(cuda_device, kv_dtype):
    """Five sequences of different lengths in one captured step, against each alone."""
    lens = [0, 5, 64, 130, 199]
    many = _paged(5, 256, cuda_device, page_size=16, kv_dtype=kv_dtype, logprobs=3)
    many.fill_random_kv(lens)
    tokens = torch.tensor([3, 10, 17, 24, 31])
    k0, v0 = many.k_cache.clone(), many.v_cache.clone()
    many.tokens.copy_(tokens)
    many.capture()
    many.k_cache.copy_(k0)
    many.v_cache.copy_(v0)
    many.graph.replay()
    torch.cuda.synchronize()
    assert many.pos.tolist() == [n + 1 for n in lens]
    for b, n in enumerate(lens):
        one = _paged(1, 256, cuda_device, page_size=16, kv_dtype=kv_dtype)
        pages = many.block_table[b].long()
        one.k_cache[:, one.block_table[0].long()] = k0[:, pages] if kv_dtype != torch.float8_e4m3fn else k0.view(torch.uint8)[:, pages].view(kv_dtype)
        one.v_cache[:, one.block_table[0].long()] = v0[:, pages] if kv_dtype != torch.float8_e4m3fn else v0.view(torch.uint8)[:, pages].view(kv_dtype)
        one.pos.fill_(n)
        one.tokens.copy_(tokens[b:b + 1])
        one.step()
        assert _rel(many.h[b], one.h[0]) < 1e-2, b
    many.release()


def test_generate_reports_logprobs(cuda_device):
    m = _paged(2, 128, cuda_device, page_size=16, logprobs=4)
    m.fill_random_kv([40, 9])
    m.capture()
    tokens, lp = m.generate(torch.tensor([5, 6]), 6)
    assert tokens.shape == (2, 6) and lp.logprob.shape == (2, 6) and lp.top_ids.shape == (2, 6, 4)
    # greedy: the token is the most likely one (equal bf16 logits: the lower id first, as argmax)
    assert torch.equal(lp.top_logprobs[:, :, 0], lp.logprob)
    last = torch.log_softmax(m.last_logits.double(), -1).cpu()
    assert (lp.logprob[:, -1].double() - last.amax(-1)).abs().max() < 1e-5
    assert (lp.entropy[:, -1].double() + (last.exp() * last).sum(-1)).abs().max() < 1e-4
    plain = _paged(2, 128, cuda_device, page_size=16)
    plain.fill_random_kv([40, 9])
    plain.capture()
    assert plain.generate(torch.tensor([5, 6]), 6).shape == (2, 6)
    # past the cache's end: an error from the device status, not a wrong token
    m.pos.fill_(128)
    with pytest.raises(RuntimeError, match="bad argument"):
        m.generate(torch.tensor([5, 6]), 1)
    assert ops.device_status(cuda_device) == _lib.EBADARG
    m.release()
    plain.release()


def test_paged_model_refusals(cuda_device):
    for kw in (dict(paged=True, fused=True), dict(kv_dtype=torch.float8_e4m3fn), dict(paged=True, kv_dtype=torch.float16)):
        with pytest.raises(ValueError):
            DecodeModel(CFG, batch=1, max_ctx=64, device=cuda_device, **kw)
    m = _paged(2, 64, cuda_device)
    with pytest.raises(ValueError):
        m.fill_random_kv([10, 65])


def test_verify_draft_logprobs(cuda_device):
    cfg = VerifyConfig(layers=1, hidden=512, heads=8, kv_heads=2, experts=8, topk=2, inter=256, vocab=1024)
    m = VerifyModel(cfg, batch=2, max_ctx=64, device=cuda_device)
    m.fill_random_kv(20)
    with pytest.raises(RuntimeError):
        m.draft_logprobs()
    m.tokens.copy_(torch.randint(0, cfg.vocab, (2, 5), device=cuda_device))
    m.logits = m.step()
    got = m.draft_logprobs(top=3)
    ref = torch.log_softmax(m.logits.double(), -1).view(2, 5, -1)
    want = torch.gather(ref[:, :-1], 2, m.tokens[:, 1:, None])[..., 0]
    lp = got.logprob.view(2, 5)
    assert (lp[:, :-1].double() - want).abs().max() < 1e-5 and (lp[:, -1] == -float("inf")).all()
    assert torch.equal(got.top_ids.view(2, 5, 3)[..., 0], m.logits.argmax(-1).view(2, 5))
    m.close()
