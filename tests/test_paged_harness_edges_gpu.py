"""The paged model and the verify model at the ends of their caches and between streams."""

import dataclasses

import pytest
import torch

from exl3_b200 import ops
from exl3_b200.verify import CONFIG5, VerifyModel
from test_paged_harness_gpu import _paged

pytestmark = pytest.mark.gpu


def test_draft_logprobs_follow_the_replayed_step(cuda_device):
    """replay() and draft_logprobs() one after the other without a wait between: the report is of the
    step just replayed, and the step replayed next leaves it alone.  Tolerance: fp32 logits of size
    S give log-probabilities off by far less than 1e-5 (1 + S)."""
    cfg = dataclasses.replace(CONFIG5, layers=6, hidden=1024, heads=8, kv_heads=2, experts=16, inter=512, vocab=32000)
    m = VerifyModel(cfg, 2, 64 + cfg.rows_per_seq, cuda_device)
    m.fill_random_kv(64)
    m.capture()
    torch.cuda.synchronize()
    drafts = [torch.randint(0, cfg.vocab, m.tokens.shape, generator=torch.Generator().manual_seed(k)).to(cuda_device)
              for k in range(4)]
    reports, snaps = [], []
    for k, draft in enumerate(drafts):
        with torch.cuda.stream(m.stream):
            m.tokens.copy_(draft)
        m.replay(3)
        reports.append(m.draft_logprobs(top=2))
        with torch.cuda.stream(m.stream):  # the logits that the report is of, as the stream has them
            snaps.append(m.logits.clone())
    torch.cuda.synchronize()
    for draft, got, logits in zip(drafts, reports, snaps):
        ref = torch.log_softmax(logits.double(), -1).view(2, cfg.rows_per_seq, -1)
        want = torch.gather(ref[:, :-1], 2, draft[:, 1:, None])[..., 0]
        lp = got.logprob.view(2, cfg.rows_per_seq)
        tol = 1e-5 * (1 + float(logits.abs().max()))
        assert (lp[:, :-1].double() - want).abs().max() < tol and (lp[:, -1] == -float("inf")).all()
        assert torch.equal(got.top_ids.view(2, cfg.rows_per_seq, 2)[..., 0], logits.argmax(-1).view(2, -1))
    assert not torch.equal(reports[0].logprob, reports[1].logprob)
    # on the model's own stream, and captured into a graph of the caller's
    with torch.cuda.stream(m.stream):
        own = m.draft_logprobs(top=2)
    torch.cuda.synchronize()
    assert torch.equal(own.logprob, reports[-1].logprob)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        held = m.draft_logprobs(top=2)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(held.logprob, own.logprob) and torch.equal(held.top_ids, own.top_ids)
    del g
    m.close()


def test_capture_with_one_position_left(cuda_device):
    """Capturing warms up without leaving the pages: a sequence with a single position left is
    captured and generates its last token."""
    m = _paged(3, 64, cuda_device, page_size=16, logprobs=2)
    m.fill_random_kv([63, 5, 40])
    before = m.k_cache.clone()
    m.tokens.copy_(torch.tensor([9, 8, 7]))
    m.capture()
    assert ops.device_status(cuda_device) == 0
    assert m.pos.tolist() == [63, 5, 40] and m.tokens.tolist() == [9, 8, 7]
    for b, n in enumerate([63, 5, 40]):  # what the sequences hold is as it was
        for p in range(n):
            page = int(m.block_table[b, p // 16])
            assert torch.equal(m.k_cache[:, page, p % 16], before[:, page, p % 16])
    tokens, lp = m.generate(torch.tensor([5, 6, 4]), 1)
    assert tokens.shape == (3, 1) and torch.isfinite(lp.logprob).all() and m.pos.tolist() == [64, 6, 41]
    assert ops.device_status(cuda_device) == 0
    m.release()


def test_generate_reports_its_own_steps(cuda_device):
    """A step outside the graph between capture() and generate() leaves generate's report its own:
    of the tokens generated, from the logits of the captured step."""
    m = _paged(2, 128, cuda_device, page_size=16, logprobs=3)
    m.fill_random_kv([40, 9])
    pos = m.pos.clone()
    m.capture()
    m.tokens.copy_(torch.tensor([700, 800]))
    m.step()  # eager, of other tokens
    eager = m.logprobs
    m.pos.copy_(pos)
    torch.cuda.synchronize()
    tokens, lp = m.generate(torch.tensor([5, 6]), 4)
    assert m.logprobs is not eager
    assert torch.equal(lp.top_ids[..., 0], tokens)  # greedy (equal logits: the lower id first, as argmax)
    last = torch.log_softmax(m.last_logits.double(), -1).cpu()
    assert (lp.logprob[:, -1].double() - last.amax(-1)).abs().max() < 1e-5
    assert all(len(set(row)) > 1 for row in lp.logprob.tolist())
    m.release()
