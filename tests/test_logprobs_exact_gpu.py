"""token_logprobs where logits are excluded, far from 0, or both: against log_softmax in 64 bits.

Tolerance of a log-probability (base-2 distances d_i = (M - x_i) log2 e, p_i the probabilities,
D = sum p_i d_i).  A term's exponent is one fused multiply-add of the logit, the fp32 constant
log2 e (off by 2^-26 of its size) and a thread's reference, and is rescaled by one more to the
row's maximum: off by (2.25 d_i + 32) 2^-24 with references at most 16 below what they meet, so
the terms' sum by ln 2 (2.25 D + 32) 2^-24.  ex2 is off by 2^-22, for the term, for the rescale
to the row's maximum, and for each raise of a thread's reference, whose distance of up to 32
carries 2^-24 too; two raises are counted.  The sum of n terms: two chains a thread (256 threads),
at most n / 512 + 16 additions deep, 2^-24 each.  The difference x - M and the result round by 2^-24 of their
sizes.  None of it grows with M itself.  Entropy: the same with each term weighted by its
distance, (1 + max over likely i of d_i) times as much."""

import math

import pytest
import torch

from exl3_b200 import logprobs as LP

pytestmark = pytest.mark.gpu


def check(x, tokens, top, got):
    xd = x.double().cpu()
    rows, n = xd.shape
    t = tokens.cpu()
    ref = torch.log_softmax(xd, dim=-1)
    p = ref.exp()
    m = xd.amax(-1, keepdim=True)
    d = torch.where(p > 0, (m - xd) * 1.4427, torch.zeros_like(xd))
    mean = (p * d).sum(-1)
    likely = torch.where(p > 1e-12, d, torch.zeros_like(d)).amax(-1)
    tol = (0.6932 * (2.25 * mean + 32) * 2.0 ** -24 + 4 * 2.0 ** -22 + 2 * 32 * 2.0 ** -24
           + (n / 512 + 16) * 2.0 ** -24)
    want = ref[torch.arange(rows), t]
    lp = got.logprob.double().cpu()
    out = want == -math.inf  # an excluded token
    assert torch.equal(lp == -math.inf, out) and torch.isfinite(lp[~out]).all()
    assert ((lp - want)[~out].abs() <= (tol + 2.0 ** -23 * (1 + want.abs()))[~out]).all(), float((lp - want)[~out].abs().max())
    ent = -torch.where(p > 0, p * ref, torch.zeros_like(p)).sum(-1)
    assert ((got.entropy.double().cpu() - ent).abs() <= (1 + likely) * tol + 2.0 ** -23 * ent).all()
    order = torch.sort(xd, dim=-1, descending=True, stable=True).indices[:, :top]  # ties: lower id first
    assert torch.equal(got.top_ids.cpu(), order)
    want = torch.gather(ref, 1, order)
    have = got.top_logprobs.double().cpu()
    out = want == -math.inf
    assert torch.equal(have == -math.inf, out)
    err = torch.where(out, torch.zeros_like(want), (have - want).abs())
    assert (err <= tol[:, None] + 2.0 ** -23 * (1 + torch.where(out, torch.zeros_like(want), want.abs()))).all()


MASKS = {
    "prefix": lambda i, n: i < n - 700,                  # whole groups of a thread before the first real logit
    "first-half": lambda i, n: i < n // 2,
    "tail": lambda i, n: i >= 700,
    "one-left": lambda i, n: i != n - 3,
    "one-left-first": lambda i, n: i != 0,
    "few-left": lambda i, n: i % 2003 != 7,              # as a top-k filter leaves a row
    "stripes": lambda i, n: (i // 8192) % 2 == 0,        # groups of excluded and of real logits in turn
    "every-other": lambda i, n: i % 2 == 0,
}


@pytest.mark.parametrize("rows", [2, 400])  # a cluster of CTAs a row, one CTA a row
@pytest.mark.parametrize("mask", sorted(MASKS))
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_excluded_tokens(cuda_device, dtype, mask, rows):
    """-inf logits are excluded tokens wherever they stand in a row."""
    n, top = 70001, 8
    g = torch.Generator(device=cuda_device)
    g.manual_seed(7)
    i = torch.arange(n, device=cuda_device)
    x = (torch.randn(2, n, generator=g, device=cuda_device) * 3).to(dtype)
    x[:, MASKS[mask](i, n)] = -math.inf
    tokens = torch.stack([x[0].argmax(), torch.full((), 4 if mask != "every-other" else 2, device=cuda_device)])
    many = x.repeat(rows // 2, 1)
    got = LP.token_logprobs(many, tokens.repeat(rows // 2), top)
    some = min(rows, 16)  # rows of an odd length begin at every alignment
    check(many[:some], tokens.repeat(some // 2), top, LP.TokenLogprobs(*(t[:some] for t in got)))
    assert torch.equal(got.top_ids, got.top_ids[:2].repeat(rows // 2, 1))
    bare = LP.token_logprobs(many, tokens.repeat(rows // 2))
    assert torch.equal(bare.logprob, got.logprob) and torch.equal(bare.entropy, got.entropy)


@pytest.mark.parametrize("kind", ["lowest", "mostly-lowest", "lowest-and-excluded", "all-far-down"])
@pytest.mark.parametrize("rows", [1, 500])
def test_fp16_rows_near_the_types_lowest_value(cuda_device, kind, rows):
    """fp16 masks of the type's lowest value beside -inf, whose exponents stand in for each other."""
    n = 40003
    i = torch.arange(n, device=cuda_device)
    low = torch.finfo(torch.float16).min
    x = {"lowest": lambda: torch.full((n,), low, device=cuda_device),
         "mostly-lowest": lambda: torch.where(i % 7777 == 3, torch.sin(i.float()), torch.full((), low, device=cuda_device)),
         "lowest-and-excluded": lambda: torch.where(i < 30000, torch.full((), -math.inf, device=cuda_device),
                                                    torch.full((), low, device=cuda_device)),
         "all-far-down": lambda: torch.where(i < 20000, torch.full((), -math.inf, device=cuda_device),
                                             -4e4 - 32.0 * (i % 3))}[kind]()
    x = x.to(torch.float16).expand(rows, n).contiguous()
    tokens = torch.full((rows,), 30005, device=cuda_device)
    got = LP.token_logprobs(x, tokens, 5)
    check(x[:1], tokens[:1], 5, LP.TokenLogprobs(*(t[:1] for t in got)))


def test_fp16_row_of_excluded_tokens_alone(cuda_device):
    """Nothing left: NaN for that row, as in the other types, and no other row's concern."""
    x = torch.zeros(3, 30000, dtype=torch.float16, device=cuda_device)
    x[1] = -math.inf
    tokens = torch.zeros(3, dtype=torch.int64, device=cuda_device)
    got = LP.token_logprobs(x, tokens, 4)
    assert torch.isnan(got.logprob[1]) and torch.isnan(got.entropy[1]) and torch.isnan(got.top_logprobs[1]).all()
    assert torch.equal(got.top_ids.cpu(), torch.arange(4).expand(3, 4))
    assert (got.logprob[::2] + math.log(30000)).abs().max() < 1e-5


@pytest.mark.parametrize("rows", [5, 600])
@pytest.mark.parametrize("offset,dtype", [(0, torch.float32), (300, torch.float32), (3000, torch.float32), (-3000, torch.float32),
                                          (30000, torch.float32), (1e6, torch.float32), (300, torch.bfloat16), (300, torch.float16),
                                          (-2000, torch.float16)])
def test_a_common_offset_costs_no_accuracy(cuda_device, offset, dtype, rows):
    n = 20001
    g = torch.Generator(device=cuda_device)
    g.manual_seed(3)
    x = (torch.randn(rows, n, generator=g, device=cuda_device) * 3 + offset).to(dtype)
    tokens = torch.randint(0, n, (rows,), generator=g, device=cuda_device)
    tokens[::2] = x[::2].argmax(-1)
    check(x, tokens, 5, LP.token_logprobs(x, tokens, 5))


def test_entropy_is_as_near_as_the_plain_form(cuda_device):
    """Rows as a language model has them, a wide body and a few tokens far above: the entropies' root
    mean square error is at most sqrt(250 / 17) = 3.8 times that of the same sums in fp32 torch, whose
    trees are about 17 additions deep where a thread's chain here has 250; all other roundings are the
    same few."""
    rows, n = 700, 128256
    g = torch.Generator(device=cuda_device)
    g.manual_seed(12)
    x = torch.randn(rows, n, generator=g, device=cuda_device) * 2
    peak = torch.randint(0, n, (rows, 8), generator=g, device=cuda_device)
    x.scatter_add_(1, peak, torch.rand(rows, 8, generator=g, device=cuda_device) * 14)
    x = x.to(torch.bfloat16)

    def entropy(t):
        y = t - t.amax(-1, keepdim=True)
        e = torch.exp(y)
        total = e.sum(-1)
        return (torch.log(total) - (e * y).sum(-1) / total).double()

    want = torch.cat([entropy(part.double()) for part in x.split(50)])
    rms = lambda t: float((t.double() - want).pow(2).mean().sqrt())  # noqa: E731
    assert rms(LP.token_logprobs(x, peak[:, 0].contiguous()).entropy) <= 3.8 * rms(entropy(x.float()))
