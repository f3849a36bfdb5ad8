"""token_logprobs against log_softmax in 64 bits.

Tolerance: exponents y = x log2 e - M2 are fp32 (off by 2^-24 of their size, |y| <= Y), the
exponential by 2^-22 and a sum of n terms in a tree of depth d by d 2^-24 (threads add up to
n / 256 terms in a row, so d <= n / 256 + 8, but errors of either sign: 2^-24 sqrt of that is
typical, and the bound is taken): log S is off by about Y 2^-24 + 2^-22 + d 2^-24, a
log-probability by that and 2^-23 of its size; the entropy by the same times (1 + Y)."""

import math

import pytest
import torch

from exl3_b200 import logprobs as LP

pytestmark = pytest.mark.gpu


def check(x, tokens, top, got):
    ref = torch.log_softmax(x.double().cpu(), dim=-1)
    rows, n = x.shape
    xd = x.double().cpu()
    m = xd.amax(-1, keepdim=True)
    p = ref.exp()
    y = float(torch.where(p > 1e-12, (m - xd), torch.zeros_like(xd)).max()) * 1.4427 + 1
    size = float(m.abs().max()) * 1.4427 + y
    tol = size * 2.0 ** -24 + 2.0 ** -22 + (n / 256 / 148 + n / 256 + 8) * 2.0 ** -24
    t = tokens.cpu()
    valid = (t >= 0) & (t < n)
    want = torch.full((rows,), -math.inf, dtype=torch.float64)
    want[valid] = ref[torch.arange(rows)[valid], t[valid]]
    lp = got.logprob.double().cpu()
    fin = torch.isfinite(want)
    assert torch.equal(torch.isfinite(lp), fin) and (lp[~fin] == -math.inf).all()
    assert ((lp - want)[fin].abs() <= tol + 2.0 ** -23 * want[fin].abs()).all()
    ent = -torch.where(p > 0, p * ref, torch.zeros_like(p)).sum(-1)
    assert ((got.entropy.double().cpu() - ent).abs() <= (1 + y) * tol + 2.0 ** -23 * ent).all()
    if not top:
        assert got.top_ids is None and got.top_logprobs is None
        return
    order = torch.sort(xd, dim=-1, descending=True, stable=True).indices[:, :top]  # ties: lower id first
    assert torch.equal(got.top_ids.cpu(), order)
    want = torch.gather(ref, 1, order)
    have = got.top_logprobs.double().cpu()
    fin = torch.isfinite(want)
    assert torch.equal(have[~fin], want[~fin])
    assert ((have - want)[fin].abs() <= tol + 2.0 ** -23 * want[fin].abs()).all()


def logits(rows, n, dtype, dev, seed=0, spread=3.0):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    return (torch.randn(rows, n, generator=g, device=dev) * spread).to(dtype)


@pytest.mark.parametrize("rows,n,dtype,top", [
    (1, 1, torch.float32, 1), (3, 2, torch.bfloat16, 2), (2, 7, torch.float16, 7), (5, 31, torch.float32, 20),
    (4, 255, torch.bfloat16, 32), (3, 2047, torch.float16, 5), (3, 2048, torch.float16, 5), (3, 2049, torch.bfloat16, 32),
    (1, 128256, torch.bfloat16, 5), (7, 32003, torch.bfloat16, 20), (80, 50257, torch.float32, 20),
    (1, 151936, torch.float32, 32), (300, 4099, torch.float16, 3), (700, 2500, torch.bfloat16, 1), (2, 100001, torch.float16, 0),
    (1200, 1000, torch.float32, 32)])
def test_matches_log_softmax(cuda_device, rows, n, dtype, top):
    x = logits(rows, n, dtype, cuda_device, seed=n)
    tokens = torch.randint(0, n, (rows,), device=cuda_device)
    tokens[0] = n - 1
    if rows > 2:
        tokens[1], tokens[2] = -1, n
    got = LP.token_logprobs(x, tokens, top)
    check(x, tokens, top, got)
    again = LP.token_logprobs(x, tokens, top)
    assert all(a is None or torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("kind", ["equal", "ascending", "descending", "one-column", "few-finite", "large-offset", "zeros",
                                  "lowest", "mostly-lowest", "peaked"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_hard_rows(cuda_device, kind, dtype):
    """Ties, orders in which one thread or one vector holds all the large elements, masks."""
    n, top = 70001, 32
    dev = cuda_device
    i = torch.arange(n, device=dev)
    low = torch.finfo(dtype).min
    x = {"equal": lambda: torch.full((n,), 1.5, device=dev),
         "ascending": lambda: i.float() / 4000,
         "descending": lambda: -i.float() / 4000,
         "one-column": lambda: torch.where((i // 8) % 256 == 37, 5.0 + (i % 1000) / 1000.0, torch.zeros((), device=dev)),
         "few-finite": lambda: torch.where(i % 9001 == 5, i / 1e4, torch.full((), -math.inf, device=dev)),
         "large-offset": lambda: 3000.0 + torch.sin(i.float()),
         "zeros": lambda: torch.where(i % 2 == 0, -0.0, 0.0),
         "lowest": lambda: torch.full((n,), low, device=dev),
         "mostly-lowest": lambda: torch.where(i % 7777 == 3, torch.sin(i.float()), torch.full((), low, device=dev)),
         "peaked": lambda: torch.where(i == 12345, 40.0, torch.zeros((), device=dev))}[kind]()
    x = x.to(dtype).expand(3, n).contiguous()
    tokens = torch.tensor([0, 12345, n - 1], device=dev)
    check(x, tokens, top, LP.token_logprobs(x, tokens, top))
    # few rows are cut over many CTAs, many rows over few: the same answer
    many = x[:1].expand(400, n).contiguous()
    got = LP.token_logprobs(many, tokens[1:2].expand(400), top)
    check(many[:2], tokens[1:2].expand(2), top, LP.TokenLogprobs(*(t[:2] for t in got)))
    for t in got:
        assert t.dtype == torch.int64 and torch.equal(t, t[:1].expand_as(t)) or t.dtype != torch.int64


def test_rows_without_an_answer(cuda_device):
    """All -inf, a NaN, an infinity: NaN for that row, ids inside the vocabulary, other rows untouched."""
    x = logits(5, 5000, torch.float32, cuda_device)
    clean = x.clone()
    x[1] = -math.inf
    x[2, 77] = float("nan")
    x[3] = float("nan")
    x[4, 1234] = math.inf
    tokens = torch.tensor([3, 3, 3, 3, 3], device=cuda_device)
    got = LP.token_logprobs(x, tokens, 8)
    check(clean[:1], tokens[:1], 8, LP.TokenLogprobs(*(t[:1] for t in got)))
    for t in got[:3]:
        assert torch.isnan(t[1:4]).all()
    assert torch.isnan(got.logprob[4]) and torch.isnan(got.entropy[4])
    assert ((got.top_ids >= 0) & (got.top_ids < 5000)).all()
    assert torch.equal(got.top_ids[1].cpu(), torch.arange(8)) and int(got.top_ids[4, 0]) == 1234
    assert all(len(set(r)) == 8 for r in got.top_ids.tolist())
    one = LP.token_logprobs(x, tokens, 1)
    assert ((one.top_ids >= 0) & (one.top_ids < 5000)).all() and int(one.top_ids[1, 0]) == 0
    assert int(one.top_ids[0, 0]) == int(got.top_ids[0, 0]) and torch.equal(one.logprob[:1], got.logprob[:1])


def test_strided_rows_streams_and_graphs(cuda_device):
    wide = logits(9, 33001, torch.bfloat16, cuda_device, seed=4)
    x = wide[:, 3:32503]  # rows that begin anywhere
    tokens = torch.randint(0, x.size(1), (9,), device=cuda_device)
    check(x, tokens, 10, LP.token_logprobs(x, tokens, 10))
    check(x.t().contiguous().t(), tokens, 10, LP.token_logprobs(x.t().contiguous().t(), tokens, 10))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graphs = []
    y = x.clone()
    for src in (x, y):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            graphs.append((g, src, LP.token_logprobs(src, tokens, 10)))
    for k in range(3):
        y.copy_(logits(9, x.size(1), torch.bfloat16, cuda_device, seed=10 + k))
        torch.cuda.synchronize()
        for (g, _, _), st in zip(graphs, (torch.cuda.Stream(), torch.cuda.Stream())):
            with torch.cuda.stream(st):
                for _ in range(4):
                    g.replay()
        torch.cuda.synchronize()
        for _, src, got in graphs:
            check(src, tokens, 10, got)
    with torch.cuda.stream(s):
        side = LP.token_logprobs(x, tokens, 10)
    torch.cuda.synchronize()
    assert torch.equal(side.top_ids, graphs[0][2].top_ids) and torch.equal(side.logprob, graphs[0][2].logprob)
    none = LP.token_logprobs(x[:0], tokens[:0], 4)
    assert none.logprob.shape == (0,) and none.top_ids.shape == (0, 4)
    del graphs


def test_python_refusals(cuda_device):
    x, t = torch.zeros(2, 100, device=cuda_device), torch.zeros(2, dtype=torch.int64, device=cuda_device)
    for bad in (dict(logits=x.double()), dict(logits=x[0]), dict(tokens=t.int()), dict(tokens=t[:1]), dict(top=33),
                dict(top=-1), dict(logits=x[:, :5], top=6), dict(tokens=t.cpu()), dict(logits=x.cpu()), dict(logits=x[:, :0])):
        with pytest.raises(RuntimeError):
            LP.token_logprobs(**{**dict(logits=x, tokens=t, top=5), **bad})
