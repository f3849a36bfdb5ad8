"""Paged-cache operators at the edges of what their documentation allows, against the definitions
of test_paged_gpu (whose tolerances hold here, except where a test derives its own)."""

import math
import threading

import pytest
import torch

from exl3_b200 import decode, ops, paged
from exl3_b200.harness import DecodeModel, DecoderConfig
from test_paged_gpu import BF16, E4M3, FP16, attention_oracle, build, half_step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens,heads,hk,dim,R,cap", [
    ([1000, 129, 40, 2], 16, 2, 128, 1, 0.0),
    ([2000, 513], 32, 4, 128, 5, 0.0),
    ([1500, 31], 24, 1, 64, 1, 0.0),
    ([700, 90], 8, 2, 64, 2, 20.0),
])
def test_e4m3_weights_keep_their_bits(cuda_device, lens, heads, hk, dim, R, cap):
    """An e4m3 cache under bf16 queries carries its softmax weights as exactly as the other types:
    before its rounding an output is off by (2 delta + 2^-15) max|v| at most, delta the scores'
    error.  What is typical: with values of random signs an output and its error are both sums of
    w_i v_i, the error's terms times a weight's relative error, so that e is about that error times
    |o|.  bf16's spacing is at least 2^-8 |o|; an error e rounds to another value with a chance of
    e / spacing.  Pairs of fp16 (2^-22) with fp32 scores of order 1 (2^-21 from 128 products) and
    fp32 sums make e about 2^-20 |o|, a share of 2^-12 of the outputs; single fp16 weights (an rms of
    2^-12.3) make it 2^-4.3 = 1/20.  The test draws the line between the two, at 1/64."""
    q, k, v, table, n, (ks, vs) = build(lens, heads, hk, dim, BF16, E4M3, 16, R, cuda_device, seed=dim + R)
    q = (q.float() / 8).to(BF16)  # scores of order 1: many weights take part
    ref, rlse, vmax, smax = attention_oracle(q, k, v, table, lens, R, dim ** -0.5, cap, 0, ks, vs)
    out = paged.attention(q, k, v, table, n, rows_per_seq=R, softcap=cap, k_scale=ks, v_scale=vs)
    delta = dim * 2.0 ** -24 * smax
    err = (out.double().cpu() - ref).abs()
    assert (err <= (2 * delta + 2.0 ** -15) * vmax + half_step(BF16) * ref.abs()).all()
    flips = (out.cpu() != ref.to(BF16)).double().mean()
    assert float(flips) < 1 / 64, float(flips)
    assert ops.device_status(cuda_device) == 0


def test_expanded_outputs_are_refused(cuda_device):
    """Several CTAs would write one address; inputs may be expanded."""
    lens, heads, hk, dim = [20, 30], 4, 2, 64
    q, k, v, table, n, _ = build(lens, heads, hk, dim, BF16, BF16, 16, 1, cuda_device)
    slots = torch.tensor([-1, -1], device=cuda_device)
    new = torch.zeros(1, hk, dim, dtype=BF16, device=cuda_device).expand(2, -1, -1)
    inv = torch.ones(dim // 2, device=cuda_device)
    for bad in (q[:1].expand(2, -1, -1), q[:, :1].expand(-1, heads, -1), q[:1, :1].expand(2, heads, -1)):
        with pytest.raises(RuntimeError, match="EBADSHAPE"):
            paged.attention(q, k, v, table, n, out=bad)
        with pytest.raises(RuntimeError, match="EBADSHAPE"):
            paged.rope_append(q, new, new, k, v, slots, slots, inv, q_out=bad)
    one = q[:1].expand(2, -1, -1)
    got = paged.attention(one, k, v, table, n)
    assert torch.equal(got, paged.attention(one.contiguous(), k, v, table, n))
    assert torch.equal(paged.rope_append(one, new, new, k, v, slots, slots, inv)[1],
                       paged.rope_append(q[:1], new[:1], new[:1], k, v, slots[:1], slots[:1], inv)[0])


def test_calls_from_several_threads(cuda_device):
    """Threads that call at once, each on a stream of its own, the first call of every kernel among
    them, get what a single thread gets."""
    jobs = []
    for heads, hk, dim, qt, ct in ((20, 1, 64, FP16, FP16), (8, 8, 64, BF16, E4M3), (18, 2, 128, FP16, E4M3), (34, 2, 128, FP16, FP16)):
        q, k, v, table, n, (ks, vs) = build([300, 77, 1], heads, hk, dim, qt, ct, 16, 1, cuda_device)
        jobs.append(dict(q=q, k_cache=k, v_cache=v, block_table=table, seq_lens=n, k_scale=ks, v_scale=vs))
    torch.cuda.synchronize()
    start, got, wrong = threading.Barrier(8), [None] * 8, []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                start.wait()
                for _ in range(20):
                    got[i] = paged.attention(**jobs[i % 4])
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # the main thread raises it
            wrong.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong
    for i in range(8):
        assert torch.equal(got[i], paged.attention(**jobs[i % 4])), i


def test_prompt_appended_to_a_dense_cache(cuda_device):
    """A prompt goes through a paged view into the dense cache of the fused decode sub-layer, which is
    called right behind it: it attends to the new rows.  (The sub-layer requests rows of earlier
    positions before its dependency wait.)  Against the same calls with a wait between; the matmuls'
    sums may add in another order, so the residual streams agree to 1e-3, and to no such thing
    with the cache as it was before."""
    dev, ctx, hk = cuda_device, 700, 2
    cfg = DecoderConfig(layers=1, hidden=512, heads=16, kv_heads=hk, head_dim=128, inter=1024, vocab=1024, K=4, cb=0)
    m = DecodeModel(cfg, batch=1, max_ctx=1024, device=dev, fused=True)
    for lin in m.layers[0]["qkv"] + [m.layers[0]["o"]]:
        lin[2].mul_(float(lin[0].size(0) * 16) ** -0.5)
    kc, vc = m.k_cache[0], m.v_cache[0]  # [1, hk, 1024, 128]
    pages = [t.permute(0, 2, 1, 3) for t in (kc, vc)]
    gen = torch.Generator(device=dev)
    gen.manual_seed(8)
    q, k, v = (torch.randn(ctx, n, 128, generator=gen, device=dev).to(BF16) for n in (16, hk, hk))
    at = torch.arange(ctx, device=dev)
    pos = torch.full((), ctx, device=dev)
    h0 = torch.randn(1, 512, generator=gen, device=dev)
    L = m.layers[0]

    def run(wait, append=True):
        kc.zero_(), vc.fill_(3.0)
        h, ss = h0.clone(), torch.zeros(2, 1, device=dev)
        torch.sum(h * h, dim=-1, out=ss[0])
        torch.cuda.synchronize()
        if append:
            paged.rope_append(q, k, v, *pages, at, at, m.inv_freq)
        if wait:
            torch.cuda.synchronize()
        decode.decode_attention(h, ss[0], ss[1], L["ln1"], cfg.eps, L["qkv"], L["o"], cfg.K, cfg.cb, kc, vc, pos, m.inv_freq)
        return h

    want, before = run(True), run(True, append=False)
    rel = lambda a, b: float((a - b).norm() / b.norm())  # noqa: E731
    assert rel(before, want) > 1e-2
    for _ in range(20):
        assert rel(run(False), want) < 1e-3
    assert ops.device_status(dev) == 0


@pytest.mark.parametrize("scale,qscale", [(2.0 ** -100, 2.0 ** -60), (2.0 ** -120, 2.0 ** -40), (2.0 ** -126, 1.0),
                                          (2.0 ** 100, 2.0 ** 60)])
def test_scores_that_vanish_leave_the_mean(cuda_device, scale, qscale):
    """A scale and queries whose product leaves fp32's range, and scores that are 0 all the same (above
    it: with keys of 0): the answer is the mean of the values, masked positions (the last stage's, a
    later row's) as ever without weight."""
    lens, heads, hk, dim, R = [3, 130, 0], 8, 2, 128, 2
    for ct in (BF16, E4M3):
        q, k, v, table, n, (ks, vs) = build(lens, heads, hk, dim, BF16, ct, 16, R, cuda_device)
        q = (q.float() * qscale).to(BF16)
        if qscale > 1:
            k.view(torch.uint8).zero_()
        ref, rlse, vmax, _ = attention_oracle(q, k, v, table, lens, R, scale, 0.0, 0, ks, vs)
        out, lse = paged.attention(q, k, v, table, n, rows_per_seq=R, scale=scale, k_scale=ks, v_scale=vs, return_lse=True)
        err = (out.double().cpu() - ref).abs()
        assert (err <= 2.0 ** -15 * vmax + half_step(BF16) * ref.abs()).all()
        empty = rlse == -math.inf
        assert torch.equal(lse.cpu() == -math.inf, empty)
        assert ((lse.double().cpu() - rlse)[~empty].abs() <= 2.0 ** -20 * (1 + rlse[~empty].abs())).all()


@pytest.mark.parametrize("window", [2 ** 31 - 257, 2 ** 31 - 258, 2 ** 31 - 2049, 2 ** 31 - 2050, 2 ** 31 - 1])
def test_windows_near_two_to_the_31(cuda_device, window):
    """Positions that a table of 2^31 could hold, a window of nearly as many, and sequences far shorter
    than their rows: the window takes nothing away."""
    page, R, dim, lens = 2 ** 20, 400, 64, [10, 450]
    k, v = (torch.randn(1, page, 1, dim, device=cuda_device).to(BF16) for _ in range(2))
    table = torch.zeros(2, 2048, dtype=torch.int32, device=cuda_device)
    n = torch.tensor(lens, dtype=torch.int32, device=cuda_device)
    q = torch.randn(2 * R, 1, dim, device=cuda_device).to(BF16)
    out, lse = paged.attention(q, k, v, table, n, rows_per_seq=R, window=window, return_lse=True)
    small, sl = paged.attention(q, k, v, table[:, :1].contiguous(), n, rows_per_seq=R, return_lse=True)
    assert torch.equal(out, small) and torch.equal(lse, sl)
    assert torch.equal(torch.isinf(lse[:, 0]).cpu(), torch.arange(2 * R) < R - lens[0])
    assert ops.device_status(cuda_device) == 0


def test_strides_of_single_rows_do_not_count(cuda_device):
    """One token, or one head, in a buffer of an odd width: its rows begin on 16-byte boundaries all the
    same, and outputs there are written in place."""
    for tokens, heads in ((1, 4), (3, 1)):
        q, k, v, table, n, _ = build([40] * tokens, heads, 1, 64, BF16, BF16, 16, 1, cuda_device)
        want = paged.attention(q, k, v, table, n)
        if tokens == 1:
            room = torch.zeros(2, heads * 64 + 3, dtype=BF16, device=cuda_device)
            out, src = (t[:, :heads * 64].view(2, heads, 64)[:1] for t in (room, room + 0))
        else:
            room = torch.zeros(tokens, 67, 64, dtype=BF16, device=cuda_device)
            out, src = (t.as_strided((tokens, 1, 64), (67 * 64, 67, 1)) for t in (room, room + 0))
        src.copy_(q)
        assert (out.stride(0) | out.stride(1)) % 8
        got = paged.attention(src, k, v, table, n, out=out)
        assert got.data_ptr() == room.data_ptr() and torch.equal(out, want)
        slots = torch.full((tokens,), -1, device=cuda_device)
        inv = torch.ones(32, device=cuda_device)
        kv = torch.zeros(tokens, 1, 64, dtype=BF16, device=cuda_device)
        want = paged.rope_append(q, kv, kv, k, v, slots + 8, slots, inv)
        out.zero_()
        assert torch.equal(paged.rope_append(src, kv, kv, k, v, slots + 8, slots, inv, q_out=out), want)
        assert int((room != 0).sum()) <= out.numel()
