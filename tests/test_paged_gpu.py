"""Paged-cache operators (exl3_b200.paged) against their definitions in 64 bits.

Tolerances, from the formats and the arithmetic:
* a result rounded once to a type with machine epsilon e is off by e/2 of its value (e4m3: 2^-4,
  half of a subnormal step, 2^-10, below its normal range);
* rotation: cos and sin are fp32 values of an angle that is exact to 2^-23 of a turn's half, so
  each of the two products is off by at most 2^-22 of its size beyond the rounding;
* attention: a score is an fp32 sum of D products, off by at most D * 2^-24 * sum |q k| * scale
  (delta); a weight is off by delta relative, as is the sum of the weights, and the weights' 16-bit
  pairs carry 2^-16 (an e4m3 cache under bf16 queries: single fp16 weights, 2^-11): the output is
  off by (2 delta + 2^-15, or 2^-11) max|v| beyond its rounding, the log-sum-exp by
  delta + 2^-20 (1 + |lse|).
"""

import math

import pytest
import torch

from exl3_b200 import _lib, ops, paged

pytestmark = pytest.mark.gpu

BF16, FP16, FP32, E4M3 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn


def half_step(t):
    return 2.0 ** -4 if t == E4M3 else torch.finfo(t).eps / 2


def make_cache(pages, page, hk, dim, dtype, gen, dev, layout="nhd"):
    """k and v pools full of values; layouts by strides."""
    shape = (pages, page, hk, dim) if layout == "nhd" else (pages, hk, page, dim)
    out = []
    for _ in range(2):
        t = torch.randn(shape, generator=gen, device=dev).to(FP16 if dtype == E4M3 else dtype)
        t = t.to(dtype) if dtype == E4M3 else t
        out.append(t if layout == "nhd" else t.permute(0, 2, 1, 3))
    return out


def poison(cache, keep):
    """NaN in every slot that `keep` (bool [pages, page]) leaves out."""
    bad = torch.full((), float("nan"), device=cache.device)
    if cache.dtype == E4M3:
        cache.view(torch.uint8)[~keep] = 0x7F  # e4m3's NaN
    else:
        cache[~keep] = bad.to(cache.dtype)


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

def attention_oracle(q, k_cache, v_cache, table, lens, R, scale, softcap, window, k_scale, v_scale):
    """float64, row by row; also max |v| and the largest scale * sum |q k|."""
    rows, heads, dim = q.shape
    page, hk = k_cache.size(1), k_cache.size(2)
    out = torch.zeros(rows, heads, dim, dtype=torch.float64)
    lse = torch.full((rows, heads), -math.inf, dtype=torch.float64)
    vmax, smax = 0.0, 0.0
    qd = q.double().cpu()
    for s, n in enumerate(lens):
        for j in range(R):
            end = n - R + 1 + j
            start = max(0, end - window) if window else 0
            if end <= start:
                continue
            pos = torch.arange(start, end)
            pg = table[s].cpu()[pos // page].long().to(k_cache.device)
            off = (pos % page).to(k_cache.device)
            k = k_cache[pg, off].double().cpu() if k_cache.dtype != E4M3 else k_cache.view(torch.uint8)[pg, off].view(E4M3).double().cpu()
            v = v_cache[pg, off].double().cpu() if v_cache.dtype != E4M3 else v_cache.view(torch.uint8)[pg, off].view(E4M3).double().cpu()
            if k_scale is not None:
                k = k * k_scale.double().cpu()[None, :, None]
                v = v * v_scale.double().cpu()[None, :, None]
            r = R * s + j
            qq = qd[r].view(hk, heads // hk, dim)
            sc = torch.einsum("hgd,nhd->hgn", qq, k) * scale
            smax = max(smax, float((torch.einsum("hgd,nhd->hgn", qq.abs(), k.abs()) * scale).max()))
            vmax = max(vmax, float(v.abs().max()))
            if softcap:
                sc = softcap * torch.tanh(sc / softcap)
            lse[r] = torch.logsumexp(sc, -1).reshape(-1)
            out[r] = torch.einsum("hgn,nhd->hgd", torch.softmax(sc, -1), v).reshape(heads, dim)
    return out, lse, vmax, smax


def build(lens, heads, hk, dim, qt, ct, page, R, dev, seed=0, layout="nhd", extra=3):
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    counts = [-(-n // page) for n in lens]
    pages = sum(counts) + extra
    k, v = make_cache(pages, page, hk, dim, ct, gen, dev, layout)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))
    table = torch.full((len(lens), max(1, max(counts))), -1, dtype=torch.int32)
    at = 0
    for s, c in enumerate(counts):
        table[s, :c] = order[at:at + c].int()
        at += c
    q = torch.randn(len(lens) * R, heads, dim, generator=gen, device=dev).mul_(2.0).to(qt)
    scales = [None, None]
    if ct == E4M3:
        scales = [torch.rand(hk, generator=gen, device=dev) * 0.5 + 0.25 for _ in range(2)]
    return q, k, v, table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev), scales


def check_attention(got, lse, ref, rlse, vmax, smax, dim, qt, ct=None):
    delta = dim * 2.0 ** -24 * smax
    weights = 2.0 ** -11 if (qt, ct) == (BF16, E4M3) else 2.0 ** -15
    tol = (2 * delta + weights) * vmax + half_step(qt) * ref.abs() + (2.0 ** -25 if qt == FP16 else 0.0)
    err = (got.double().cpu() - ref).abs()
    assert not torch.isnan(err).any()
    assert (err <= tol).all(), float((err - tol).max())
    if lse is not None:
        l = lse.double().cpu()
        empty = rlse == -math.inf
        assert torch.equal(l == -math.inf, empty)
        assert ((l - rlse)[~empty].abs() <= delta + 2.0 ** -20 * (1 + rlse[~empty].abs())).all()


CASES = [
    # lens, heads, kv_heads, dim, q, cache, page, rows, window, softcap
    ([1], 8, 1, 128, BF16, BF16, 16, 1, 0, 0.0),
    ([0, 1, 2, 0], 8, 8, 64, FP16, FP16, 1, 1, 0, 0.0),
    ([63, 64, 65, 15, 16, 17], 16, 2, 128, BF16, BF16, 16, 1, 0, 0.0),
    ([128, 129, 1000, 0, 5, 127], 28, 4, 128, FP16, FP16, 24, 1, 0, 0.0),
    ([700, 3, 511], 64, 8, 64, BF16, BF16, 64, 1, 0, 30.0),
    ([5000], 5, 1, 128, BF16, BF16, 128, 1, 0, 0.0),
    ([127, 128, 129, 31, 33, 0, 1], 32, 4, 128, BF16, E4M3, 64, 1, 0, 0.0),
    ([257, 600], 8, 2, 64, FP16, E4M3, 7, 1, 0, 50.0),
    ([300, 4, 65], 32, 4, 128, BF16, E4M3, 16, 5, 0, 0.0),   # 40 rows of a kv head: three warps
    ([300, 2, 64, 0], 16, 2, 128, FP16, FP16, 16, 3, 0, 0.0),  # 24 rows; a sequence shorter than its rows
    ([200, 70], 64, 8, 64, BF16, BF16, 32, 7, 0, 0.0),       # 56 rows: two blocks
    ([90], 32, 2, 128, BF16, BF16, 16, 13, 0, 0.0),          # 208 rows: five blocks
    ([1000, 64, 63, 1], 16, 2, 128, BF16, BF16, 16, 1, 1, 0.0),  # window of one: the row itself
    ([1000, 129, 40], 16, 2, 64, FP16, FP16, 16, 1, 100, 0.0),
    ([1000, 129, 40, 3], 16, 2, 128, BF16, E4M3, 24, 4, 65, 20.0),
    ([4097, 1, 2050, 33], 64, 8, 128, BF16, BF16, 16, 1, 2048, 0.0),
    ([300, 0, 3, 40], 16, 2, 128, BF16, BF16, 16, 5, 2 ** 31 - 1, 0.0),  # a window of everything
    ([300, 17], 16, 2, 64, FP16, FP16, 16, 1, 0, 1e5),       # a cap far above the scores: they stay as they are
    ([300, 17], 16, 2, 64, FP16, FP16, 16, 1, 0, 0.5),       # and far below
    ([1000, 200, 33], 24, 1, 128, BF16, E4M3, 16, 1, 0, 0.0),  # three tiles of rows
    ([1000, 200, 33], 24, 1, 64, FP16, FP16, 16, 1, 0, 30.0),
    ([17] * 130, 8, 4, 64, BF16, BF16, 16, 1, 0, 0.0),       # more sequences than threads of a CTA
    ([40] * 300, 16, 4, 128, FP16, FP16, 16, 1, 0, 0.0),     # more items than CTAs
]


@pytest.mark.parametrize("lens,heads,hk,dim,qt,ct,page,R,window,cap", CASES)
def test_attention_matches_definition(cuda_device, lens, heads, hk, dim, qt, ct, page, R, window, cap):
    """Every slot outside the visible positions holds NaN, unused table entries -1."""
    q, k, v, table, n, (ks, vs) = build(lens, heads, hk, dim, qt, ct, page, R, cuda_device, seed=len(lens) + dim)
    scale = dim ** -0.5
    ref = attention_oracle(q, k, v, table, lens, R, scale, cap, window, ks, vs)
    keep = torch.zeros(k.shape[:2], dtype=torch.bool, device=cuda_device)
    for s, ln in enumerate(lens):
        first = max(0, ln - R + 1 - window) if window else 0
        assert 0 <= first <= ln
        for p in range(first, ln):
            keep[int(table[s, p // page]), p % page] = True
        if window:  # pages wholly before the window may have been given back
            table[s, :first // page] = -1
    poison(k, keep)
    poison(v, keep)
    out, lse = paged.attention(q, k, v, table, n, rows_per_seq=R, softcap=cap, window=window, k_scale=ks, v_scale=vs,
                               return_lse=True)
    check_attention(out, lse, *ref, dim, qt, ct)
    again = paged.attention(q, k, v, table, n, rows_per_seq=R, softcap=cap, window=window, k_scale=ks, v_scale=vs)
    assert torch.equal(again, out)  # the same bits every time
    assert ops.device_status(cuda_device) == 0


@pytest.mark.parametrize("seqs", [20011, 50000])
def test_attention_many_short_sequences(cuda_device, seqs):
    """Far more sequences than a CTA keeps lengths of: a sequence of one token answers with its
    value exactly, an empty one with zeros, and a long one among them with the definition's."""
    gen = torch.Generator(device=cuda_device)
    gen.manual_seed(seqs)
    pages = seqs + 700
    k, v = make_cache(pages, 1, 1, 64, BF16, gen, cuda_device)
    table = torch.full((seqs, 600), -1, dtype=torch.int32, device=cuda_device)
    order = torch.randperm(pages, generator=gen, device=cuda_device).int()
    table[:, 0] = order[:seqs]
    table[7777, 1:] = order[seqs:seqs + 599]
    lens = torch.randint(0, 2, (seqs,), generator=gen, device=cuda_device, dtype=torch.int32)
    lens[7777] = 600
    q = torch.randn(seqs, 1, 64, generator=gen, device=cuda_device).to(BF16)
    out, lse = paged.attention(q, k, v, table, lens, return_lse=True)
    want = torch.where((lens > 0)[:, None], v[table[:, 0].long(), 0, 0], torch.zeros((), dtype=BF16, device=cuda_device))
    rest = torch.arange(seqs, device=cuda_device) != 7777
    assert torch.equal(out[rest, 0], want[rest])
    assert torch.equal(torch.isinf(lse[:, 0]), lens == 0)
    ref = attention_oracle(q[7777:7778], k, v, table[7777:7778], [600], 1, 0.125, 0.0, 0, None, None)
    check_attention(out[7777:7778], lse[7777:7778], *ref, 64, BF16)


def test_attention_strided_inputs_and_head_major_pool(cuda_device):
    """q a slice of a fused q/k/v output, the pool [pages, kv_heads, page, dim], out a slice,
    the block table a slice of a wider one."""
    lens, heads, hk, dim, page = [77, 200, 12], 16, 4, 128, 16
    q, k, v, table, n, _ = build(lens, heads, hk, dim, BF16, BF16, page, 1, cuda_device, layout="hnd")
    assert not k.is_contiguous()
    fused = torch.randn(3, (heads + 2 * hk) * dim, device=cuda_device).to(BF16)
    fused[:, :heads * dim] = q.reshape(3, -1)
    qs = fused[:, :heads * dim].view(3, heads, dim)
    wide = torch.full((3, table.size(1) + 5), -7, dtype=torch.int32, device=cuda_device)
    wide[:, :table.size(1)] = table
    out = torch.zeros(3, heads + 3, dim, dtype=BF16, device=cuda_device)
    paged.attention(qs, k, v, wide[:, :table.size(1)], n, out=out[:, 1:heads + 1])
    ref = attention_oracle(q, k, v, table, lens, 1, dim ** -0.5, 0.0, 0, None, None)
    check_attention(out[:, 1:heads + 1], None, *ref, dim, BF16)
    assert not out[:, 0].any() and not out[:, heads + 1:].any()
    # an odd storage offset is copied, not refused
    odd = torch.empty(q.numel() + 1, dtype=BF16, device=cuda_device)[1:].view(q.shape).copy_(q)
    assert torch.equal(paged.attention(odd, k, v, table, n), out[:, 1:heads + 1])


def test_attention_infinite_and_nan_scores(cuda_device):
    """A NaN in a key that a row sees makes its rows NaN, as the definition has it, and no others."""
    lens, heads, hk, dim = [100, 100], 4, 2, 64
    q, k, v, table, n, _ = build(lens, heads, hk, dim, BF16, BF16, 16, 1, cuda_device)
    k[int(table[0, 2]), 3, 1] = float("nan")
    out = paged.attention(q, k, v, table, n)
    assert torch.isnan(out[0, 2:]).all() and torch.isfinite(out[0, :2]).all() and torch.isfinite(out[1]).all()


@pytest.mark.parametrize("qscale", [2.0 ** -60, 2.0 ** 60, 0.0])
def test_attention_e4m3_takes_queries_of_any_size(cuda_device, qscale):
    """bf16 queries far outside fp16's range against an e4m3 cache."""
    lens, heads, hk, dim = [130], 8, 2, 128
    q, k, v, table, n, (ks, vs) = build(lens, heads, hk, dim, BF16, E4M3, 16, 1, cuda_device)
    q = (q.float() * qscale).to(BF16)
    scale = dim ** -0.5 / qscale if qscale else 1.0
    ref = attention_oracle(q, k, v, table, lens, 1, scale, 0.0, 0, ks, vs)
    out, lse = paged.attention(q, k, v, table, n, scale=scale, k_scale=ks, v_scale=vs, return_lse=True)
    check_attention(out, lse, *ref, dim, BF16, E4M3)


def test_attention_offsets_past_32_bits(cuda_device):
    """The last pages of a pool of more than 2^32 bytes."""
    page, hk, dim = 64, 8, 128
    pages = 2 ** 32 // (page * hk * dim) + 40
    k = torch.empty((pages, page, hk, dim), dtype=E4M3, device=cuda_device)
    v = torch.empty_like(k)
    gen = torch.Generator(device=cuda_device)
    gen.manual_seed(1)
    lens = [150]
    table = torch.tensor([[pages - 1, pages - 7, pages - 30]], dtype=torch.int32, device=cuda_device)
    for t in (k, v):
        for p in table[0].tolist():
            t[p] = torch.randn(page, hk, dim, generator=gen, device=cuda_device).to(E4M3)
    q = torch.randn(1, 16, dim, generator=gen, device=cuda_device).to(BF16)
    n = torch.tensor(lens, dtype=torch.int32, device=cuda_device)
    ref = attention_oracle(q, k, v, table, lens, 1, dim ** -0.5, 0.0, 0, None, None)
    check_attention(paged.attention(q, k, v, table, n), None, *ref, dim, BF16, E4M3)
    # and the append writes there
    slot = torch.tensor([(pages - 1) * page + 63], device=cuda_device)
    kn = torch.ones(1, hk, dim, dtype=BF16, device=cuda_device)
    paged.rope_append(q, kn, kn, k, v, torch.zeros_like(slot), slot,
                      torch.ones(dim // 2, device=cuda_device))
    assert (k[pages - 1, 63].float() == 1).all() and (v[pages - 1, 63].float() == 1).all()


def test_attention_graphs_streams_and_growing_lengths(cuda_device):
    """Two graphs captured on one stream, replayed on two streams at once, with lengths that
    grow between replays; a call on a side stream; an empty batch."""
    lens, heads, hk, dim, page = [900, 30], 16, 2, 128, 16
    qa, k, v, table, n, _ = build([1000, 200], heads, hk, dim, BF16, BF16, page, 1, cuda_device)
    n.copy_(torch.tensor(lens, dtype=torch.int32))
    qb = -qa
    paged.attention(qa, k, v, table, n)
    s = torch.cuda.Stream()
    graphs, outs = [], []
    s.wait_stream(torch.cuda.current_stream())
    for q in (qa, qb):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(paged.attention(q, k, v, table, n))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for cur in ([900, 30], [901, 31], [1000, 200], [0, 1]):
        n.copy_(torch.tensor(cur, dtype=torch.int32))
        torch.cuda.synchronize()
        for _ in range(5):
            for g, st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    g.replay()
        torch.cuda.synchronize()
        for q, o in zip((qa, qb), outs):
            assert torch.equal(o, paged.attention(q, k, v, table, n))
            check_attention(o, None, *attention_oracle(q, k, v, table, cur, 1, dim ** -0.5, 0.0, 0, None, None), dim, BF16)
    with torch.cuda.stream(streams[0]):
        side = paged.attention(qa, k, v, table, n)
    torch.cuda.synchronize()
    assert torch.equal(side, outs[0])
    none = paged.attention(qa[:0], k, v, table[:0], n[:0])
    assert none.shape == (0, heads, dim)
    del graphs


def test_attention_records_bad_pages_and_lengths(cuda_device):
    q, k, v, table, n, _ = build([40, 40], 8, 2, 64, BF16, BF16, 16, 1, cuda_device)
    good = paged.attention(q, k, v, table, n)
    bad = table.clone()
    bad[1, 1] = k.size(0)
    out = paged.attention(q, k, v, bad, n)
    assert ops.device_status(cuda_device) == _lib.EBADARG
    assert torch.equal(out[0], good[0]) and torch.isfinite(out).all()
    n2 = torch.tensor([40, 10 ** 9], dtype=torch.int32, device=cuda_device)
    out = paged.attention(q, k, v, table, n2)
    assert ops.device_status(cuda_device) == _lib.EBADARG
    assert torch.equal(out[0], good[0])
    n3 = torch.tensor([40, -5], dtype=torch.int32, device=cuda_device)
    out = paged.attention(q, k, v, table, n3)  # no tokens
    assert ops.device_status(cuda_device) == 0
    assert torch.equal(out[0], good[0]) and not out[1].any()


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------

def rotate_oracle(x, positions, inv_freq, interleaved):
    """(value, |x| + |y| of the pair) in float64."""
    x = x.double().cpu().clone()
    r = 2 * inv_freq.numel()
    i = torch.arange(0, r, 2) if interleaved else torch.arange(r // 2)
    j = i + 1 if interleaved else i + r // 2
    ang = torch.outer(positions.double().cpu(), inv_freq.double().cpu())[:, None, :]
    a, b = x[:, :, i].clone(), x[:, :, j].clone()
    size = torch.zeros_like(x)
    size[:, :, i] = size[:, :, j] = a.abs() + b.abs()
    x[:, :, i] = a * torch.cos(ang) - b * torch.sin(ang)
    x[:, :, j] = b * torch.cos(ang) + a * torch.sin(ang)
    return x, size


@pytest.mark.parametrize("tokens,heads,hk,dim,src,ct,page,rotary,inter", [
    (1, 64, 8, 128, FP16, BF16, 16, 128, False),
    (1, 1, 1, 64, BF16, BF16, 1, 64, True),
    (7, 28, 4, 128, BF16, E4M3, 24, 128, False),
    (33, 5, 1, 64, FP32, FP16, 64, 32, True),
    (33, 8, 8, 128, FP16, FP16, 7, 64, False),
    (129, 16, 2, 64, FP32, E4M3, 16, 64, False),
    (50, 8, 2, 128, BF16, BF16, 16, 0, False),
    (5000, 8, 2, 64, FP16, BF16, 16, 64, False),   # tiles of four tokens, the last one partial
    (4739, 5, 1, 128, FP32, E4M3, 24, 128, True),
])
def test_append_matches_definition(cuda_device, tokens, heads, hk, dim, src, ct, page, rotary, inter):
    dev = cuda_device
    gen = torch.Generator(device=dev)
    gen.manual_seed(tokens + dim)
    fused = torch.randn(tokens, (heads + 2 * hk) * dim, generator=gen, device=dev).to(src)
    q, k, v = (t.view(tokens, -1, dim) for t in fused.split([heads * dim, hk * dim, hk * dim], dim=1))
    pages = -(-tokens // page) + 2
    kc, vc = make_cache(pages, page, hk, dim, ct, gen, dev)
    k0, v0 = kc.clone(), vc.clone()
    slots = torch.randperm(pages * page, generator=gen, device=dev)[:tokens]
    if tokens > 4:
        slots[::5] = -1  # padding
    positions = torch.randint(0, 1 << 20, (tokens,), generator=gen, device=dev)
    positions[0] = 2 ** 31 - 1
    inv = (1.0 / 1e4 ** (torch.arange(0, rotary, 2, dtype=torch.float64) / max(rotary, 1))).float().to(dev)
    ks = vs = None
    if ct == E4M3:
        ks, vs = (torch.rand(hk, generator=gen, device=dev) * 0.01 + 0.004 for _ in range(2))  # some values saturate
    qo = paged.rope_append(q, k, v, kc, vc, positions, slots, inv, interleaved=inter, k_scale=ks, v_scale=vs)
    assert qo.dtype == (BF16 if ct == E4M3 else ct)
    ref, size = rotate_oracle(q, positions, inv, inter)
    tiny = 2.0 ** -25 if qo.dtype == FP16 else 0.0
    assert ((qo.double().cpu() - ref).abs() <= half_step(qo.dtype) * ref.abs() + 2.0 ** -22 * size + tiny).all()
    kept = (slots >= 0).cpu()
    at = slots[slots >= 0]
    for cache, old, new, sc, rot in ((kc, k0, k, ks, True), (vc, v0, v, vs, False)):
        want, size = rotate_oracle(new, positions, inv if rot else inv[:0], inter)
        raw = cache.reshape(-1, hk, dim)
        got = (raw.view(torch.uint8)[at].view(ct) if ct == E4M3 else raw[at]).double().cpu()
        want, size = want[kept], size[kept]
        if sc is not None:
            f = sc.double().cpu()[None, :, None]
            want, size = (want / f).clamp(-448, 448), size / f
        tiny = 2.0 ** -10 if ct == E4M3 else 2.0 ** -25 if ct == FP16 else 0.0
        slack = 2.0 ** -22 * (size + want.abs())  # of the rotation and the division
        assert ((got - want).abs() <= half_step(ct) * want.abs() + slack + tiny).all()
        # slots that no token names are as they were
        mask = torch.ones(pages * page, dtype=torch.bool, device=dev)
        mask[at] = False
        bytes_ = lambda t: t.reshape(-1, hk, dim).view(torch.uint8)[mask]  # noqa: E731
        assert torch.equal(bytes_(cache), bytes_(old))
    assert ops.device_status(dev) == 0


def test_append_far_positions_turn_exactly(cuda_device):
    """Angles of positions up to 2^31 are those of 64-bit arithmetic: an fp32 product would be off
    by whole turns."""
    pos = torch.tensor([0, 1, 131071, 10 ** 6 + 1, 2 ** 31 - 1, -5], device=cuda_device)
    x = torch.zeros(6, 1, 128, device=cuda_device)
    x[..., :64] = 1.0
    inv = (1.0 / 5e5 ** (torch.arange(0, 128, 2, dtype=torch.float64) / 128)).float().to(cuda_device)
    kc = torch.zeros(1, 8, 1, 128, dtype=FP16, device=cuda_device)
    q = paged.rope_append(x, x, x, kc, torch.zeros_like(kc), pos, torch.arange(6, device=cuda_device), inv)
    ang = torch.outer(pos.double().cpu(), inv.double().cpu())
    ref = torch.cat([torch.cos(ang), torch.sin(ang)], dim=-1)
    # fp16 half step, and 2^-22 of the pair's size 1
    assert ((q[:, 0].double().cpu() - ref).abs() <= 2.0 ** -11 * ref.abs() + 2.0 ** -22 + 2.0 ** -25).all()


def test_append_in_place_strides_and_bad_slots(cuda_device):
    dev = cuda_device
    gen = torch.Generator(device=dev)
    gen.manual_seed(2)
    fused = torch.randn(9, 12 * 128, generator=gen, device=dev).to(BF16)
    q, k, v = (t.view(9, -1, 128) for t in fused.split([8 * 128, 2 * 128, 2 * 128], dim=1))
    kc, vc = make_cache(4, 16, 2, 128, BF16, gen, dev, layout="hnd")
    pos = torch.arange(9, device=dev) * 100
    inv = torch.rand(64, generator=gen, device=dev)
    slots = torch.arange(9, device=dev) + 20
    want = paged.rope_append(q, k, v, kc, vc, pos, slots, inv)
    k1 = kc.clone()
    kc.zero_()
    before = fused.clone()
    got = paged.rope_append(q, k, v, kc, vc, pos, slots, inv, q_out=q)
    assert got.data_ptr() == q.data_ptr() and torch.equal(q, want)
    assert torch.equal(fused[:, 8 * 128:], before[:, 8 * 128:])
    assert torch.equal(kc[1, 4:13], k1[1, 4:13]) and not kc[0].any() and not kc[2:].any()
    assert ops.device_status(dev) == 0
    slots[3], slots[4] = 64, 2 ** 40
    ref = kc.clone()
    paged.rope_append(want, k, v, kc, vc, pos, slots, inv)
    assert ops.device_status(dev) == _lib.EBADARG
    assert torch.equal(kc, ref)  # the good slots hold the same values, the bad ones were not written
    assert paged.rope_append(q[:0], k[:0], v[:0], kc, vc, pos[:0], slots[:0], inv).shape == (0, 8, 128)


def test_append_then_attention_in_a_graph(cuda_device):
    """The two as a decode step uses them: appended, then attended to, captured once and
    replayed while the sequences grow, against the definition on what the caches hold."""
    dev = cuda_device
    heads, hk, dim, page, S = 8, 2, 128, 16, 3
    gen = torch.Generator(device=dev)
    gen.manual_seed(3)
    kc, vc = make_cache(40, page, hk, dim, BF16, gen, dev)
    table = torch.randperm(40, generator=torch.Generator().manual_seed(1))[:S * 8].view(S, 8).int().to(dev)
    fused = torch.empty(S, (heads + 2 * hk) * dim, dtype=FP16, device=dev)
    q, k, v = (t.view(S, -1, dim) for t in fused.split([heads * dim, hk * dim, hk * dim], dim=1))
    pos = torch.tensor([0, 15, 77], device=dev)
    lens = (pos + 1).int()
    inv = (1.0 / 1e4 ** (torch.arange(0, dim, 2, dtype=torch.float64) / dim)).float().to(dev)

    def step():
        slots = table.gather(1, (pos // page)[:, None])[:, 0].long() * page + pos % page
        qr = paged.rope_append(q, k, v, kc, vc, pos, slots, inv)
        lens.copy_(pos + 1)
        return qr, paged.attention(qr, kc, vc, table, lens)

    fused.normal_(generator=gen)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        qr, out = step()
    for _ in range(20):
        fused.normal_(generator=gen)
        g.replay()
        torch.cuda.synchronize()
        ref = attention_oracle(qr, kc, vc, table, (pos + 1).tolist(), 1, dim ** -0.5, 0.0, 0, None, None)
        check_attention(out, None, *ref, dim, BF16)
        for i in range(S):
            p = int(pos[i])
            want, size = rotate_oracle(k[i:i + 1], pos[i:i + 1], inv, False)
            have = kc[int(table[i, p // page]), p % page].double().cpu()
            assert ((have - want[0]).abs() <= 2.0 ** -8 * want[0].abs() + 2.0 ** -22 * size[0]).all()
        pos.add_(1)


def test_python_refusals(cuda_device):
    dev = cuda_device
    kc = torch.zeros(4, 16, 2, 128, dtype=BF16, device=dev)
    q = torch.zeros(3, 8, 128, dtype=BF16, device=dev)
    kv = torch.zeros(3, 2, 128, dtype=BF16, device=dev)
    i64 = torch.zeros(3, dtype=torch.int64, device=dev)
    inv = torch.zeros(64, device=dev)
    table, lens = torch.zeros(3, 4, dtype=torch.int32, device=dev), torch.zeros(3, dtype=torch.int32, device=dev)
    ok_a = dict(q=q, k=kv, v=kv, k_cache=kc, v_cache=kc.clone(), positions=i64, slots=i64 - 1, inv_freq=inv)
    ok_b = dict(q=q, k_cache=kc, v_cache=kc, block_table=table, seq_lens=lens)
    paged.rope_append(**ok_a)
    paged.attention(**ok_b)
    scale = torch.ones(2, device=dev)
    f8 = kc.to(E4M3)
    for kw in (dict(k_cache=kc.half()), dict(k_cache=kc.float(), v_cache=kc.float()), dict(k_cache=kc[..., :96], v_cache=kc[..., :96]),
               dict(k_cache=kc[0], v_cache=kc[0]), dict(k_cache=kc[:0], v_cache=kc[:0]), dict(v_cache=kc[:2]),
               dict(k_cache=kc[:1].expand(4, -1, -1, -1), v_cache=kc[:1].expand(4, -1, -1, -1)),
               dict(k_scale=scale), dict(k_cache=f8, v_cache=f8, k_scale=scale[:1]), dict(k_cache=f8, v_cache=f8, v_scale=scale.double())):
        for f, ok in ((paged.rope_append, ok_a), (paged.attention, ok_b)):
            with pytest.raises(RuntimeError):
                f(**{**ok, **kw})
    for kw in (dict(q=q.half()), dict(q=q[..., :64]), dict(k=kv[:2]), dict(v=kv[:, :1]), dict(positions=i64.int()),
               dict(slots=i64[:2]), dict(inv_freq=inv.double()), dict(inv_freq=inv[:12]), dict(q_out=q.half()),
               dict(q_out=q.transpose(0, 1)), dict(inv_freq=torch.zeros(72, device=dev)), dict(slots=(i64 - 1).cpu())):
        with pytest.raises(RuntimeError):
            paged.rope_append(**{**ok_a, **kw})
    for kw in (dict(q=q.half()), dict(q=q.float()), dict(q=q[:, :7]), dict(q=q[:2]), dict(rows_per_seq=2), dict(rows_per_seq=0),
               dict(block_table=table.long()), dict(block_table=table[0]), dict(block_table=table[:, :0]),
               dict(seq_lens=lens.long()), dict(seq_lens=lens[:2]), dict(softcap=-1.0), dict(window=-1),
               dict(softcap=float("inf")), dict(softcap=1e-7), dict(scale=0.0), dict(scale=-1.0), dict(out=q.half()), dict(out=q[:2]), dict(seq_lens=lens.cpu())):
        with pytest.raises(RuntimeError):
            paged.attention(**{**ok_b, **kw})
