"""Measured cases of the paged-cache and log-probability operators, with their plain forms.

Three operators of a serving step around the EXL3 linears:

* ``append``: ``exl3_b200.paged.rope_append`` - the position rotation of q and k, and k and v
  written into a paged cache;
* ``attention``: ``exl3_b200.paged.attention`` - the new tokens of each sequence over its pages;
* ``logprobs``: ``exl3_b200.logprobs.token_logprobs`` - log-probability of given tokens, the
  entropy and the top alternatives.

With ``own`` false ``run`` computes them in elementary torch operations, with ``own`` true
through the package.  ``exact`` restates the definitions in 64 bits.
"""

import math
import os
import random
import sys

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "e4m3": torch.float8_e4m3fn}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4, "e4m3": 1}
_E4M3_MAX = 448.0


def _package():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sglang-exl3_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from exl3_b200 import logprobs, paged

    return paged, logprobs


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------

def _append(tokens, heads, kv_heads, dim, src, cache, page, first=0, rotary=0, interleaved=False, padded=0):
    return {"op": "append", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim, "src": src,
            "cache": cache, "page": page, "first": first, "rotary": rotary or dim, "interleaved": interleaved,
            "padded": padded}


def _attention(seqs, longest, heads, kv_heads, dim, q, cache, page, rows=1, softcap=0.0, window=0, ragged=True):
    return {"op": "attention", "seqs": seqs, "longest": longest, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "q": q, "cache": cache, "page": page, "rows": rows, "softcap": softcap, "window": window,
            "ragged": ragged}


def _logprobs(rows, vocab, src, top):
    return {"op": "logprobs", "rows": rows, "vocab": vocab, "src": src, "top": top}


def listed():
    return [
        # one new token of one sequence far into its context, 64 / 8 heads of 128: a latency
        dict(_append(1, 64, 8, 128, "fp16", "bf16", 16, first=100000), name="append-1-token"),
        # a decode batch with an 8-bit cache, some rows of the batch being padding
        dict(_append(64, 64, 8, 128, "bf16", "e4m3", 64, first=4000, padded=5), name="append-batch-64-e4m3"),
        # a short prompt of odd length, fp32 projections, half of a 64-wide head rotated in adjacent pairs
        dict(_append(1357, 32, 8, 64, "fp32", "fp16", 1, rotary=32, interleaved=True), name="append-prompt-1357"),
        # prompts filling a prefill batch, 64 / 8 heads of 128
        dict(_append(16384, 64, 8, 128, "fp16", "bf16", 16), name="append-prompt-16384"),
        # one sequence in the middle of a chat: a latency
        dict(_attention(1, 2049, 64, 8, 128, "bf16", "bf16", 16, ragged=False), name="attention-1x2049"),
        # a small batch of sequences of very different lengths, one of them not begun
        dict(_attention(9, 8191, 64, 8, 128, "bf16", "bf16", 16), name="attention-9-ragged"),
        # speculative verify: 5 rows per sequence, 32 / 4 heads, an 8-bit cache
        dict(_attention(16, 8192, 32, 4, 128, "bf16", "e4m3", 64, rows=5), name="attention-verify-16x5-e4m3"),
        # capped scores in a sliding window over 64-wide heads, as layers of local attention have
        dict(_attention(33, 12345, 32, 8, 64, "fp16", "fp16", 32, softcap=30.0, window=4096),
             name="attention-window-cap"),
        # a full serving batch of long sequences
        dict(_attention(64, 16384, 64, 8, 128, "bf16", "bf16", 64), name="attention-64x16384"),
        # the answer to one user: one row of logits, five alternatives
        dict(_logprobs(1, 128256, "bf16", 5), name="logprobs-1-row"),
        # a verify step's 16 x 5 rows of fp32 logits, twenty alternatives
        dict(_logprobs(80, 151936, "fp32", 20), name="logprobs-verify-80"),
        # scoring a prompt: every position's token
        dict(_logprobs(2048, 128256, "bf16", 1), name="logprobs-prompt-2048"),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("append", "attention", "attention", "logprobs"))
    heads, kv_heads = rng.choice(((64, 8), (32, 8), (32, 4), (28, 4), (16, 16), (8, 1), (5, 1)))
    dim = rng.choice((64, 128, 128))
    if op == "append":
        # up to the prefill batch's bytes: 16384 tokens of 64 + 2 * 8 heads of 128
        src = rng.choice(("fp16", "bf16", "fp32"))
        most = 16384 * 80 * 128 // ((heads + 2 * kv_heads) * dim * (2 if src == "fp32" else 1))
        tokens = _log_uniform(rng, 1, min(16384, most))
        return _append(tokens, heads, kv_heads, dim, src, rng.choice(("fp16", "bf16", "e4m3")),
                       rng.choice((1, 16, 24, 64)), first=rng.choice((0, 37, 5000, 131072)),
                       rotary=rng.choice((dim, dim, dim // 2)), interleaved=rng.choice((False, True)),
                       padded=rng.choice((0, 0, min(3, tokens - 1))))
    if op == "attention":
        seqs = _log_uniform(rng, 1, 200)
        longest = _log_uniform(rng, 1, 32768)
        while seqs * longest * kv_heads * dim > 64 * 16384 * 8 * 128:
            longest //= 2
        q = rng.choice(("bf16", "fp16"))
        return _attention(seqs, longest, heads, kv_heads, dim, q, rng.choice((q, q, "e4m3")),
                          rng.choice((1, 16, 24, 64, 128)), rows=rng.choice((1, 1, 1, 2, 4, 5)),
                          softcap=rng.choice((0.0, 0.0, 50.0)), window=rng.choice((0, 0, 1 + longest // 3)),
                          ragged=rng.choice((False, True, True)))
    src = rng.choice(("bf16", "fp16", "fp32"))
    vocab = _log_uniform(rng, 1000, 160000)
    most = 2048 * 128256 * 2 // (vocab * _BYTES[src])
    return _logprobs(_log_uniform(rng, 1, min(2048, most)), vocab, src, min(vocab, rng.choice((0, 1, 5, 20, 32))))


def _lengths(case):
    """Tokens of each sequence, its new ones among them: by the case alone, so that its work is known."""
    n, longest = case["seqs"], case["longest"]
    if not case["ragged"]:
        return [longest] * n
    rng = random.Random(n * 1000003 + longest)
    got = [int(round(longest * rng.uniform(0.25, 1.0))) for _ in range(n)]
    got[rng.randrange(n)] = longest
    if n > 4:  # a sequence that has not begun
        got[got.index(min(got))] = 0
    return got


def work(case):
    if case["op"] == "append":
        q, kv = case["tokens"] * case["heads"] * case["dim"], 2 * case["tokens"] * case["kv_heads"] * case["dim"]
        kv_read = 2 * (case["tokens"] - case["padded"]) * case["kv_heads"] * case["dim"]
        b = (q + kv) * _BYTES[case["src"]] + q * 2 + kv_read * _BYTES[case["cache"]]
        return {"bytes": b, "flops": 3 * (q + kv // 2)}
    if case["op"] == "attention":
        seen, pairs = 0, 0  # positions read, (row, position) pairs
        for n in _lengths(case):
            ends = [n - case["rows"] + 1 + j for j in range(case["rows"])]
            spans = [(max(0, e - case["window"]) if case["window"] else 0, max(0, e)) for e in ends]
            pairs += sum(e - s for s, e in spans)
            seen += max(e for _, e in spans) - min(s for s, e in spans if e > 0) if any(e > 0 for _, e in spans) else 0
        rows = case["seqs"] * case["rows"] * case["heads"]
        b = 2 * seen * case["kv_heads"] * case["dim"] * _BYTES[case["cache"]] + rows * (case["dim"] * 4 + 4)
        return {"bytes": b, "flops": 4 * pairs * case["heads"] * case["dim"]}
    n = case["rows"] * case["vocab"]
    return {"bytes": n * _BYTES[case["src"]] + case["rows"] * (16 + 12 * case["top"]), "flops": 6 * n}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _randn(shape, gen, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, device="cuda", generator=gen, dtype=torch.float32) * scale).to(dtype)


def _pages(shape, gen, dtype):
    """A cache full of values: the pages in use and those of other sequences alike."""
    if dtype != torch.float8_e4m3fn:
        return torch.randn(shape, device="cuda", generator=gen, dtype=dtype)
    return torch.randn(shape, device="cuda", generator=gen, dtype=torch.float16).clamp_(-_E4M3_MAX, _E4M3_MAX).to(dtype)


def _scales(kv_heads, gen, lo, hi):
    return torch.rand(kv_heads, device="cuda", generator=gen) * (hi - lo) + lo


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    if case["op"] == "append":
        T, hq, hk, d, page = case["tokens"], case["heads"], case["kv_heads"], case["dim"], case["page"]
        dtype, cache = _TYPES[case["src"]], _TYPES[case["cache"]]
        # q, k and v are column slices of the fused projection's output, as the linears leave them
        fused = _randn((T, (hq + 2 * hk) * d), gen, dtype)
        q, k, v = (t.view(T, -1, d) for t in fused.split([hq * d, hk * d, hk * d], dim=1))
        pages = 1 + 2 * (-(-T // page))
        # page 0 belongs to no sequence; tokens fill pages that lie anywhere in the pool
        order = torch.randperm(pages - 1, device="cuda", generator=gen) + 1
        at = torch.arange(T, device="cuda")
        slots = order[at // page] * page + at % page
        positions = at + case["first"] if T > 64 else case["first"] + torch.randint(0, 500, (T,), device="cuda",
                                                                                    generator=gen)
        if case["padded"]:
            slots[T - case["padded"]:] = -1  # rows of a padded batch: rotated, not written
        r = case["rotary"]
        inv = 1.0 / (5e5 ** (torch.arange(0, r, 2, device="cuda", dtype=torch.float64) / r))
        quant = case["cache"] == "e4m3"
        return {"case": case, "q": q, "k": k, "v": v, "slots": slots, "positions": positions,
                "inv_freq": inv.float(), "k_cache": _pages((pages, page, hk, d), gen, cache),
                "v_cache": _pages((pages, page, hk, d), gen, cache),
                "k_scale": _scales(hk, gen, 0.01, 0.05) if quant else None,
                "v_scale": _scales(hk, gen, 0.01, 0.05) if quant else None}
    if case["op"] == "attention":
        S, R, hq, hk, d, page = (case[x] for x in ("seqs", "rows", "heads", "kv_heads", "dim", "page"))
        lengths = _lengths(case)
        counts = [-(-n // page) for n in lengths]
        pages = 1 + sum(counts)
        order = (torch.randperm(pages - 1, generator=torch.Generator().manual_seed(seed)) + 1).to(torch.int32)
        table = torch.full((S, max(1, -(-case["longest"] // page))), -1, dtype=torch.int32)
        at = 0
        for s, n in enumerate(counts):
            table[s, :n] = order[at:at + n]
            at += n
        cache = _TYPES[case["cache"]]
        quant = case["cache"] == "e4m3"
        # a query looks for some keys more than for others: scores spread over a few units
        return {"case": case, "q": _randn((S * R, hq, d), gen, _TYPES[case["q"]], 2.0 / (0.35 if quant else 1.0)),
                "k_cache": _pages((pages, page, hk, d), gen, cache), "v_cache": _pages((pages, page, hk, d), gen, cache),
                "table": table.cuda(), "lengths": torch.tensor(lengths, dtype=torch.int32).cuda(),
                "k_scale": _scales(hk, gen, 0.3, 0.4) if quant else None,
                "v_scale": _scales(hk, gen, 0.3, 0.4) if quant else None}
    rows, vocab = case["rows"], case["vocab"]
    # logits of a language model: a wide body and a few tokens far above it
    x = torch.randn((rows, vocab), device="cuda", generator=gen, dtype=torch.float32).mul_(2.0)
    peak = torch.randint(0, vocab, (rows, 8), device="cuda", generator=gen)
    x.scatter_add_(1, peak, torch.rand((rows, 8), device="cuda", generator=gen) * 14.0)
    tokens = peak[:, 0].clone()
    return {"case": case, "logits": x.to(_TYPES[case["src"]]), "tokens": tokens}


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def _rotate(x, cos, sin, interleaved):
    """x [T, heads, dim] in fp32, its first 2 * cos.size(-1) dims rotated."""
    r = 2 * cos.size(-1)
    body, rest = x[..., :r], x[..., r:]
    c, s = cos[:, None, :], sin[:, None, :]
    a, b = (body[..., 0::2], body[..., 1::2]) if interleaved else (body[..., :r // 2], body[..., r // 2:])
    first, second = a * c - b * s, b * c + a * s
    if interleaved:
        return torch.cat([torch.stack([first, second], dim=-1).flatten(-2), rest], dim=-1)
    return torch.cat([first, second, rest], dim=-1)


def _to_cache(x, scale, dtype):
    if scale is None:
        return x.to(dtype)
    return (x / scale[None, :, None]).clamp(-_E4M3_MAX, _E4M3_MAX).to(dtype)


def _plain_append(st):
    case = st["case"]
    angle = st["positions"].double()[:, None] * st["inv_freq"].double()[None, :]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    q = _rotate(st["q"].float(), cos, sin, case["interleaved"])
    k = _rotate(st["k"].float(), cos, sin, case["interleaved"])
    at = st["slots"].clamp(min=0)  # page 0 belongs to nobody: padding writes its slot's own value there
    kept = (st["slots"] >= 0)[:, None, None]
    for cache, new, scale in ((st["k_cache"], k, st["k_scale"]), (st["v_cache"], st["v"].float(), st["v_scale"])):
        flat = cache.view(-1, cache.size(2), cache.size(3))
        if flat.dtype == torch.float8_e4m3fn:
            bits = flat.view(torch.uint8)
            bits[at] = torch.where(kept, _to_cache(new, scale, flat.dtype).view(torch.uint8), bits[at])
        else:
            flat[at] = torch.where(kept, _to_cache(new, scale, flat.dtype), flat[at])
    q_type = st["k_cache"].dtype if st["k_scale"] is None else torch.bfloat16
    return q.to(q_type), st["k_cache"], st["v_cache"]


def _plain_attention(st):
    case = st["case"]
    S, R, hq, hk, d, page = (case[x] for x in ("seqs", "rows", "heads", "kv_heads", "dim", "page"))
    n = st["table"].size(1) * page
    at = st["table"].clamp(min=0).long()
    k = st["k_cache"].view(torch.uint8)[at].view(st["k_cache"].dtype).float().view(S, n, hk, d)
    v = st["v_cache"].view(torch.uint8)[at].view(st["v_cache"].dtype).float().view(S, n, hk, d)
    if st["k_scale"] is not None:
        k, v = k * st["k_scale"][None, None, :, None], v * st["v_scale"][None, None, :, None]
    q = st["q"].float().view(S, R, hk, hq // hk, d).permute(0, 2, 3, 1, 4).reshape(S, hk, -1, d)  # [S, hk, G R, d]
    s = torch.matmul(q, k.permute(0, 2, 3, 1)) * (d ** -0.5)
    if case["softcap"]:
        s = case["softcap"] * torch.tanh(s / case["softcap"])
    s = s.view(S, hk, hq // hk, R, n)
    end = st["lengths"][:, None] - R + 1 + torch.arange(R, device=s.device)[None, :]  # [S, R]: positions below are seen
    pos = torch.arange(n, device=s.device)[None, None, :]
    seen = pos < end[:, :, None]
    if case["window"]:
        seen = seen & (pos >= end[:, :, None] - case["window"])
    s = s.masked_fill(~seen[:, None, None], float("-inf"))
    m = s.amax(dim=-1, keepdim=True)
    m = torch.where(m == float("-inf"), torch.zeros_like(m), m)  # a row that sees nothing
    p = torch.exp(s - m)
    total = p.sum(dim=-1, keepdim=True)
    o = torch.matmul(p.view(S, hk, -1, n), v.permute(0, 2, 1, 3)).view(S, hk, hq // hk, R, d)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    lse = (m + torch.log(total))[..., 0]  # a row that sees nothing: -inf
    out = o.permute(0, 3, 1, 2, 4).reshape(S * R, hq, d).to(st["q"].dtype)
    return out, lse.permute(0, 3, 1, 2).reshape(S * R, hq)


def _plain_logprobs(st):
    top = st["case"]["top"]
    x = st["logits"].float()
    m = x.amax(dim=-1, keepdim=True)
    y = x - m
    e = torch.exp(y)
    total = e.sum(dim=-1, keepdim=True)
    log_total = torch.log(total)
    logprob = (torch.gather(y, 1, st["tokens"][:, None]) - log_total)[:, 0]
    entropy = log_total[:, 0] - (e * y).sum(dim=-1) / total[:, 0]
    if not top:
        return logprob, entropy
    # unique keys, so that of equal logits the lower index comes first
    bits = x.view(torch.int32).long()
    order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
    n = x.size(1)
    key = order * (1 << 20) + (n - 1 - torch.arange(n, device=x.device))
    ids = n - 1 - (torch.topk(key, top, dim=-1, sorted=True).values & ((1 << 20) - 1))
    return logprob, entropy, torch.gather(y, 1, ids) - log_total, ids


def run(st):
    case = st["case"]
    if own:
        paged, logprobs = _package()
        if case["op"] == "append":
            q = paged.rope_append(st["q"], st["k"], st["v"], st["k_cache"], st["v_cache"], st["positions"],
                                  st["slots"], st["inv_freq"], interleaved=case["interleaved"],
                                  k_scale=st["k_scale"], v_scale=st["v_scale"])
            return q, st["k_cache"], st["v_cache"]
        if case["op"] == "attention":
            return paged.attention(st["q"], st["k_cache"], st["v_cache"], st["table"], st["lengths"],
                                   rows_per_seq=case["rows"], softcap=case["softcap"], window=case["window"],
                                   k_scale=st["k_scale"], v_scale=st["v_scale"], return_lse=True)
        got = logprobs.token_logprobs(st["logits"], st["tokens"], top=case["top"])
        return tuple(got) if case["top"] else (got.logprob, got.entropy)
    if case["op"] == "append":
        return _plain_append(st)
    return _plain_attention(st) if case["op"] == "attention" else _plain_logprobs(st)


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------

def _exact_append(st):
    """Pairs (i, j) of a head's dims turned by position * inv_freq, as complex numbers."""
    case = st["case"]
    r, T = case["rotary"], case["tokens"]
    if case["interleaved"]:
        i, j = torch.arange(0, r, 2), torch.arange(1, r, 2)
    else:
        i, j = torch.arange(r // 2), torch.arange(r // 2, r)
    i, j = i.cuda(), j.cuda()
    turn = torch.polar(torch.ones((T, 1, r // 2), dtype=torch.float64, device="cuda"),
                       torch.outer(st["positions"].double(), st["inv_freq"].double())[:, None, :])

    def turned(x):
        x = x.double().clone()
        z = torch.complex(x[:, :, i].contiguous(), x[:, :, j].contiguous()) * turn
        x[:, :, i], x[:, :, j] = z.real, z.imag
        return x

    out = [turned(st["q"])]
    rows = torch.nonzero(st["slots"] >= 0)[:, 0]
    for cache, new, scale in ((st["k_cache"], turned(st["k"]), st["k_scale"]),
                              (st["v_cache"], st["v"].double(), st["v_scale"])):
        if scale is not None:
            new = (new / scale.double()[:, None]).clamp(-_E4M3_MAX, _E4M3_MAX)
        full = cache.double()
        slot = st["slots"][rows]
        full[slot // case["page"], slot % case["page"]] = new[rows]
        out.append(full)
    return tuple(out)


def _exact_attention(st):
    """Sequence by sequence, head by head: softmax over the positions that a row sees."""
    case = st["case"]
    R, hq, hk, d, page = (case[x] for x in ("rows", "heads", "kv_heads", "dim", "page"))
    group = hq // hk
    out = torch.zeros((case["seqs"] * R, hq, d), dtype=torch.float64, device="cuda")
    lse = torch.full((case["seqs"] * R, hq), float("-inf"), dtype=torch.float64, device="cuda")
    for s, n in enumerate(_lengths(case)):
        if n == 0:
            continue
        pages = st["table"][s, :-(-n // page)].long()
        kv = []
        for cache, scale in ((st["k_cache"], st["k_scale"]), (st["v_cache"], st["v_scale"])):
            x = cache.view(torch.uint8)[pages].view(cache.dtype).double().flatten(0, 1)[:n].transpose(0, 1)
            kv.append(x if scale is None else x * scale.double()[:, None, None])  # [hk, n, d]
        for j in range(R):
            stop = n - R + 1 + j
            start = max(0, stop - case["window"]) if case["window"] else 0
            if stop <= start:
                continue
            q = st["q"][s * R + j].double().view(hk, group, d)
            score = torch.einsum("hgd,hnd->hgn", q, kv[0][:, start:stop]) / math.sqrt(d)
            if case["softcap"]:
                score = torch.tanh(score / case["softcap"]) * case["softcap"]
            out[s * R + j] = torch.einsum("hgn,hnd->hgd", torch.softmax(score, -1), kv[1][:, start:stop]).reshape(hq, d)
            lse[s * R + j] = torch.logsumexp(score, -1).reshape(hq)
    return out, lse


def _exact_logprobs(st):
    case = st["case"]
    got = []
    for x, t in zip(st["logits"].split(64), st["tokens"].split(64)):
        lp = torch.log_softmax(x.double(), dim=-1)
        part = [lp[torch.arange(len(t), device=t.device), t], -(lp.exp() * lp).sum(-1)]
        if case["top"]:
            part += [torch.sort(lp, dim=-1, descending=True, stable=True).values[:, :case["top"]]]
        got.append(part)
    outs = [torch.cat(p) for p in zip(*got)]
    return tuple(outs) + ((None,) if case["top"] else ())


def exact(case, seed):
    st = prepare(case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "logprobs": _exact_logprobs}[case["op"]](st)
