"""Log-probabilities of given tokens, the distribution's entropy and its top alternatives
from logits (``exl3b200_token_logprobs``): what a serving step reports beside its tokens, and
what a speculative verify step weighs its draft tokens with.  One pass over the logits."""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib
from .ops import _OUT_DTYPES, _require_cuda


class TokenLogprobs(NamedTuple):
    logprob: torch.Tensor                  # fp32 [rows]
    entropy: torch.Tensor                  # fp32 [rows], nats
    top_logprobs: Optional[torch.Tensor]   # fp32 [rows, top], most likely first; None with top = 0
    top_ids: Optional[torch.Tensor]        # int64 [rows, top]


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0) -> TokenLogprobs:
    """``logits [rows, vocab]`` fp16, bf16 or fp32 (row-strided views serve), ``tokens`` int64
    ``[rows]``.  ``logprob`` is -inf for an id outside the vocabulary (a row that asks for no
    token passes -1); equal logits rank by id; -inf logits are excluded tokens; a row of only
    those, or with a NaN or +inf, gives NaN.  ``top`` at most 32."""
    if logits.dtype not in _OUT_DTYPES or logits.dim() != 2 or logits.size(1) < 1:
        raise RuntimeError("logits must be fp16, bf16 or fp32 [rows, vocab]")
    rows, vocab = logits.shape
    if tokens.dtype != torch.int64 or tokens.shape != (rows,):
        raise RuntimeError("tokens must be int64 [rows]")
    top = int(top)
    if not 0 <= top <= min(_lib.LOGPROBS_MAX_TOP, vocab):
        raise RuntimeError(f"top must be 0..{_lib.LOGPROBS_MAX_TOP} and at most the vocabulary")
    index = logits.get_device()
    if index < 0 or tokens.get_device() != index:
        _require_cuda(logits, tokens)
    if logits.stride(1) != 1 or (rows > 1 and logits.stride(0) < vocab):
        logits = logits.contiguous()
    tokens = tokens.contiguous()
    lp, entropy = torch.empty_like(tokens, dtype=torch.float32), torch.empty_like(tokens, dtype=torch.float32)
    top_ids = top_lp = None
    if top:
        top_ids = tokens.new_empty((rows, top))
        top_lp = torch.empty_like(top_ids, dtype=torch.float32)
    if rows:
        _lib.launch("exl3b200_token_logprobs", index, logits.data_ptr(), logits.stride(0), rows, vocab,
                    _OUT_DTYPES[logits.dtype], tokens.data_ptr(), top, lp.data_ptr(), entropy.data_ptr(),
                    top_lp.data_ptr() if top else None, top_ids.data_ptr() if top else None)
    return TokenLogprobs(lp, entropy, top_lp, top_ids)
