"""Scores of given tokens under rows of logits.

The reference measures its packed models by perplexity (measure_ppl.py:40-65,
measure_quad_ppl.py:57-85); :func:`token_logprobs` gives what such a
measurement, and a server that reports log probabilities, takes from the
logits, in one pass over them.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib

MAX_TOP = 32
_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}


class TokenLogprobs(NamedTuple):
    logprob: torch.Tensor        # float32 [rows]
    entropy: torch.Tensor        # float32 [rows], in nats
    top_ids: torch.Tensor        # int32 [rows, top]
    top_logprobs: torch.Tensor   # float32 [rows, top]


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0,
                   status: torch.Tensor | None = None) -> TokenLogprobs:
    """Log probability of ``tokens[r]`` under ``softmax(logits[r])``, the row's
    entropy, and its ``top`` likeliest tokens (at most 32).

    ``logits`` ``[rows, vocab]`` FP16, BF16 or float32 with contiguous rows;
    ``tokens`` int32 ``[rows]``.  A negative token asks for no score (0); one
    past the vocabulary gets NaN and sets ``status`` (device int32) to 4.
    Equal logits are ranked by the lower index, NaN before every number.
    """
    dev = _lib.require_cuda(logits, tokens, status)
    if logits.dim() != 2 or logits.dtype not in _DTYPES or (logits.stride(1) != 1 and logits.shape[1] > 1):
        raise ValueError("logits must be FP16, BF16 or float32 [rows, vocab] with contiguous rows")
    rows, vocab = logits.shape
    if tokens.dtype != torch.int32 or tokens.shape != (rows,) or not tokens.is_contiguous():
        raise ValueError(f"tokens must be contiguous int32 [{rows}]")
    if not 0 <= top <= min(MAX_TOP, vocab):
        raise ValueError(f"top must be 0..{MAX_TOP} and at most the vocabulary")
    score = torch.empty(2, rows, dtype=torch.float32, device=dev)
    ids = torch.empty(rows, top, dtype=torch.int32, device=dev)
    lps = torch.empty(rows, top, dtype=torch.float32, device=dev)
    with torch.cuda.device(dev):
        _lib.call("pp_token_logprobs", logits.data_ptr(), _DTYPES[logits.dtype], logits.stride(0), rows, vocab,
                  tokens.data_ptr(), top, score[0].data_ptr(), score[1].data_ptr(), ids.data_ptr(), lps.data_ptr(),
                  _lib.ptr(status), _lib.stream_handle(dev))
    return TokenLogprobs(score[0], score[1], ids, lps)
