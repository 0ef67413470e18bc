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
    index = logits.get_device()
    if index < 0 or tokens.get_device() != index or (status is not None and status.get_device() != index):
        _lib.require_cuda(logits, tokens, status)
    dtype = _DTYPES.get(logits.dtype)
    if logits.dim() != 2 or dtype is None or (logits.stride(1) != 1 and logits.shape[1] > 1):
        raise ValueError("logits must be FP16, BF16 or float32 [rows, vocab] with contiguous rows")
    rows, vocab = logits.shape
    if tokens.dtype is not torch.int32 or tokens.shape != (rows,) or not tokens.is_contiguous():
        raise ValueError(f"tokens must be contiguous int32 [{rows}]")
    if status is not None and (status.dtype is not torch.int32 or status.numel() < 1):
        raise ValueError("status must be an int32 tensor")
    if not 0 <= top <= min(MAX_TOP, vocab):
        raise ValueError(f"top must be 0..{MAX_TOP} and at most the vocabulary")
    logprob = torch.empty_like(tokens, dtype=torch.float32)
    entropy = torch.empty_like(logprob)
    ids = tokens.new_empty((rows, top))
    lps = torch.empty_like(ids, dtype=torch.float32)
    fn = _lib.load().pp_token_logprobs
    args = (logits.data_ptr(), dtype, logits.stride(0), rows, vocab, tokens.data_ptr(), top, logprob.data_ptr(),
            entropy.data_ptr(), ids.data_ptr(), lps.data_ptr(), _lib.ptr(status), _lib.stream_handle(logits.device))
    if torch.cuda.current_device() != index:
        with torch.cuda.device(index):
            rc = fn(*args)
    else:
        rc = fn(*args)
    if rc:
        _lib.check(rc)
    return TokenLogprobs(logprob, entropy, ids, lps)
