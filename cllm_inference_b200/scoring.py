"""What a sampler reports of logits (include/cllm_cuda.h, cllm_cuda_token_scores).

The reference samples greedily and reports no probabilities
(src/core/sampler.cpp:32-34); this gives, per row of logits, the log
probability and the rank of a token, the entropy and the best alternatives.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib

_raw_stream = torch._C._cuda_getCurrentRawStream  # torch's current stream of a device, as an integer
_current_device = torch._C._cuda_getDevice


class TokenScores(NamedTuple):
    logprob: torch.Tensor | None  # fp32 [rows], None without tokens
    rank: torch.Tensor | None     # int32 [rows], 0: the most likely
    entropy: torch.Tensor         # fp32 [rows], nats
    top_ids: torch.Tensor         # int32 [rows][top_k]
    top_logprobs: torch.Tensor    # fp32 [rows][top_k]


def token_scores(logits: torch.Tensor, tokens: torch.Tensor | None = None, top_k: int = 0) -> TokenScores:
    """Scores of fp32 CUDA logits [rows][vocab] (rows apart or one expanded) and int32 tokens of one device, on torch's
    current stream of it."""
    device = logits.get_device()
    if device < 0 or logits.dtype != torch.float32 or logits.dim() != 2 or (
            logits.shape[1] > 1 and logits.stride(1) != 1):
        raise _lib.CudaError(_lib.ERR_INVALID_ARG, "token_scores: logits must be a 2-D fp32 CUDA tensor with dense rows")
    if _current_device() != device:  # the C call launches on the current device
        with torch.cuda.device(device):
            return token_scores(logits, tokens, top_k)
    rows, vocab = logits.shape
    if tokens is not None and (tokens.get_device() != device or tokens.dtype != torch.int32 or tokens.numel() != rows or
                               not tokens.is_contiguous()):
        raise _lib.CudaError(_lib.ERR_INVALID_ARG, "token_scores: tokens must be int32, contiguous, one per row, beside the logits")
    k = max(0, top_k)
    entropy = logits.new_empty(rows)
    logprob = rank = None
    tp = lp = rp = 0
    if tokens is not None:
        logprob, rank = torch.empty_like(entropy), torch.empty_like(tokens)
        tp, lp, rp = tokens.data_ptr(), logprob.data_ptr(), rank.data_ptr()
    logprobs = logits.new_empty((rows, k))
    ids = torch.empty_like(logprobs, dtype=torch.int32)
    rc = _lib.load().cllm_cuda_token_scores(
        logits.data_ptr(), logits.stride(0) if rows > 1 else vocab, rows, vocab, tp, top_k, lp, entropy.data_ptr(),
        rp, ids.data_ptr(), logprobs.data_ptr(), _raw_stream(device))
    if rc:
        _lib.check(rc)
    return TokenScores(logprob, rank, entropy, ids, logprobs)
