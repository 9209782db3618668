"""What a sampler reports of logits (include/cllm_cuda.h, cllm_cuda_token_scores).

The reference samples greedily and reports no probabilities
(src/core/sampler.cpp:32-34); this gives, per row of logits, the log
probability and the rank of a token, the entropy and the best alternatives.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib


class TokenScores(NamedTuple):
    logprob: torch.Tensor | None  # fp32 [rows], None without tokens
    rank: torch.Tensor | None     # int32 [rows], 0: the most likely
    entropy: torch.Tensor         # fp32 [rows], nats
    top_ids: torch.Tensor         # int32 [rows][top_k]
    top_logprobs: torch.Tensor    # fp32 [rows][top_k]


def token_scores(logits: torch.Tensor, tokens: torch.Tensor | None = None, top_k: int = 0) -> TokenScores:
    """Scores of fp32 CUDA logits [rows][vocab] (any row stride), on torch's current stream."""
    if not logits.is_cuda or logits.dtype != torch.float32 or logits.dim() != 2 or (
            logits.shape[1] > 1 and logits.stride(1) != 1):
        raise _lib.CudaError(_lib.ERR_INVALID_ARG, "token_scores: logits must be a 2-D fp32 CUDA tensor with dense rows")
    rows, vocab = logits.shape
    if tokens is not None and (not tokens.is_cuda or tokens.dtype != torch.int32 or tokens.numel() != rows or
                               not tokens.is_contiguous()):
        raise _lib.CudaError(_lib.ERR_INVALID_ARG, "token_scores: tokens must be int32, contiguous, one per row")
    dev = logits.device
    entropy = torch.empty(rows, dtype=torch.float32, device=dev)
    logprob = rank = None
    if tokens is not None:
        logprob = torch.empty(rows, dtype=torch.float32, device=dev)
        rank = torch.empty(rows, dtype=torch.int32, device=dev)
    ids = torch.empty((rows, max(0, top_k)), dtype=torch.int32, device=dev)
    logprobs = torch.empty((rows, max(0, top_k)), dtype=torch.float32, device=dev)
    _lib.check(_lib.load().cllm_cuda_token_scores(
        logits.data_ptr(), logits.stride(0) if rows > 1 else vocab, rows, vocab,
        0 if tokens is None else tokens.data_ptr(), top_k, 0 if tokens is None else logprob.data_ptr(),
        entropy.data_ptr(), 0 if tokens is None else rank.data_ptr(), ids.data_ptr(), logprobs.data_ptr(),
        torch.cuda.current_stream(dev).cuda_stream))
    return TokenScores(logprob, rank, entropy, ids, logprobs)
