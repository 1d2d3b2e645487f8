"""Scores of given tokens from rows of logits.

``token_logprobs`` returns, in one pass over the logits, what a log-likelihood
evaluation or a server's ``logprobs`` answer takes from a whole
``log_softmax``: the log probability of each row's target token, the entropy
of the row's distribution and its ``top`` most likely tokens.  It stands next
to the greedy sampler's ``fdl_softmax_argmax``; no probabilities are
materialised.  Forward only: nothing is recorded for autograd, and logits with a
forward-mode tangent are refused.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch
from torch.compiler import is_compiling

from . import _lib

MAX_TOP = 32

_lib.load_if_built()


class TokenScores(NamedTuple):
    logprob: torch.Tensor                 # fp32 [rows]
    entropy: torch.Tensor                 # fp32 [rows], nats
    top_logprob: Optional[torch.Tensor]   # fp32 [rows, top], descending
    top_token: Optional[torch.Tensor]     # int64 [rows, top]


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, top: int = 0) -> TokenScores:
    """Log probability of ``targets`` (int64, one per row; below 0: no target,
    scored 0), entropy and the ``top`` <= 32 best tokens of ``logits``
    [rows, vocab] (bf16, fp16 or fp32; rows may be strided, or one row
    expanded to score several targets).

    Equal logits rank by index, lower first.  -inf logits are tokens of
    probability 0.  A row that is no distribution (NaN, +inf, all -inf) comes
    out as NaN with tokens -1, and is reported in the device status.  The four
    results share one allocation: whoever keeps one alone, or saves it, clones
    it.
    """
    if logits.dim() != 2:
        raise ValueError(f"token_logprobs: logits must be [rows, vocab], got {tuple(logits.shape)}")
    if not 0 <= top <= min(MAX_TOP, logits.shape[1]):
        raise ValueError(f"token_logprobs: top={top} is outside [0, min({MAX_TOP}, vocab={logits.shape[1]})]")
    # straight into the library for plain CUDA tensors, through torch.ops.fdl
    # otherwise and while compiling
    if is_compiling():
        r = torch.ops.fdl.token_logprobs(logits, targets, top)
    else:
        r = _lib.direct().token_logprobs(logits, targets, top)
        if r is NotImplemented:
            r = torch.ops.fdl.token_logprobs(logits, targets, top)
    logprob, entropy, top_logprob, top_token = r
    if not top:
        top_logprob = top_token = None
    return TokenScores(logprob, entropy, top_logprob, top_token)
