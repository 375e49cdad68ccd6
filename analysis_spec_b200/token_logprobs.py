"""Log-probabilities of given tokens under rows of logits, with entropy and top alternatives.

What a rollout and its training step take from the logits: the log-probabilities of the
emitted tokens (kept for the policy ratio), the entropy, the greedy sample and the draft's
candidates (top alternatives), and for training their gradient. Replaces the
log_softmax / gather / argmax / topk sequence on a float32 copy of the logits: one launch
reads each row once in its own dtype, one more launch writes the gradient.
"""
from typing import NamedTuple, Optional

import torch

from . import _ops


class TokenLogprobs(NamedTuple):
    logprobs: Optional[torch.Tensor]      # float32, the tokens' shape; None without tokens
    entropy: torch.Tensor                 # float32, one per row
    top_logprobs: Optional[torch.Tensor]  # float32 (..., top); None with top = 0
    top_ids: Optional[torch.Tensor]       # int64 (..., top), best first, equal logits by the lower id


def token_logprobs(logits, tokens=None, *, rows=None, top=0, temperature=1.0):
    """Log-probability of each row's token under softmax(logits / temperature), the row's entropy
    and its `top` (at most 32) likeliest entries.

    ``logits`` ([batch,] [rows,] vocabulary), bf16 / fp16 / fp32, unit stride on the vocabulary;
    ``tokens`` int64 of the leading shape, or None. A row whose token is negative is skipped (not
    read; zeros, ids -1, no gradient). ``rows`` (batch, n) int64 takes row rows[b, i] of sequence
    b's logits for output (b, i) (negative: skipped); no gradient flows through it. A token outside
    the vocabulary or a row outside the logits is skipped and reported by ``_ops.device_error``.
    A row of -inf alone has log-probability -inf and entropy 0; NaN or +inf in a row makes its
    numbers NaN. The outputs carry a gradient to ``logits`` (not twice differentiable;
    forward-mode tangents are refused). Before a backward pass is captured into a CUDA graph, drop every
    eager graph of the same leaves: torch ends the process otherwise (refused where ``logits`` are the leaf).
    """
    return TokenLogprobs(*_ops.token_logprobs(logits, tokens, rows, top, temperature))
