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


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, top, temperature):
        logprobs, entropy, stats, top_logprobs, top_ids = _ops.token_logprobs(logits, tokens, None, top, temperature)
        ctx.save_for_backward(logits, tokens, entropy, stats, top_ids)
        ctx.temperature = temperature
        ctx.set_materialize_grads(False)
        if top_ids is not None:
            ctx.mark_non_differentiable(top_ids)
        return logprobs, entropy, top_logprobs, top_ids

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_logprobs, grad_entropy, grad_top_logprobs, _):
        logits, tokens, entropy, stats, top_ids = ctx.saved_tensors
        if grad_logprobs is None and grad_entropy is None and grad_top_logprobs is None:
            return None, None, None, None
        return _ops.token_logprobs_backward(logits, tokens, entropy, stats, top_ids, ctx.temperature, grad_logprobs,
                                            grad_entropy, grad_top_logprobs), None, None, None


def token_logprobs(logits, tokens=None, *, rows=None, top=0, temperature=1.0):
    """Log-probability of each row's token under softmax(logits / temperature), the row's entropy
    and its `top` (at most 32) likeliest entries.

    ``logits`` ([batch,] [rows,] vocabulary), bf16 / fp16 / fp32, unit stride on the vocabulary;
    ``tokens`` int64 of the leading shape, or None. A row whose token is negative is skipped (not
    read; zeros, ids -1, no gradient). ``rows`` (batch, n) int64 takes row rows[b, i] of sequence
    b's logits for output (b, i) (negative: skipped); no gradient flows through it. A token outside
    the vocabulary or a row outside the logits is skipped and reported by ``_ops.device_error``.
    A row of -inf alone has log-probability -inf and entropy 0; NaN or +inf in a row makes its
    numbers NaN. The outputs carry a gradient to ``logits`` (not twice differentiable).
    """
    temperature = float(temperature)
    if logits.requires_grad and torch.is_grad_enabled():
        if rows is not None:
            raise ValueError('token_logprobs: rows selects verified rows of a rollout and carries no gradient; '
                             'detach the logits or index them first')
        return TokenLogprobs(*_TokenLogprobs.apply(logits, tokens, top, temperature))
    logprobs, entropy, _, top_logprobs, top_ids = _ops.token_logprobs(logits, tokens, rows, top, temperature)
    return TokenLogprobs(logprobs, entropy, top_logprobs, top_ids)
