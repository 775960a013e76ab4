"""What ranks the continuations of a text, from the logits of a step.

    token_log_probs   log probability of given tokens, entropy, the most likely tokens

Everything is enqueued on the current stream of the logits' device, nothing synchronises, and the call can be captured in a CUDA graph.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _native
from .ops import load_ops

load_ops()
_scores = torch.ops.tensorrt.b200_token_log_probs.default


class TokenScores(NamedTuple):
    log_probs: torch.Tensor         # float32 [..]: of the given tokens
    entropy: torch.Tensor           # float32 [..], in nats
    top_log_probs: torch.Tensor     # float32 [.., top]
    top_tokens: torch.Tensor        # int32 [.., top]


def token_log_probs(logits: torch.Tensor, tokens: torch.Tensor | None = None, *, top: int = 0, scale: float = 1.0) -> TokenScores:
    """Of softmax(logits * scale) over the last dimension (float32, float16 or bfloat16 [.., vocabulary], computed in 32 bits): the log probability of
    `tokens` [..] (int32 or int64; 0 for one outside the vocabulary, as padding has, and without tokens), the entropy, and the `top` (up
    to 64) most likely tokens, descending, of equal ones the lower first.  Logits of -inf have no probability.  A row whose largest logit is not
    finite (nothing but -inf, an infinity, a NaN) has no distribution: NaN, as torch.log_softmax gives."""
    args = (logits, tokens, top, float(scale))
    out = _native.token_log_probs(*args)
    return TokenScores(*(_scores(*args) if out is None else out))
