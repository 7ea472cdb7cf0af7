"""Log probabilities of given tokens on the sm_100a kernels, with the entropy of their
distributions and the likeliest alternatives.

    logprob = x[t] - ln sum e^x          the given token t's
    entropy = - sum p ln p               p = e^x / sum e^x, in nats

over the last dimension of logits x [..., vocab] in bfloat16, float16 or float32. Sums and
results are float32. The logits are read once forward and once back, and nothing of their
size is kept but the gradient.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from .._ext import C
from .flash import host_status


class TokenLogprobs(NamedTuple):
    """logprobs, entropy: float32, the targets' shape. top_logprobs (float32), top_indices
    (int64): [..., top], the likeliest first, of equally likely ones the lowest index; None
    without `top`."""
    logprobs: torch.Tensor
    entropy: torch.Tensor
    top_logprobs: Optional[torch.Tensor]
    top_indices: Optional[torch.Tensor]


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, top: int = 0,
                   ignore_index: int = -100) -> TokenLogprobs:
    """TokenLogprobs of the tokens targets [...] under logits [..., vocab].

    targets: int32 or int64. Where one is ignore_index its logprob is 0 and passes no
    gradient; the entropy and the alternatives are the row's all the same. A target outside
    the vocab gives NaN, no gradient, and KernelStatusError at a later call (this one, a
    paged call that raises, check_errors()). top: 0 to 32. Logits of -inf have probability
    0; in a row of nothing else every token's logprob is -inf, the entropy 0, and no
    gradient passes. A NaN or +inf makes its row's results NaN, and counts as the largest
    among the alternatives.
    logprobs and entropy are differentiable (once, in reverse mode) in logits, the
    alternatives are not. Strided rows are read in place; the gradient is contiguous."""
    if logits.is_cuda:
        h = host_status(logits.device)
        h.poll()  # an error of an earlier call surfaces here
        status = h.word
    else:
        status = torch.zeros(1, dtype=torch.int32)
    return TokenLogprobs(*C().token_logprobs(logits, targets, top, ignore_index, status))
