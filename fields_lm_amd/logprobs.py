"""Log probabilities of given tokens, with entropy and top alternatives and their gradients, on the HIP path only
(``csrc/logprobs.hip``, host side ``csrc/host.cpp``): what a loss starts from, a scored text consists of and a
generation loop returns beside each token."""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _native as nat
from ._train import _stock_grads


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor                # [...] fp32
    entropy: Optional[torch.Tensor]       # [...] fp32
    top_logprobs: Optional[torch.Tensor]  # [..., K] fp32, largest first
    top_tokens: Optional[torch.Tensor]    # [..., K] int64


def _ops(logits, tokens, top_tokens, temperature, ignore_index):
    """(logprobs, entropy, top logprobs) in stock ops, for a differentiable backward."""
    d = logits.float()
    top = d.detach().amax(-1, keepdim=True)
    empty = top == float("-inf")
    d = (d - torch.where(empty, 0.0, top)) / temperature
    e = torch.exp(d)
    total = torch.where(empty, 1.0, e.sum(-1, keepdim=True))
    lp = d - torch.log(total)
    kept = tokens != ignore_index
    at = torch.where(kept, tokens, 0)
    inside = (at >= 0) & (at < logits.shape[-1])
    got = lp.gather(-1, torch.where(inside, at, 0)[..., None])[..., 0]
    # (a product with NaN, not a choice of it: the gradient of a token outside the vocabulary is NaN)
    factor = torch.where(inside | empty[..., 0], 1.0, float("nan"))
    got = torch.where(kept & ~empty[..., 0], got * factor, 0.0)
    live = e > 0
    entropy = torch.log(total) - torch.where(live, e * torch.where(live, d, 0.0), 0.0).sum(-1, keepdim=True) / total
    tops = torch.where(empty, 0.0, lp.gather(-1, top_tokens)) if top_tokens is not None else None
    return got, entropy[..., 0], tops


def stock_gradient(logits, tokens, top_tokens, temperature, ignore_index, *grads) -> Optional[torch.Tensor]:
    """The logits' gradient in stock ops, for a backward that must itself be differentiable. Its zeros are the kernel's:
    a row whose gradients are all 0 passes nothing whatever its logits hold, and neither does a gradient of 0 for a token
    outside the vocabulary."""
    g, h, top = grads
    quiet = torch.ones(tokens.shape, dtype=torch.bool, device=tokens.device)
    if g is not None:
        quiet = (g == 0) | (tokens == ignore_index)
        tokens = torch.where(quiet & ((tokens < 0) | (tokens >= logits.shape[-1])), ignore_index, tokens)
    if h is not None:
        quiet = quiet & (h == 0)
    if top is not None:
        quiet = quiet & (top == 0).all(-1)
    # Only rows with NaN or +inf are hidden (0 times those is no 0): the others' zeros come about, and stay a function
    # of the gradients.
    hidden = (quiet & ~(logits.detach().amax(-1) < float("inf")))[..., None]
    given = [(i, o) for i, o in enumerate(grads) if o is not None]

    def fn(x):
        outs = _ops(torch.where(hidden, 0.0, x), tokens, top_tokens, temperature, ignore_index)
        return tuple(outs[i] for i, _ in given)

    return _stock_grads(fn, (logits,), tuple(o for _, o in given))[0]


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, temperature: float = 1.0, top_k: int = 0,
                   entropy: bool = False, ignore_index: int = -100) -> TokenLogprobs:
    """Log probabilities of ``tokens`` under softmax(logits / temperature), in one pass over the logits.

    logits [..., V] (V up to 2^23) fp32 or bf16 on a ROCm device, rows any distance apart (a slice of positions is
    read in place); tokens [...] int64 on the same device. temperature: 2^-20 to 2^20. ``entropy`` adds each row's
    entropy, ``top_k`` (up to 64) its largest logits' log probabilities and tokens: largest first, of equal ones the
    lowest index first, NaN above all. Everything is computed and returned in fp32.

    A token equal to ``ignore_index`` has log probability 0 and passes no gradient; one outside the vocabulary has
    NaN, and so has its gradient. -inf masks a logit; a row of -inf alone has log probabilities -inf, entropy 0 and
    gradient 0; NaN or +inf in a row make its results NaN. Rows whose incoming gradients are all 0 get zeros
    without their logits being read.

    Gradients flow to ``logits`` from the log probabilities, the entropy and the alternatives' log probabilities. A
    backward that is to be differentiated itself (``create_graph``) runs stock operations, with the same zeros and NaN.
    Under graph capture the backward pass is refused while a graph of the default stream holds the logits' leaves.
    """
    return TokenLogprobs(*nat.host().token_logprobs(logits, tokens, temperature, top_k, entropy, ignore_index))
