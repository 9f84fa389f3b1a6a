"""Log probabilities of given tokens, with entropy and top alternatives and their gradients, on the HIP path only
(``csrc/logprobs.hip``): what a loss starts from, a scored text consists of and a generation loop returns
beside each token."""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import _native as nat
from ._dispatch import no_grad_needed
from ._train import _stock_grads

MAX_TOP, MAX_VOCAB = 64, 1 << 23
MIN_TEMPERATURE, MAX_TEMPERATURE = 2.0 ** -20, 2.0 ** 20


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor                # [...] fp32
    entropy: Optional[torch.Tensor]       # [...] fp32
    top_logprobs: Optional[torch.Tensor]  # [..., K] fp32, largest first
    top_tokens: Optional[torch.Tensor]    # [..., K] int64


def _strides(t: torch.Tensor, dims: int) -> Optional[Tuple[int, int, int, int]]:
    """The first ``dims`` dimensions of ``t`` as (outer, inner) with their strides; None where two do not do."""
    groups = []  # (size, stride), dimensions that step as one merged
    for size, stride in zip(t.shape[:dims], t.stride()[:dims]):
        if size == 1:
            continue
        if groups and groups[-1][1] == size * stride:
            groups[-1] = (groups[-1][0] * size, stride)
        else:
            groups.append((size, stride))
    if len(groups) > 2:
        return None
    groups = [(1, 0)] * (2 - len(groups)) + groups
    return groups[0][0], groups[1][0], groups[0][1], groups[1][1]


def _rows(logits: torch.Tensor, tokens: torch.Tensor):
    """(logits, tokens, row arguments of the library's calls): both seen as outer x inner rows; what does not
    step like that is copied."""
    if logits.stride(-1) != 1 and logits.shape[-1] > 1:
        logits = logits.contiguous()
    dims = tokens.ndim
    if logits.is_contiguous() and tokens.is_contiguous():
        return logits, tokens, (1, tokens.numel(), 0, logits.shape[-1]), (0, 1)
    a, b = _strides(logits, dims), _strides(tokens, dims)
    if a is None:
        logits = logits.contiguous()
        a = _strides(logits, dims)
    if b is None:
        tokens = tokens.contiguous()
        b = _strides(tokens, dims)
    if a[:2] != b[:2]:  # one of them is merged further than the other: split it as the other is
        rows = tokens.numel()
        if a[:2] == (1, rows):
            a = (b[0], b[1], a[3] * b[1], a[3])
        elif b[:2] == (1, rows):
            b = (a[0], a[1], b[3] * a[1], b[3])
        else:
            tokens = tokens.contiguous()
            b = (a[0], a[1], a[1], 1)
    return logits, tokens, a, b[2:]


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
    got = torch.where(kept & ~empty[..., 0], got * torch.where(inside, 1.0, float("nan")), 0.0)
    live = e > 0
    entropy = torch.log(total) - torch.where(live, e * torch.where(live, d, 0.0), 0.0).sum(-1, keepdim=True) / total
    tops = torch.where(empty, 0.0, lp.gather(-1, top_tokens)) if top_tokens is not None else None
    return got, entropy[..., 0], tops


def _forward(logits, tokens, temperature, top_k, want_entropy, ignore_index, want_stats):
    """(logprobs, entropy, top logprobs, top tokens, statistics for the backward), None where not wanted."""
    lib, dev, vocab = nat.load(), logits.device, logits.shape[-1]

    def new(shape, dtype=torch.float32):
        return torch.empty(shape, device=dev, dtype=dtype)

    shape = tuple(tokens.shape)
    logprobs = new(shape)
    entropy = new(shape) if want_entropy else None
    top = new((*shape, top_k)) if top_k else None
    top_tokens = new((*shape, top_k), torch.int64) if top_k else None
    stats = new((*shape, 2)) if want_stats else None
    x, t, (outer, inner, so, si), (to, ti) = _rows(logits, tokens)
    code = nat.dtype_code(x.dtype)
    nbytes = int(lib.fl_token_logprobs_workspace_bytes(outer * inner, vocab, code, top_k))
    ws = new((nbytes,), torch.uint8) if nbytes else None
    with nat.on(dev):
        nat.check(lib.fl_token_logprobs(
            nat.ptr(x), code, outer, inner, vocab, so, si, nat.ptr(t), to, ti, ignore_index, temperature, top_k,
            nat.ptr(logprobs), nat.ptr(entropy), nat.ptr(top), nat.ptr(top_tokens), nat.ptr(stats), nat.ptr(ws), nbytes,
            nat.stream_handle(dev)), "fl_token_logprobs")
    return logprobs, entropy, top, top_tokens, stats


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, temperature, top_k, want_entropy, ignore_index):
        ctx.set_materialize_grads(False)
        *outs, stats = _forward(logits, tokens, temperature, top_k, want_entropy, ignore_index, True)
        _, entropy, _, top_tokens = outs
        ctx.save_for_backward(logits, tokens, stats, entropy, top_tokens)
        ctx.args = temperature, top_k, ignore_index
        if top_tokens is not None:
            ctx.mark_non_differentiable(top_tokens)
        return tuple(outs)

    @staticmethod
    def backward(ctx, g_lp, g_entropy, g_top, _):
        logits, tokens, stats, entropy, top_tokens = ctx.saved_tensors
        temperature, top_k, ignore_index = ctx.args
        none = (None,) * 5
        if g_lp is None and g_entropy is None and g_top is None:
            return (None, *none)
        if torch.is_grad_enabled():  # a backward that must itself be differentiable
            given = [(i, g) for i, g in enumerate((g_lp, g_entropy, g_top)) if g is not None]

            def fn(x):
                outs = _ops(x, tokens, top_tokens, temperature, ignore_index)
                return tuple(outs[i] for i, _ in given)

            return (_stock_grads(fn, (logits,), tuple(g for _, g in given))[0], *none)
        g_lp, g_entropy, g_top = (None if g is None else g.contiguous() for g in (g_lp, g_entropy, g_top))
        out = torch.empty(logits.shape, device=logits.device, dtype=logits.dtype)
        x, t, (outer, inner, so, si), (to, ti) = _rows(logits, tokens)
        with nat.on(logits.device):
            nat.check(nat.load().fl_token_logprobs_backward(
                nat.ptr(x), nat.dtype_code(x.dtype), outer, inner, logits.shape[-1], so, si, nat.ptr(t), to, ti,
                ignore_index, temperature, top_k, nat.ptr(stats), nat.ptr(entropy), nat.ptr(top_tokens), nat.ptr(g_lp),
                nat.ptr(g_entropy), nat.ptr(g_top), nat.ptr(out), nat.stream_handle(logits.device)),
                "fl_token_logprobs_backward")
        return (out, *none)


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, temperature: float = 1.0, top_k: int = 0,
                   entropy: bool = False, ignore_index: int = -100) -> TokenLogprobs:
    """Log probabilities of ``tokens`` under softmax(logits / temperature), in one pass over the logits.

    logits [..., V] fp32 or bf16 on a ROCm device, rows any distance apart (a slice of positions is read in place);
    tokens [...] int64 on the same device. ``entropy`` adds each row's entropy, ``top_k`` (up to 64) its largest
    logits' log probabilities and tokens: largest first, of equal ones the lowest index first, NaN above all.
    Everything is computed and returned in fp32.

    A token equal to ``ignore_index`` has log probability 0 and passes no gradient; one outside the vocabulary has
    NaN, and so has its gradient. -inf masks a logit; a row of -inf alone has log probabilities -inf, entropy 0 and
    gradient 0; NaN or +inf in a row make its results NaN. Rows whose incoming gradients are all 0 get zeros
    without their logits being read.

    Gradients flow to ``logits`` from the log probabilities, the entropy and the alternatives' log probabilities.
    """
    if not logits.is_cuda:
        raise RuntimeError("token_logprobs requires a ROCm (cuda) device")
    if logits.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"logits must be float32 or bfloat16, got {logits.dtype}")
    if tokens.dtype != torch.int64:
        raise TypeError(f"tokens must be int64, got {tokens.dtype}")
    if tokens.device != logits.device:
        raise ValueError("logits and tokens must be on one device")
    if logits.ndim < 1 or tokens.shape != logits.shape[:-1]:
        raise ValueError(f"tokens {tuple(tokens.shape)} must be the logits' rows {tuple(logits.shape)}")
    vocab, top_k, temperature = logits.shape[-1], int(top_k), float(temperature)
    if not 0 < vocab <= MAX_VOCAB:
        raise ValueError(f"a row must have 1 to {MAX_VOCAB} logits, got {vocab}")
    if not MIN_TEMPERATURE <= temperature <= MAX_TEMPERATURE:
        raise ValueError(f"temperature must be {MIN_TEMPERATURE} to {MAX_TEMPERATURE}, got {temperature}")
    if not 0 <= top_k <= min(MAX_TOP, vocab):
        raise ValueError(f"top_k must be 0 to {min(MAX_TOP, vocab)}, got {top_k}")
    if tokens.numel() == 0:
        empty = logits.sum(-1, dtype=torch.float32)  # no rows; keeps the graph
        return TokenLogprobs(empty, empty.clone() if entropy else None,
                             empty[..., None].expand(*empty.shape, top_k).clone() if top_k else None,
                             tokens[..., None].expand(*tokens.shape, top_k).clone() if top_k else None)
    args = logits, tokens, temperature, top_k, bool(entropy), int(ignore_index)
    if no_grad_needed(logits) and forward_ad._current_level < 0:  # (a tangent is refused by the function, not lost)
        return TokenLogprobs(*_forward(*args, False)[:4])
    return TokenLogprobs(*_TokenLogprobs.apply(*args))
