"""Logarithms of given tokens' probabilities, and the clipped policy loss with a KL term (csrc/kernels/losses.cu), from a model's logits as they come.

    lp = x[token] / temperature - ln sum_j exp(x_j / temperature)
    loss = sum w (-min(q A, clip(q, 1 - low, 1 + high) A) + kl (exp(d) - d - 1)) / sum w,   q = exp(lp - old),  d = reference - lp

Nothing of the logits' size is written but their gradient.  A row of weight 0 is not read, has a logarithm of 0 and a gradient of 0: padding, prompts, and the
last position of a sequence, whose next token nobody knows, are left out this way, at no copy.  A token outside the vocabulary under another weight gives NaN.
Logits of -inf have no probability; a row of nothing else gives NaN, as one with NaN or +inf does.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional, Tuple, Union

import torch

from .._ext import require_native
from .checks import ordinary


class PolicyLoss(NamedTuple):
    loss: torch.Tensor              # one fp32 value, with a gradient to the logits
    logprobs: torch.Tensor          # like tokens, fp32: what a next step takes as ``old``, or a reference's
    divergence: torch.Tensor        # weighted mean of exp(d) - d - 1; 0 without a reference
    clipped: torch.Tensor           # weighted share of tokens whose ratio is held at a border


def _check(what: str, logits: torch.Tensor, tokens: torch.Tensor, temperature: float) -> None:
    if logits.dim() < 1 or logits.shape[-1] == 0:
        raise ValueError(f"{what}: logits [..., vocab] expected, not {tuple(logits.shape)}")
    if tokens.shape != logits.shape[:-1]:
        raise ValueError(f"{what}: tokens {tuple(logits.shape[:-1])} expected, not {tuple(tokens.shape)}")
    if tokens.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"{what}: tokens of int64 or int32 expected, not {tokens.dtype}")
    if tokens.device != logits.device:
        raise RuntimeError(f"{what}: tokens on {logits.device} expected, not on {tokens.device}")
    if not (1e-30 <= temperature < math.inf):
        raise ValueError(f"{what}: a temperature of {temperature}")


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, temperature: float = 1.0) -> torch.Tensor:
    """logits [..., vocab]; tokens [...]: the logarithm of each token's probability in its row, fp32.  On the GPU bf16, fp16 and fp32 logits whose rows are
    contiguous and lie at one or two distances (a slice of positions, say; others are copied); on the CPU any floating type.  What preference losses and
    sequence likelihoods are sums of."""
    if logits.is_cuda and ordinary(logits):
        return require_native().token_logprobs(logits, tokens, temperature)
    _check("token_logprobs", logits, tokens, temperature)
    ok = (tokens >= 0) & (tokens < logits.shape[-1])
    return torch.where(ok, _plain_logprobs(logits, tokens, temperature), math.nan).float()


def _plain_logprobs(logits, tokens, temperature):
    return torch.log_softmax(logits.double() / temperature, -1).gather(-1, tokens.long().clamp(0, logits.shape[-1] - 1).unsqueeze(-1)).squeeze(-1)


def _like_tokens(what: str, t: Optional[torch.Tensor], tokens: torch.Tensor) -> Optional[torch.Tensor]:
    if t is None:
        return None
    if t.device != tokens.device:
        raise RuntimeError(f"policy_loss: {what} on {tokens.device} expected, not on {t.device}")
    if t.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"policy_loss: {what} gets no gradient; detach it")
    if t.dtype == torch.float32 and t.shape == tokens.shape:
        return t.contiguous()
    return t.to(torch.float32).broadcast_to(tokens.shape).contiguous()


def policy_loss(logits: torch.Tensor, tokens: torch.Tensor, old: torch.Tensor, advantages: torch.Tensor, *, weights: Optional[torch.Tensor] = None,
                reference: Optional[torch.Tensor] = None, kl: float = 0.0, clip: Tuple[float, float] = (0.2, 0.2), temperature: float = 1.0,
                total: Union[None, float, torch.Tensor] = None) -> PolicyLoss:
    """logits [..., vocab]; tokens [...]; old: the logarithms of the tokens' probabilities when they were drawn (ops/sampling.py gives them); advantages,
    weights (a mask, say) and reference are broadcast to the tokens.  ``total``: what the weighted sums are divided by in place of the weights' own sum, a number
    or one fp32 value on the device, where a batch is spread over several calls or ranks; a sum of 0 gives a loss of 0.  A ratio exactly at its border still
    has a gradient.  Only the logits get one, and it cannot be differentiated again on the GPU."""
    low, high = clip
    if logits.is_cuda and ordinary(logits):
        return PolicyLoss(*require_native().policy_loss(logits, tokens, old, advantages, reference, weights, total, kl, low, high, temperature))
    _check("policy_loss", logits, tokens, temperature)
    if not (0 <= low < math.inf and 0 <= high < math.inf and 0 <= kl < math.inf):
        raise ValueError(f"policy_loss: clip {clip}, kl {kl}")
    old, advantages, weights, reference = (_like_tokens(n, t, tokens) for n, t in (("old", old), ("advantages", advantages), ("weights", weights), ("reference", reference)))
    if isinstance(total, torch.Tensor):
        if total.numel() != 1 or total.device != logits.device:
            raise ValueError("policy_loss: total, a number or one value on the logits' device")
        if total.requires_grad and torch.is_grad_enabled():
            raise RuntimeError("policy_loss: total gets no gradient; detach it")
        total = total.reshape(()).float()
    elif total is not None:
        total = torch.full((), float(total), device=logits.device)
    return _plain_policy(logits, tokens, old, advantages, weights, reference, kl, low, high, temperature, total)


def _plain_policy(logits, tokens, old, advantages, weights, reference, kl, low, high, temperature, total):
    w = torch.ones(tokens.shape, dtype=torch.float64, device=logits.device) if weights is None else weights.double()
    counts = w != 0
    x = torch.where(counts.unsqueeze(-1), logits, torch.zeros_like(logits))          # rows of weight 0 are not looked at
    ok = (tokens >= 0) & (tokens < logits.shape[-1])
    lp = torch.where(counts, torch.where(ok, _plain_logprobs(x, tokens, temperature), math.nan), 0.0)
    total = w.sum() if total is None else total.double()
    share = torch.where(total == 0, 0.0, w / torch.where(total == 0, 1.0, total))

    def mean(t):
        return (share * torch.where(counts, t, 0.0)).sum()

    A, q = advantages.double(), torch.exp(torch.where(counts, lp - old.double(), 0.0))
    free, held = q * A, q.clamp(1 - low, 1 + high) * A
    term = -torch.where((free <= held) | q.isnan(), free, held.detach())
    far = torch.zeros_like(lp)
    if reference is not None:
        d = torch.where(counts, reference.double() - lp, 0.0)
        far = torch.expm1(d) - d
        term = term + kl * far
    return PolicyLoss(mean(term).float(), lp.detach().float(), mean(far.detach()).float(), mean((free > held).double()).float())
