"""The next tokens by chance (csrc/kernels/sampling.cu): temperature, top-k, top-p and min-p, drawn by uniform numbers that the caller gives.

The tokens of a row are taken in the order of their logits, largest first and of equals the lowest index first, with weights
exp((logit - largest) / temperature).  The first ``top_k`` stay; of these the first ones whose weights make up ``top_p`` of theirs; of these those of at
least ``min_p`` times the largest weight; one always.  The token is the first whose weight brings the running sum above ``u`` times the sum of those
left.  Sums run in 64 bits, so the same numbers give the same tokens wherever they are computed.

A temperature of 0 is the greedy choice.  A logit of -inf is never chosen; a row of nothing else gives token 0 with a logarithm of -inf.  A row with a
NaN gives its first NaN, as the greedy choice does, with a logarithm of NaN.
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Optional, Tuple, Union

import torch

from .._ext import require_native

Limit = Union[float, int, torch.Tensor]


def _limit(value: Limit, dtype, rows: int, device, name: str):
    """(tensor or None, value for all rows) as the kernel takes it."""
    if not isinstance(value, torch.Tensor):
        return None, value
    if value.dtype == dtype and value.shape == (rows,) and value.is_contiguous():      # the kernel sees to the device
        return value, 0
    if value.dim() == 0:
        value = value.expand(rows)
    if value.shape != (rows,):
        raise ValueError(f"sample: {name} of shape {tuple(value.shape)} for {rows} rows")
    if value.device != device:
        raise RuntimeError(f"sample: {name} on {device} expected, not on {value.device}")
    if dtype == torch.int32 and value.dtype != torch.int32:
        value = value.clamp(0, 2 ** 31 - 1)
    return value.to(dtype).contiguous(), 0


def sample(logits: torch.Tensor, u: torch.Tensor, temperature: Limit = 1.0, top_k: Limit = 0, top_p: Limit = 1.0,
           min_p: Limit = 0.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """logits [rows, vocab]; u [rows], fp32 or fp64 in [0, 1); the limits numbers, or tensors with one for each row (top_k 0, top_p 1 and min_p 0 leave
    nothing out).  Returns the tokens [rows] int64 and the logarithm of each one's probability among those that were left, fp32.
    On the GPU bf16 and fp16, and logarithms without a gradient; on the CPU any floating type."""
    if logits.dim() != 2 or logits.shape[1] == 0:
        raise ValueError(f"sample: logits [rows, vocab] expected, not {tuple(logits.shape)}")
    rows, dev = logits.shape[0], logits.device
    if u.shape != (rows,) or u.dtype not in (torch.float32, torch.float64):
        raise ValueError(f"sample: u [{rows}] of fp32 or fp64 expected, not {tuple(u.shape)} of {u.dtype}")
    if u.device != dev:
        raise RuntimeError(f"sample: u on {dev} expected, not on {u.device}")
    given = (_limit(temperature, torch.float32, rows, dev, "temperature"), _limit(top_k, torch.int32, rows, dev, "top_k"),
             _limit(top_p, torch.float32, rows, dev, "top_p"), _limit(min_p, torch.float32, rows, dev, "min_p"))
    if logits.is_cuda:
        if logits.stride(1) != 1:
            logits = logits.contiguous()
        (t, t_all), (k, k_all), (p, p_all), (m, m_all) = given
        return require_native().sample(logits, u.contiguous(), t, t_all, k, k_all, p, p_all, m, m_all)
    return _plain_sample(logits, u, *(torch.full((rows,), all_, dtype=torch.float64) if t is None else t.double() for t, all_ in given))


def _plain_sample(logits, u, temperature, top_k, top_p, min_p):
    tokens, logprobs = torch.zeros(len(u), dtype=torch.int64), torch.full((len(u),), -math.inf)
    for r in range(len(u)):
        x = logits[r].double()
        if x.isnan().any():
            tokens[r], logprobs[r] = x.isnan().nonzero()[0, 0], math.nan
            continue
        v, order = torch.sort(x, descending=True, stable=True)
        have = int((v > -math.inf).sum())
        if have == 0:
            continue
        if not float(temperature[r].float()) > 0:
            tokens[r], logprobs[r] = order[0], 0.0
            continue
        d = torch.where(v == v[0], torch.zeros_like(v), (v - v[0]) / temperature[r].float().double())[:have]
        w = d.exp()
        c = w.cumsum(0)
        k, p, m = int(top_k[r]), top_p[r].float().double(), min_p[r].float().double()
        n = k if 0 < k < have else have
        if p < 1:
            n = min(n, int((c < p * c[n - 1]).sum()) + 1)
        if m > 0:
            n = min(n, int((w >= m).sum()))
        n = max(n, 1)
        at = float(u[r])
        at = min(at, 1 - 2.0 ** -53) if at >= 0 else 0.0
        j = min(int((c <= at * c[n - 1]).sum()), n - 1)
        tokens[r], logprobs[r] = order[j], d[j] - c[n - 1].log()
    return tokens, logprobs


@dataclass
class Sampler:
    """What a model's ``choose`` takes in place of the greedy choice: draws by the numbers in ``u`` [rows], which the caller fills before every step
    (a captured step reads them anew), and leaves the logarithms of the probabilities in ``logprobs`` where that is given."""
    u: torch.Tensor
    temperature: Limit = 1.0
    top_k: Limit = 0
    top_p: Limit = 1.0
    min_p: Limit = 0.0
    logprobs: Optional[torch.Tensor] = None

    def __call__(self, logits: torch.Tensor) -> torch.Tensor:
        tokens, logprobs = sample(logits, self.u, self.temperature, self.top_k, self.top_p, self.min_p)
        if self.logprobs is not None:
            self.logprobs.copy_(logprobs)
        return tokens
