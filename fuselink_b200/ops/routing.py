"""Routing of tokens to experts (csrc/kernels/routing.cu): scores, a balance bias, groups, top-k, weights, loads, and the balance term.

A token's scores are the softmax or the sigmoid of its logits.  The choice goes by score + bias: of ``groups`` groups of consecutive experts the
``topk_groups`` whose one or two best sum to most, of their experts the ``topk`` best; of equals the lowest first, a NaN before all numbers.  Without a bias
experts are ordered by their logits.  The weights are the scores of those chosen, without the bias.  The choice is made in 64 bits, so that
neighbouring values are told apart the same way wherever it is computed.

``balance`` is E / (T k) sum_e load_e mean_t p_te / sum_e' p_te': 1 where experts are chosen evenly.  The gradient is that of weights and balance;
choice and loads are constants of it.  On the GPU choice and weights are those of logits and offset added exactly; the balance term, and what every expert's gradient
has from it or from weights that are not renormalised, go by the sum as fp32 has it, 2^-24 of the logit off.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from .._ext import require_native
from .checks import ordinary

SCORES = ("softmax", "sigmoid")


class Routing(NamedTuple):
    weights: torch.Tensor               # [tokens, topk] fp32
    experts: torch.Tensor               # [tokens, topk] int32, best first
    load: torch.Tensor                  # [experts] int32: tokens that chose each
    balance: Optional[torch.Tensor]     # one fp32 value, where asked for


def route(logits: torch.Tensor, topk: int, *, score: str = "softmax", bias: Optional[torch.Tensor] = None, offset: Optional[torch.Tensor] = None,
          groups: int = 1, topk_groups: Optional[int] = None, group_best: int = 2, renormalize: bool = True, scale: float = 1.0,
          balance: bool = False) -> Routing:
    """logits [tokens, experts]; bias and offset [experts] fp32, constants: ``offset`` is added to the logits, ``bias`` to the scores for the choice
    alone.  ``renormalize``: a token's weights sum to ``scale``; else they are its scores times ``scale``.  A token whose chosen scores are all 0
    (logits of -inf) has weights of 0 and no gradient from them.  On the GPU bf16, fp16 and fp32, at most 1024 experts, 32 choices and 32 groups; on the
    CPU any floating type."""
    if logits.is_cuda and ordinary(logits):
        return Routing(*require_native().route(logits, topk, score, groups, topk_groups, group_best, renormalize, scale, bias, offset, balance))
    if logits.dim() != 2 or logits.shape[1] == 0:
        raise ValueError(f"route: logits [tokens, experts] expected, not {tuple(logits.shape)}")
    T, E = logits.shape
    if score not in SCORES:
        raise ValueError(f"route: score {score!r}; one of {SCORES} expected")
    if groups < 1 or E % groups:
        raise ValueError(f"route: {E} experts do not make {groups} equal groups")
    topk_groups = groups if topk_groups is None else topk_groups
    if not 1 <= topk_groups <= groups:
        raise ValueError(f"route: {topk_groups} of {groups} groups")
    if not 1 <= topk <= E // groups * topk_groups:
        raise ValueError(f"route: {topk} of the {E // groups * topk_groups} experts in {topk_groups} groups")
    if groups == 1:
        group_best = 1
    if group_best not in (1, 2) or group_best > E // groups:
        raise ValueError(f"route: a group goes by its 1 or 2 best of {E // groups}, not by {group_best}")
    if not (scale == scale and 0 < abs(scale) < float("inf")):
        raise ValueError(f"route: a factor of {scale}")
    for name, t in (("bias", bias), ("offset", offset)):
        if t is None:
            continue
        if t.shape != (E,) or t.dtype != torch.float32:
            raise ValueError(f"route: {name} [{E}] fp32 expected, not {tuple(t.shape)} of {t.dtype}")
        if t.device != logits.device:
            raise RuntimeError(f"route: {name} on {logits.device} expected, not on {t.device}")
        if t.requires_grad and torch.is_grad_enabled():
            raise RuntimeError("route: bias and offset get no gradient; detach them")
    return _plain_route(logits, topk, score, bias, offset, groups, topk_groups, group_best, renormalize, scale, balance)


def _plain_route(logits, topk, score, bias, offset, groups, topk_groups, group_best, renormalize, scale, balance):
    T, E = logits.shape
    x = logits.double() if offset is None else logits.double() + offset.double()
    if score == "softmax":
        nothing = (x == -float("inf")).all(1, keepdim=True)
        p = torch.where(nothing, 0.0, torch.softmax(torch.where(nothing, 0.0, x), 1))
    else:
        p = torch.sigmoid(x)
    with torch.no_grad():
        c = p if bias is None else p + bias.double()
        left = torch.ones(T, E, dtype=torch.bool, device=x.device)
        if groups > 1:
            best = torch.sort(c.view(T, groups, E // groups), dim=2, descending=True)[0][:, :, :group_best].sum(2)
            kept = torch.sort(best, dim=1, descending=True, stable=True)[1][:, :topk_groups]
            left = torch.zeros(T, groups, dtype=torch.bool, device=x.device).scatter(1, kept, True).repeat_interleave(E // groups, 1)
        order = torch.sort(x if bias is None else c, dim=1, descending=True, stable=True)[1]
        idx = order.gather(1, torch.sort((~left.gather(1, order)).int(), dim=1, stable=True)[1])[:, :topk]     # those left, in their order
        load = torch.zeros(E, dtype=torch.int32, device=x.device).index_add(0, idx.reshape(-1), torch.ones(T * topk, dtype=torch.int32, device=x.device))
    w = p.gather(1, idx)
    if renormalize:
        total = w.sum(1, keepdim=True)
        w = torch.where(total == 0, 0.0, w / torch.where(total == 0, 1.0, total))
    term = None
    if balance:
        total = p.sum(1, keepdim=True)
        share = torch.where(total == 0, 0.0, p / torch.where(total == 0, 1.0, total))
        term = ((load.double() * share.sum(0)).sum() * (E / (max(T, 1) ** 2 * topk))).float()
    return Routing((w * scale).float(), idx.int(), load, term)
