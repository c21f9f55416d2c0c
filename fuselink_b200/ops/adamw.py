"""AdamW over many tensors at once (csrc/kernels/adamw.cu), with moments in fp32 or as 8-bit codes, and on request an fp32 copy of 16-bit weights.

    m = b1 m + (1 - b1) g      v = b2 v + (1 - b2) g^2      w = w (1 - lr decay) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)

Codes are e4m3 of m and of sqrt(v) with a scale for each 256 values of a tensor, as they lie in memory: the smallest power of two, 2^-100 at least, that keeps their
largest finite magnitude within 448.  A root above 0 keeps the smallest code at least; values that are not finite are kept as NaN.

A step with a ``seed`` rounds to one of the two codes around a value, to the upper one with a chance equal to the value's place between them.  That is what training takes, and
what :class:`AdamW` does: a code's step is 6 to 12% of its value, a step of the optimizer changes a moment by less (its root by 0.05% with b2 = 0.999), and the nearest code
would for the most part be the old one for good.  What decides is a hash of the place in the tensor, of the count of steps and of the seed (:func:`draws`), so that a step can
be done again, and tensors that several ranks hold stay equal.  Without a seed codes are the nearest ones, for single steps.  The step itself uses the moments before
they become codes.  The roundings of m, v and the root are IEEE's, one by one, so that the codes are the same on the CPU and on the GPU.

The number of steps is a tensor's own and lives on its device, and the learning rate may: a captured step counts on when it is replayed.
"""
from __future__ import annotations

import math
from typing import List, Optional, Sequence, Tuple, Union

import torch

from .._ext import require_native

FP8 = torch.float8_e4m3fn
BLOCK = 256
LEAST_SCALE = 2.0 ** -100


def _settings(lr, betas, eps, weight_decay):
    if not isinstance(lr, torch.Tensor) and not 0 <= lr < math.inf:
        raise ValueError(f"adamw: a learning rate of {lr}")
    if not all(0 <= b < 1 for b in betas) or not 0 <= eps < math.inf or not 0 <= weight_decay < math.inf:
        raise ValueError(f"adamw: betas {tuple(betas)}, eps {eps}, weight_decay {weight_decay}")


def step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], m: Sequence[torch.Tensor], v: Sequence[torch.Tensor], steps: Sequence[torch.Tensor], *,
         lr: Union[float, torch.Tensor], betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.01,
         scales: Optional[Tuple[Sequence[torch.Tensor], Sequence[torch.Tensor]]] = None, master: Optional[Sequence[torch.Tensor]] = None,
         seed: Optional[int] = None) -> None:
    """One step on ``params`` in place, each with its gradient, moments and count of steps (one int64 value, which the call raises by one).  m, v: fp32, laid out as
    their parameter; with ``scales`` (of m, of the root) e4m3 codes, and scales fp32 [ceil(n / 256)], rounded at random by ``seed`` (32 bits of it), which many steps
    need, or without one to the nearest.  ``master``: fp32 copies of bf16 or fp16 parameters; the
    step works on these and rounds them to the parameters.  ``lr``: a number, or one fp32 value on the device.  On the GPU bf16, fp16 and fp32, all on one device,
    parameters without gaps, each one once; gradients of their parameter's type."""
    _settings(lr, betas, eps, weight_decay)
    m_scales, v_scales = scales if scales is not None else ((), ())
    if len(params) > 0 and params[0].is_cuda:
        on_device = isinstance(lr, torch.Tensor)
        require_native().adamw_step(params, grads, m, v, steps, m_scales, v_scales, master or (), 0.0 if on_device else lr, lr if on_device else None,
                                    betas[0], betas[1], eps, weight_decay, scales is not None, seed)
        return
    _plain(params, grads, m, v, steps, lr, betas, eps, weight_decay, scales, master, seed)


@torch.no_grad()
def _plain(params, grads, m, v, steps, lr, betas, eps, weight_decay, scales, master, seed):
    if any(len(x) != len(params) for x in [grads, m, v, steps, *(scales or ()), *([master] if master else ())]):
        raise RuntimeError("adamw: one of each for every parameter")
    for i, p in enumerate(params):
        if grads[i].layout != torch.strided or grads[i].shape != p.shape or grads[i].dtype != p.dtype:
            raise RuntimeError("adamw: a dense gradient of its parameter's type, shape and device")
        _plain_step(p, grads[i], m[i], v[i], steps[i], lr, betas, eps, weight_decay, (scales[0][i], scales[1][i]) if scales is not None else None,
                    master[i] if master else None, seed)


def _in_memory(t: torch.Tensor) -> torch.Tensor:
    """The values of a tensor without gaps, in the order in which they lie in memory."""
    return t.detach().as_strided((t.numel(),), (1,))


_WORD, _BY, _AND = 0xffffffff, 0x9e3779b9, 0x6a09e667      # 2^32 times the fractional parts of the golden section and of the root of 2


def _mix(x: torch.Tensor) -> torch.Tensor:
    x = x * _BY & _WORD
    x = (x ^ x >> 15) * _AND & _WORD
    return x ^ x >> 16


def draws(n: int, step: int, seed: int = 0, device=None) -> torch.Tensor:
    """The 32 bits, as int64, by which the ``n`` values of a tensor are rounded in its step number ``step``, the first being 1: a hash of each four values' place,
    of the step and of the seed, and numbers that follow it.  Roots go by the upper 20 of them, means by the lower 20."""
    x = _mix(_mix(_mix(torch.tensor(seed & _WORD, device=device)) ^ step & _WORD) ^ torch.arange((n + 3) // 4, device=device) & _WORD)
    four = [x]
    for _ in range(3):
        four.append(four[-1] * _BY + _AND & _WORD)
    return torch.stack(four, 1).reshape(-1)[:n]


def _rounded_by(x: torch.Tensor, bits: torch.Tensor) -> torch.Tensor:
    """x, of at most 448, rounded to e4m3: up where its 20 bits below those of a code and ``bits`` make a whole step.  Codes below 2^-6 are as far apart as those above."""
    small = torch.where(x.abs() < 2.0 ** -6, 2.0 ** -6, 0.0)
    y = ((x.abs() + small).view(torch.int32) + bits.int() & -(1 << 20)).view(torch.float32) - small
    return torch.where(x.isnan(), x, torch.copysign(y, x))


def encode(x: torch.Tensor, root: bool = False, draws: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(codes like x, scales [ceil(n / 256)]) of fp32 values; ``root``: none above 0 becomes the code of 0.  To the nearest code, or with ``draws``, 32 bits for each
    value as it lies in memory, to the one below or above."""
    flat = _in_memory(x)
    blocks = torch.nn.functional.pad(flat, (0, -flat.numel() % BLOCK)).view(-1, BLOCK)
    finite = torch.where(blocks.isfinite(), blocks, torch.zeros_like(blocks))
    scale = scale_of(finite.abs().amax(1)) if blocks.numel() else flat.new_empty(0)
    scaled = torch.where(blocks.isinf(), torch.full_like(blocks, math.nan), blocks / scale[:, None])
    if draws is not None:
        bits = torch.nn.functional.pad(draws, (0, -flat.numel() % BLOCK)).view(-1, BLOCK)
        scaled = _rounded_by(scaled, bits >> 12 if root else bits & 0xfffff)
    codes = scaled.to(FP8).view(torch.uint8)
    if root:
        codes = torch.where((blocks > 0) & (codes == 0), torch.ones_like(codes), codes)
    out = torch.empty_like(x, dtype=FP8)
    _in_memory(out).copy_(codes.view(FP8).reshape(-1)[:flat.numel()])
    return out, scale


def decode(codes: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """The fp32 values that codes stand for; of the second moment its root."""
    flat = _in_memory(codes).float()
    out = torch.empty_like(codes, dtype=torch.float32)
    _in_memory(out).copy_(flat * scale.repeat_interleave(BLOCK)[:flat.numel()])
    return out


def scale_of(amax: torch.Tensor) -> torch.Tensor:
    """The smallest power of two, 2^-100 at least, that brings a finite amax within 448."""
    frac, e = torch.frexp(amax)                            # amax = frac 2^e, frac in [0.5, 1); 448 = 0.875 * 2^9
    s = torch.ldexp(torch.ones_like(amax), torch.where(frac <= 0.875, e - 9, e - 8))
    return torch.where(amax > 0, s, torch.zeros_like(s)).clamp(min=LEAST_SCALE)


def _plain_step(p, grad, m, v, steps, lr, betas, eps, weight_decay, scales, master, seed):
    b1, b2 = betas
    lr = float(lr)
    steps += 1
    t = int(steps)
    g = grad.float()
    old_m, old_v = (m, v) if scales is None else (decode(m, scales[0]), decode(v, scales[1]).square())
    new_m = old_m * b1 + g * (1 - b1)
    new_v = old_v * b2 + (g * g) * (1 - b2)
    root = new_v.sqrt()
    w = p.float() if master is None else master
    w = w * (1 - lr * weight_decay) - (lr / (1 - b1 ** t)) * (new_m / (root * (1 - b2 ** t) ** -0.5 + eps))
    p.copy_(w)
    if master is not None:
        master.copy_(w)
    if scales is None:
        m.copy_(new_m)
        v.copy_(new_v)
        return
    like = torch.empty_like(m, dtype=torch.float32)         # laid out as the parameter, whatever the gradient's strides
    bits = None if seed is None else draws(p.numel(), t, seed, p.device)
    for codes, scale, x, is_root in ((m, scales[0], new_m, False), (v, scales[1], root, True)):
        c, s = encode(like.copy_(x), is_root, bits)
        codes.view(torch.uint8).copy_(c.view(torch.uint8))
        scale.copy_(s)


class AdamW(torch.optim.Optimizer):
    """The optimizer around :func:`step`: ``state_bits`` 32 or 8, the latter rounded at random by ``seed`` (the same on ranks that hold the same parameters), ``master`` keeps fp32 copies of bf16 and fp16 parameters, from which the next step starts:
    parameters that are written otherwise (loaded, broadcast) call for ``refresh_masters``.  Parameters without a gradient are left out of a step, their counts too.  ``lr`` of a group may be one fp32 value on the device, which a schedule writes between replays of a captured step; the first
    step, which makes the state, is not captured.  Sparse gradients are refused."""

    def __init__(self, params, lr: Union[float, torch.Tensor] = 1e-3, betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.01, *,
                 state_bits: int = 32, master: bool = False, seed: int = 0):
        _settings(lr, betas, eps, weight_decay)
        if state_bits not in (8, 32):
            raise ValueError(f"adamw: moments in 8 or 32 bits, not {state_bits}")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits, master=master, seed=seed))

    def __setstate__(self, state):
        super().__setstate__(state)
        for group in self.param_groups:
            group.setdefault("seed", 0)                      # saved before there was one

    def _new_state(self, p: torch.Tensor, group: dict) -> dict:
        if not p.is_floating_point() or p.layout != torch.strided:
            raise RuntimeError(f"adamw: a dense floating parameter expected, not {p.dtype} {p.layout}")
        if p.is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("adamw: the first step makes the state and cannot be captured")
        zeros = torch.zeros_like(p, dtype=torch.float32, requires_grad=False)
        state = dict(step=torch.zeros((), dtype=torch.int64, device=p.device))
        if group["state_bits"] == 8:
            (state["exp_avg"], state["exp_avg_scale"]), (state["root_avg_sq"], state["root_avg_sq_scale"]) = encode(zeros), encode(zeros, root=True)
        else:
            state["exp_avg"], state["exp_avg_sq"] = zeros, torch.zeros_like(zeros)
        if group["master"] and p.dtype in (torch.bfloat16, torch.float16):
            state["master"] = p.detach().float()
        return state

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            calls: dict = {}                                 # by device and by whether there is an fp32 copy
            for p in group["params"]:
                g = p.grad
                if g is None:
                    continue
                if g.layout != torch.strided:
                    raise RuntimeError("adamw: sparse gradients are not taken")
                state = self.state[p]
                if not state:
                    state.update(self._new_state(p, group))
                lists: List[list] = calls.setdefault((p.device, "master" in state), [[] for _ in range(8)])
                eight = group["state_bits"] == 8
                for to, x in zip(lists, (p, g, state["exp_avg"], state["root_avg_sq" if eight else "exp_avg_sq"], state["step"],
                                         state.get("exp_avg_scale"), state.get("root_avg_sq_scale"), state.get("master"))):
                    to.append(x)
            for (_, has_master), (ps, gs, ms, vs, steps, m_scales, v_scales, masters) in calls.items():
                step(ps, gs, ms, vs, steps, lr=group["lr"], betas=group["betas"], eps=group["eps"], weight_decay=group["weight_decay"],
                     scales=(m_scales, v_scales) if group["state_bits"] == 8 else None, master=masters if has_master else None, seed=group["seed"])
        return loss

    @torch.no_grad()
    def refresh_masters(self) -> None:
        """Takes the fp32 copies anew from the parameters."""
        for p, state in self.state.items():
            if "master" in state:
                state["master"].copy_(p)

    def load_state_dict(self, state_dict):
        """As the base class does, which turns floating state to the parameter's type: here it keeps its own."""
        super().load_state_dict(state_dict)
        saved = {i: s for i, s in state_dict["state"].items()}
        order = [i for g in state_dict["param_groups"] for i in g["params"]]
        for i, p in zip(order, (p for g in self.param_groups for p in g["params"])):
            for name, t in saved.get(i, {}).items():
                if isinstance(t, torch.Tensor):
                    self.state[p][name] = t.detach().to(p.device, copy=True)
