"""Routing (csrc/kernels/routing.cu) against its definition in 64 bits, which the CPU computes."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DT = [torch.bfloat16, torch.float16, torch.float32]


def _logits(tokens, experts, dt, seed=1, scale=2.0):
    return (scale * torch.randn(tokens, experts, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")).to(dt)


def _check(logits, topk, seed=3, **how):
    from fuselink_b200.ops.routing import route
    a, b = logits.detach().clone().requires_grad_(True), logits.detach().cpu().double().requires_grad_(True)
    got = route(a, topk, **how)
    want = route(b, topk, **{k: v.cpu() if torch.is_tensor(v) else v for k, v in how.items()})
    assert torch.equal(got.experts.cpu(), want.experts) and torch.equal(got.load.cpu(), want.load)
    assert got.experts.dtype == torch.int32 and int(got.load.sum()) == logits.shape[0] * topk
    # in half steps of fp32: an exponential 4, its argument (a sum with an offset, a difference from the largest) up to 16 each, 1 + e, two quotients and a factor 4;
    # a sum over the chosen one per term, over all experts one per term of a lane and 5 for the tree
    half, E = 2.0 ** -24, logits.shape[1]
    torch.testing.assert_close(got.weights.cpu(), want.weights, rtol=(E / 32 + topk + 45) * half, atol=1e-44, equal_nan=True)
    outs, wants = [got.weights], [want.weights]
    dw = torch.randn(got.weights.shape, generator=torch.Generator().manual_seed(seed))
    grads = [dw]
    if how.get("balance"):
        # shares are as weights are, with the hardware's exponential and reciprocal (8 more); a warp adds up one in 3552 tokens, a CTA eight warps' sums; CTAs' sums
        # are whole numbers of 2^-32, half a unit off for each of at most T / 8 CTAs and E experts, against a result of at least 1 / E
        rtol = (E / 32 + 53 + 8 + logits.shape[0] / 3552) * half + 2.0 ** -33 / 8 * E * E
        torch.testing.assert_close(got.balance.cpu(), want.balance, rtol=rtol, atol=0, equal_nan=True)
        outs.append(got.balance), wants.append(want.balance), grads.append(torch.tensor(0.7))
    ga, = torch.autograd.grad(outs, a, [g.cuda() for g in grads])
    gb, = torch.autograd.grad(wants, b, grads)
    if logits.shape[0]:
        T, scale = logits.shape[0], abs(how.get("scale", 1.0))
        # scores and weights as above, and products some more: (E / 32 + topk + 64) half steps of the largest terms, which may cancel; then the type's own rounding
        size = 2 * scale * dw.abs().sum(1, keepdim=True) + (2 * 0.7 * E / T if how.get("balance") else 0.0)
        tol = (E / 32 + topk + 64) * half * 2 * size + torch.finfo(logits.dtype).eps / 2 * gb.abs() + torch.finfo(logits.dtype).tiny
        ok = gb.isfinite().all(1)
        assert ((ga.cpu().double() - gb).abs() <= tol)[ok].all()
        assert torch.equal(ga.isnan().any(1).cpu(), gb.isnan().any(1))
    return got, ga


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts,topk,groups,kept", [(1, 1, 1, 1), (4, 2, 1, 1), (31, 7, 1, 1), (32, 32, 1, 1), (33, 3, 1, 1), (64, 6, 1, 1), (64, 8, 8, 3), (96, 8, 4, 2), (160, 6, 8, 3), (256, 8, 8, 4),
                                                      (300, 5, 10, 10), (512, 8, 32, 1), (1024, 10, 1, 1), (1000, 16, 8, 8)])
def test_route(experts, topk, groups, kept, score, dt):
    bias = 0.1 * torch.randn(experts, generator=torch.Generator(device="cuda").manual_seed(9), device="cuda")
    for tokens in (1, 77):
        x = _logits(tokens, experts, dt, seed=tokens)
        _check(x, topk, score=score, groups=groups, topk_groups=kept, bias=bias, balance=True, scale=2.5)
        _check(x, topk, score=score, groups=groups, topk_groups=kept, group_best=1, balance=False, renormalize=False)
        _check(x, topk, score=score, groups=groups, topk_groups=kept, offset=bias * 10, balance=True, renormalize=False, scale=0.5)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("tokens", [0, 8, 9, 4735, 4737, 20001])
def test_many_tokens(tokens, score):
    bias = 0.05 * torch.randn(128, generator=torch.Generator(device="cuda").manual_seed(9), device="cuda")
    _check(_logits(tokens, 128, torch.bfloat16), 8, score=score, groups=4, topk_groups=2, bias=bias, balance=True, scale=2.5)
    _check(_logits(tokens, 64, torch.float32), 6, score=score, balance=True)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("groups", [1, 4])
def test_equal_and_neighbouring_values(groups, biased, score):
    """Logits of a few values, so that most are equal to another's; and logits in fp32 whose scores lie within a few steps of fp32 of one another."""
    bias = (torch.arange(64, device="cuda") % 3).float() * 0.25 if biased else None
    coarse = (_logits(500, 64, torch.float32, scale=1.0) * 2).round() / 2
    for x in (coarse, coarse.to(torch.bfloat16), torch.zeros(40, 64, device="cuda")):
        _check(x, 8, score=score, groups=groups, topk_groups=max(1, groups // 2), bias=bias)
    near = 0.3 + 2.0 ** -22 * torch.randint(0, 7, (800, 64), generator=torch.Generator(device="cuda").manual_seed(4), device="cuda").float()
    _check(near, 8, score=score, groups=groups, topk_groups=max(1, groups // 2), bias=bias)
    large = 40 + _logits(200, 64, torch.float32)                      # where a logistic function is 1 in 64 bits too
    _check(large, 8, score=score, groups=groups, topk_groups=max(1, groups // 2), bias=bias)
    if biased:                                                         # a bias that makes up for the scores but for their last places
        s = torch.sigmoid(near[0].double()) if score == "sigmoid" else torch.softmax(near[0].double(), 0)
        _check(near[:1].repeat(5, 1), 8, score=score, groups=groups, topk_groups=max(1, groups // 2), bias=(1 - s).float())


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups", [1, 4])
def test_rows_that_are_not_ordinary(groups, score, dt):
    """Experts masked by -inf and by the type's lowest value, fewer left than are chosen, none; NaN and +inf."""
    x = _logits(12, 32, dt)
    x[0, 5:] = -math.inf
    x[1, 2:] = -math.inf
    x[2] = -math.inf
    x[3, 8:] = torch.finfo(dt).min
    x[4] = torch.finfo(dt).min
    x[5, 7] = math.nan
    x[6, 3], x[6, 30] = math.inf, -math.inf
    x[7, 20:22] = math.inf
    x[8] = math.nan
    x[9] = torch.finfo(dt).max
    for how in (dict(renormalize=True), dict(renormalize=False), dict(bias=torch.linspace(-1, 1, 32, device="cuda"))):
        got, grad = _check(x, 4, score=score, groups=groups, topk_groups=max(1, groups // 2), **how)
        e = got.experts.long()
        assert ((e >= 0) & (e < 32)).all() and (torch.sort(e, 1)[0].diff(dim=1) > 0).all()
        assert (got.weights[2] == 0).all() and (grad[2] == 0).all()


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("scale", [1.0, 2.5, 0.3])
def test_the_only_choice_weighs_all_and_has_no_gradient(scale, score, dt):
    from fuselink_b200.ops.routing import route
    x = _logits(300, 96, dt).requires_grad_(True)
    r = route(x, 1, score=score, scale=scale, groups=4, topk_groups=2)
    assert (r.weights == torch.tensor(scale)).all()
    g, = torch.autograd.grad(r.weights, x, torch.randn(300, 1, device="cuda"))
    assert (g == 0).all()


@pytest.mark.parametrize("groups", [1, 4])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_biases_that_are_not_ordinary(score, groups):
    """Experts that a bias of -inf or the lowest number leaves out, one that +inf always takes, and a NaN, which comes before all numbers."""
    x = _logits(60, 64, torch.bfloat16)
    bias = 0.1 * torch.randn(64, generator=torch.Generator(device="cuda").manual_seed(9), device="cuda")
    bias[::3] = -math.inf
    bias[1] = torch.finfo(torch.float32).min
    _check(x, 6, score=score, groups=groups, topk_groups=max(1, groups // 2), bias=bias)
    bias[17] = math.inf
    got, _ = _check(x, 6, score=score, groups=groups, topk_groups=max(1, groups // 2), bias=bias)
    assert (got.experts[:, 0] == 17).all()
    bias[40] = math.nan
    got, _ = _check(x, 6, score=score, groups=groups, topk_groups=max(1, groups // 2), bias=bias)
    assert (got.experts[:, 0] == 40).all()


def test_strides_offsets_and_captured_calls():
    from fuselink_b200.ops.routing import route
    wide = _logits(50, 100, torch.bfloat16)
    x = wide[:, 3:67]                                                  # rows of another distance at odd places
    _check(x, 6, score="sigmoid", balance=True)
    _check(_logits(64, 30, torch.float32).t(), 5)
    _check(wide[:1, :40].expand(9, 40), 5)                             # one row for all tokens
    full = _logits(40, 64, torch.float32)
    bias = torch.linspace(-0.1, 0.1, 64, device="cuda")

    def both():
        leaf = full.detach().requires_grad_(True)
        r = route(leaf, 6, score="sigmoid", groups=8, topk_groups=4, bias=bias, balance=True)
        return [r.weights.detach(), r.experts, r.load, r.balance.detach(), torch.autograd.grad(r.weights.sum() + 2 * r.balance, leaf)[0]]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    for seed in (5, 6):
        full.copy_(_logits(40, 64, torch.float32, seed=seed))
        bias.mul_(-1.5)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, both()))


def test_one_gradient_and_differences():
    from fuselink_b200.ops.routing import route
    x = _logits(20, 16, torch.float32)
    for score in ("softmax", "sigmoid"):
        leaf = x.clone().requires_grad_(True)
        r = route(leaf, 3, score=score, balance=True)
        for out in (r.weights.square().sum(), r.balance):
            got, = torch.autograd.grad(out, leaf, retain_graph=True)
            d = torch.randn(20, 16, generator=torch.Generator(device="cuda").manual_seed(8), device="cuda")
            h = 2.0 ** -7

            def f(at):
                s = route(at, 3, score=score, balance=True)
                assert torch.equal(s.experts, r.experts)               # the step is too small for another choice
                return s.weights.double().square().sum() if out.dim() == 0 and out is not r.balance else s.balance.double()

            step = h * d * 2.0 ** -4
            want = (f(x + step) - f(x - step)) / 2 / (h * 2.0 ** -4)
            # third derivatives are of order 1 times d^3: h^2 / 6; fp32 results over the step: 20 * 2^-24 / h
            assert abs((got * d).double().sum() - want) <= 20 * (h * 2.0 ** -4) ** 2 * 30 + 60 * 2.0 ** -24 / (h * 2.0 ** -4)


def test_what_is_refused():
    from fuselink_b200.ops.routing import route
    x, b = _logits(8, 64, torch.float32), torch.zeros(64, device="cuda")
    for bad, how in ((ValueError, dict(score="tanh")), (ValueError, dict(groups=3)), (ValueError, dict(groups=8, topk_groups=9)), (ValueError, dict(groups=8, topk_groups=0)),
                     (ValueError, dict(bias=b[:5])), (ValueError, dict(bias=b.double())), (RuntimeError, dict(offset=b.cpu())), (ValueError, dict(scale=0.0)),
                     (ValueError, dict(groups=64, topk_groups=64)), (RuntimeError, dict(bias=b.clone().requires_grad_(True)))):
        with pytest.raises(bad):
            route(x, 4, **how)
    for bad, args in ((ValueError, (x, 65)), (ValueError, (x, 0)), (ValueError, (x[0], 2)), (RuntimeError, (x, 33)), (RuntimeError, (x.double(), 2)),
                      (RuntimeError, (_logits(2, 1025, torch.float32), 2))):
        with pytest.raises(bad):
            route(*args)
    leaf = x.clone().requires_grad_(True)
    with pytest.raises(RuntimeError, match="differentiated"):
        torch.autograd.grad(route(leaf, 2).weights.square().sum(), leaf, create_graph=True)
    out = torch.vmap(lambda t: route(t, 2).weights)(torch.stack([x, -x]))        # under a transform: the framework's operations
    torch.testing.assert_close(out[0], route(x, 2).weights, rtol=(2 + 2 + 45) * 2.0 ** -24, atol=0)           # as in _check
