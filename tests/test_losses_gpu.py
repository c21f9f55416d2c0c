"""Log-probabilities of tokens and the policy loss (csrc/kernels/losses.cu) against their definition in 64 bits, which the CPU computes."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DT = [torch.bfloat16, torch.float16, torch.float32]
HALF = 2.0 ** -24


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _logits(shape, dt, seed=1, scale=3.0):
    return (scale * torch.randn(*shape, generator=_gen(seed), device="cuda")).to(dt)


def _tokens(shape, vocab, seed=2):
    return torch.randint(0, vocab, shape, generator=_gen(seed), device="cuda")


def _off(vocab, scale, temperature):
    """How far a row's logarithm may be: a thread adds up vocab / 512 exponentials, joined over some 20 more sums; an exponent's argument, at most
    12 scale log2(e) / T between largest and smallest logit, is off by two half steps and the hardware's exponential by 4; the result's own step."""
    return (vocab / 512 + 24 + 2 * 12 * scale * 1.45 / temperature) * HALF


def _check_gradient(got, logits, tokens, each, temperature, lp_off):
    x = logits.detach().cpu().double() / temperature
    p = torch.softmax(x, -1)
    onehot = torch.zeros_like(p).scatter_(-1, tokens.cpu().unsqueeze(-1), 1.0)
    g = each.cpu().double().unsqueeze(-1) / temperature
    want = g * (onehot - p)
    # a probability is off as its row's logarithm is; a factor and a product round
    tol = g.abs() * p * (lp_off + 8 * HALF) + want.abs() * (torch.finfo(got.dtype).eps / 2 + 4 * HALF) + torch.finfo(got.dtype).tiny
    assert ((got.cpu().double() - want).abs() <= tol).all()


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("shape,temperature", [((1, 1), 1.0), ((3, 2), 0.7), ((2, 5, 7), 1.0), ((33, 1000), 1.3), ((5, 4095), 1.0), ((3, 4, 50257), 0.7), ((2, 128256), 1.0), ((700, 33), 1.0), ((1, 300001), 1.0)])
def test_token_logprobs(shape, temperature, dt):
    from fuselink_b200.ops.losses import token_logprobs
    x, t = _logits(shape, dt).requires_grad_(True), _tokens(shape[:-1], shape[-1])
    lp = token_logprobs(x, t, temperature=temperature)
    want = token_logprobs(x.detach().cpu(), t.cpu(), temperature=temperature)
    off = _off(shape[-1], 3.0, temperature)
    assert lp.shape == t.shape and lp.dtype == torch.float32
    assert ((lp.cpu() - want).abs() <= off + 2 * HALF * want.abs()).all()
    assert torch.equal(token_logprobs(x.detach(), t, temperature=temperature), lp)
    g = torch.randn(t.shape, generator=_gen(5), device="cuda")
    got, = torch.autograd.grad(lp, x, g)
    assert got.shape == x.shape and got.dtype == dt
    _check_gradient(got, x, t, g, temperature, off)


def _policy_inputs(shape, vocab, dt, seed=1, temperature=1.0, reference=True):
    from fuselink_b200.ops.losses import token_logprobs
    x, t = _logits((*shape, vocab), dt, seed), _tokens(shape, vocab, seed + 1)
    lp = token_logprobs(x.cpu(), t.cpu(), temperature=temperature).cuda()
    drift = 0.2 * torch.randn(shape, generator=_gen(seed + 2), device="cuda")
    for border in (math.log(0.8), math.log(1.28)):                    # none where a rounding decides on which side it lies
        drift = torch.where((drift - border).abs() < 1e-2, drift + 0.05, drift)
    A = torch.randn(shape, generator=_gen(seed + 3), device="cuda")
    w = (torch.rand(shape, generator=_gen(seed + 4), device="cuda") < 0.8).float() * torch.rand(shape, generator=_gen(seed + 5), device="cuda").add(0.5)
    ref = lp + 0.3 * torch.randn(shape, generator=_gen(seed + 6), device="cuda") if reference else None
    return x, t, dict(old=lp - drift, advantages=A, weights=w, reference=ref, kl=0.05 if reference else 0.0, clip=(0.2, 0.28), temperature=temperature)


def _cpu(how):
    return {k: v.cpu() if torch.is_tensor(v) else v for k, v in how.items()}


def _check_policy(x, t, how, upstream=1.0):
    from fuselink_b200.ops.losses import policy_loss
    a, b = x.detach().requires_grad_(True), x.detach().cpu().double().requires_grad_(True)
    got, want = policy_loss(a, t, **how), policy_loss(b, t.cpu(), **_cpu(how))
    T, V = how.get("temperature", 1.0), x.shape[-1]
    off = _off(V, 3.0, T)
    live = how["weights"].cpu() != 0 if how.get("weights") is not None else torch.ones_like(want.logprobs, dtype=torch.bool)
    assert (got.logprobs.cpu()[~live] == 0).all()
    assert ((got.logprobs.cpu() - want.logprobs).abs() <= off + 2 * HALF * want.logprobs.abs()).all()
    # a term moves by |q A| + kl |1 - exp d| times what its logarithm is off
    w = how["weights"].cpu().double() if how.get("weights") is not None else torch.ones(t.shape, dtype=torch.float64)
    total = how.get("total")
    total = w.sum() if total is None else torch.as_tensor(total).cpu().double()
    share = w.abs() / total.abs() if total != 0 else w * 0
    q = torch.exp((want.logprobs - how["old"].cpu()).double()) * live
    more = torch.expm1((how["reference"].cpu() - want.logprobs).double()) * live if how.get("reference") is not None else torch.zeros_like(q)
    q, more = torch.where(live, q, 0.0), torch.where(live, more, 0.0)
    slope = torch.where(live, q * how["advantages"].cpu().double().abs(), 0.0) + how.get("kl", 0.0) * more.abs()
    assert abs(got.loss.item() - want.loss.item()) <= (share * slope).sum() * off + 2 * HALF * abs(want.loss.item()) + 1e-30
    assert abs(got.divergence.item() - want.divergence.item()) <= (share * more.abs()).sum() * off + 2 * HALF * want.divergence.item() + 1e-30
    assert abs(got.clipped.item() - want.clipped.item()) <= 2 * HALF * abs(want.clipped.item())
    ga, = torch.autograd.grad(got.loss, a, torch.tensor(upstream, device="cuda"), retain_graph=True)
    gb, = torch.autograd.grad(want.loss, b, torch.tensor(upstream))
    p = torch.where(live.unsqueeze(-1), torch.softmax(x.detach().cpu().double() / T, -1), 0.0)
    each = (share * (slope + how.get("kl", 0.0))).unsqueeze(-1) * abs(upstream) / T
    onehot = torch.zeros_like(p).scatter_(-1, t.cpu().clamp(0, V - 1).unsqueeze(-1), 1.0)
    tol = each * (p + onehot) * (3 * off + 16 * HALF) + gb.abs() * torch.finfo(x.dtype).eps / 2 + torch.finfo(x.dtype).tiny
    assert ga.shape == x.shape and ((ga.cpu().double() - gb).abs() <= tol).all()
    again, = torch.autograd.grad(got.loss, a, torch.tensor(upstream, device="cuda"))     # computed anew: the first one has its owner
    assert torch.equal(again, ga) and (again.data_ptr() != ga.data_ptr() or x.numel() == 0)
    with torch.no_grad():
        plain = policy_loss(a, t, **how)
    assert all(torch.equal(x, y) for x, y in zip(plain, got))
    return got, ga


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("shape,vocab,temperature", [((1,), 1, 1.0), ((7,), 33, 1.0), ((3, 50), 1000, 0.7), ((2, 9), 50257, 1.0), ((2, 3, 5), 257, 1.0), ((4,), 128256, 1.0), ((1300,), 65, 1.2)])
def test_policy_loss(shape, vocab, temperature, dt):
    for reference in (False, True):
        x, t, how = _policy_inputs(shape, vocab, dt, temperature=temperature, reference=reference)
        if vocab > 1:
            _check_policy(x, t, how)
            _check_policy(x, t, how, upstream=0.3)
        _check_policy(x, t, dict(how, weights=None))


def test_totals_and_rows_without_weight():
    from fuselink_b200.ops.losses import policy_loss
    x, t, how = _policy_inputs((6, 10), 500, torch.bfloat16)
    _check_policy(x, t, dict(how, total=7.5))
    _check_policy(x, t, dict(how, total=torch.tensor(33.0, device="cuda")))
    # rows of weight 0 may hold anything, and any token
    x[0], x[1, 3], t[0] = math.nan, math.inf, -100
    how["weights"][0], how["weights"][1, 3] = 0, 0
    for name in ("old", "advantages", "reference"):
        how[name][0] = math.nan
    got, grad = _check_policy(x, t, how)
    assert (grad[0] == 0).all() and (got.logprobs[0] == 0).all() and got.loss.isfinite()
    none, grad = _check_policy(x, t, dict(how, weights=torch.zeros(6, 10, device="cuda")))
    assert none.loss == 0 and none.divergence == 0 and none.clipped == 0 and (grad == 0).all()
    none, grad = _check_policy(x[:0], t[:0], {k: v[:0] if torch.is_tensor(v) else v for k, v in how.items()})
    assert none.loss == 0 and grad.shape == (0, 10, 500)
    # a mask and advantages that are broadcast
    leaf = x[2:].detach().clone().requires_grad_(True)
    a = policy_loss(leaf, t[2:], how["old"][2:], how["advantages"][2:, :1], weights=how["weights"][2:] > 0)
    b = policy_loss(leaf, t[2:].int(), how["old"][2:], how["advantages"][2:, :1].expand(4, 10), weights=(how["weights"][2:] > 0).float())
    assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("vocab", [64, 999, 1001])
def test_logits_that_lie_otherwise(vocab, dt):
    """Slices of positions, of requests and of the vocabulary, rows at odd places, dimensions in another order, one row for all."""
    from fuselink_b200.ops.losses import token_logprobs
    full = _logits((5, 7, vocab + 3), dt)
    for x in (full[:, :-1], full[:, 1:, :vocab], full[1:4, :, 1:vocab], full[::2], full[:, ::3, 2:], full.transpose(0, 1), full[0, 0].expand(3, 4, vocab + 3), full[2, 3], full[:1, :1],
              full.view(5, 7, 1, vocab + 3)[:, :, :, 1:], full[:, :, ::2]):
        t, g = _tokens(x.shape[:-1], x.shape[-1]), torch.randn(x.shape[:-1], generator=_gen(4), device="cuda")
        leaf = x.detach().requires_grad_(True)
        assert leaf.stride() == x.stride()
        lp = token_logprobs(leaf, t)
        off = _off(x.shape[-1], 3.0, 1.0)
        assert ((lp.cpu() - token_logprobs(x.cpu(), t.cpu())).abs() <= off + 2 * HALF * lp.cpu().abs()).all()
        _check_gradient(torch.autograd.grad(lp, leaf, g)[0], x, t, g, 1.0, off)
        if x.dim() > 1:
            how = dict(old=lp.detach() + 0.1, advantages=g, weights=None, reference=lp.detach() - 0.2, kl=0.1, clip=(0.2, 0.2))
            _check_policy(x, t, how, upstream=0.5)
    kept = full[:, :-1].clone()
    token_logprobs(full.requires_grad_(True)[:, :-1], _tokens((5, 6), vocab)).sum().backward()       # through the slice
    assert (full.grad[:, -1] == 0).all() and torch.equal(full.detach()[:, :-1], kept)


@pytest.mark.parametrize("dt", DT)
def test_rows_that_are_not_ordinary(dt):
    from fuselink_b200.ops.losses import token_logprobs
    x, t = _logits((12, 700), dt), _tokens((12,), 700)
    x[0, 1:] = -math.inf; t[0] = 0
    x[1, ::2] = -math.inf; t[1] = 2                                    # a token that is masked
    x[2, ::2] = torch.finfo(dt).min; t[2] = 1
    x[3] = -math.inf
    x[4, 9] = math.nan
    x[5, 9] = math.inf
    t[6], t[7] = 700, -1
    x[8] = 1.5
    x[9] = x[9] * 100 if dt != torch.float16 else x[9] * 20
    leaf = x.requires_grad_(True)
    lp = token_logprobs(leaf, t)
    want = token_logprobs(x.detach().cpu(), t.cpu())
    assert lp[0] == 0 and lp[1] == -math.inf and lp[3:8].isnan().all() and torch.equal(lp.isnan().cpu(), want.isnan())
    ok = want.isfinite()
    # row 9: arguments of thousands, off by as many half steps
    off = _off(700, torch.where(torch.arange(12) == 9, 300.0, 3.0), 1.0)
    assert ((lp.cpu() - want).abs() <= off + 2 * HALF * want.abs())[ok].all()
    g, = torch.autograd.grad(lp.nan_to_num(0, 0, 0).sum() + 0 * lp[0], leaf, retain_graph=True)
    assert (g[0] == 0).all() and (g[2].float().abs()[::2] == 0).all()
    g, = torch.autograd.grad(lp, leaf, torch.ones(12, device="cuda"))
    assert g[3:8].isnan().all() and g[:3].isfinite().all() and g[8:].isfinite().all()
    assert (g[1, ::2].float() == torch.nn.functional.one_hot(t[1], 700)[::2]).all()


def test_a_ratio_at_its_border_has_a_gradient():
    from fuselink_b200.ops.losses import policy_loss
    x, t = torch.zeros(2, 8, device="cuda").requires_grad_(True), torch.zeros(2, dtype=torch.int64, device="cuda")
    old = torch.full((2,), -math.log(8), device="cuda")
    lp = policy_loss(x, t, old, old, clip=(0.0, 0.0)).logprobs
    r = policy_loss(x, t, lp, torch.tensor([1.0, -1.0], device="cuda"), clip=(0.0, 0.0))
    assert r.clipped <= 0.5 and r.loss.abs() <= 2 * HALF               # q is 1 but for the rounding of lp


def test_captured_and_on_another_stream():
    from fuselink_b200.ops.losses import policy_loss
    x, t, how = _policy_inputs((4, 30), 2000, torch.bfloat16)

    def both(scale=1.0):
        leaf = x.detach().requires_grad_(True)
        r = policy_loss(leaf, t, **how)
        return [r.loss.detach(), r.logprobs, r.divergence, r.clipped, torch.autograd.grad(r.loss * scale, leaf)[0]]

    want = both(0.5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
        other = both(0.5)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    for scale in (1.0, 0.5):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = both(scale)
        for seed in (21, 22):
            x2, t2, how2 = _policy_inputs((4, 30), 2000, torch.bfloat16, seed=seed)
            x.copy_(x2), t.copy_(t2)
            for k, v in how2.items():
                if torch.is_tensor(v):
                    how[k].copy_(v)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, both(scale)))


def test_differences_of_the_loss():
    from fuselink_b200.ops.losses import policy_loss, token_logprobs
    x, t, how = _policy_inputs((3, 20), 50, torch.float32)
    leaf = x.clone().requires_grad_(True)
    d = torch.randn(x.shape, generator=_gen(9), device="cuda")
    h = 2.0 ** -9
    for f in (lambda y: policy_loss(y, t, **how).loss, lambda y: token_logprobs(y, t).mean()):
        got = (torch.autograd.grad(f(leaf), leaf)[0] * d).double().sum()
        want = (f(x + h * d) - f(x - h * d)).double() / (2 * h)
        # third derivatives along d are of order |d|^3 ~ 50; an fp32 result over the step
        assert abs(got - want) <= 50 * h * h + 4 * _off(50, 3.0, 1.0) / h


def test_what_is_refused():
    from fuselink_b200.ops.losses import policy_loss, token_logprobs
    x, t = _logits((4, 9), torch.float32), _tokens((4,), 9)
    f = torch.zeros(4, device="cuda")
    for bad, args, how in ((ValueError, (x, t[:3]), {}), (ValueError, (x, t.float()), {}), (RuntimeError, (x, t.cpu()), {}), (ValueError, (x, t), dict(temperature=0.0)),
                           (ValueError, (x, t), dict(temperature=math.nan)), (ValueError, (x, t), dict(temperature=1e-40)), (ValueError, (x[:, :0], t), {}), (RuntimeError, (x.double(), t), {})):
        with pytest.raises(bad):
            token_logprobs(*args, **how)
    for bad, how in ((RuntimeError, dict(old=f.cpu())), (RuntimeError, dict(advantages=torch.zeros(3, device="cuda"))), (RuntimeError, dict(weights=f.clone().requires_grad_(True))),
                     (ValueError, dict(clip=(-0.1, 0.2))), (ValueError, dict(kl=-1.0)), (ValueError, dict(kl=math.nan)), (ValueError, dict(total=f)), (ValueError, dict(total=torch.tensor(1.0))),
                     (RuntimeError, dict(total=torch.ones((), device="cuda").requires_grad_(True)))):
        with pytest.raises(bad):
            policy_loss(x, t, **{**dict(old=f, advantages=f), **how})
    leaf = x.clone().requires_grad_(True)
    for out in (token_logprobs(leaf, t).square().sum(), policy_loss(leaf, t, f, f + 1).loss):
        with pytest.raises(RuntimeError, match="differentiated"):
            torch.autograd.grad(out, leaf, create_graph=True)
