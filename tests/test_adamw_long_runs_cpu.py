"""AdamW with moments in 8 bits over many steps (ops/adamw.py) against moments in 32 bits: a code's step is far larger than what a step changes of a moment."""
import pytest
import torch

from fuselink_b200.ops import adamw

N = 2048
# A step moves a moment by (1 - b) |new - old|, of N(0, 1) gradients' root by less than (1 - b) / 2 of it on average.  A rounding of no sign between codes d apart has a variance of
# d times that at most, and a mean that forgets at a rate of 1 - b keeps a variance of d / 4 times the root: 2^-5 of its square, since d is 2^-3 of it at most.  Means of quotients
# and of roots move by half of that, 2^-6.  Four times as much, for the mean over 2048 weights (a spread of 0.5%) and for a gradient that has just changed.
NEAR = 2.0 ** -4


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _both(betas, steps, gradient, at):
    """{step: (median ratio of the roots, ratio of the mean sizes of the weights' steps)} of 8 bits to 32."""
    p, q = (torch.nn.Parameter(torch.zeros(N)) for _ in range(2))
    eight, whole = (adamw.AdamW([x], lr=1e-3, betas=betas, weight_decay=0.0, state_bits=b) for x, b in ((p, 8), (q, 32)))
    seen = {}
    for t in range(1, steps + 1):
        p.grad = gradient(t)
        q.grad = p.grad.clone()
        before = p.detach().clone(), q.detach().clone()
        eight.step(), whole.step()
        if t in at:
            root = adamw.decode(eight.state[p]["root_avg_sq"], eight.state[p]["root_avg_sq_scale"])
            seen[t] = (float((root / whole.state[q]["exp_avg_sq"].sqrt()).median()), float((p.detach() - before[0]).abs().mean() / (q.detach() - before[1]).abs().mean()))
    return seen


@pytest.mark.parametrize("betas", [(0.9, 0.999), (0.9, 0.95)])
def test_gradients_of_one_size(betas):
    g = _gen(1)
    for t, (root, size) in _both(betas, 2000, lambda t: torch.randn(N, generator=g), (20, 200, 1000, 2000)).items():
        assert abs(root - 1) <= NEAR and abs(size - 1) <= NEAR, (t, root, size)


@pytest.mark.parametrize("to", [0.1, 10.0])
def test_gradients_that_fall_and_rise(to):
    """From step 201 on gradients have another size: the second moment follows within some 1 / (1 - b2) steps."""
    g = _gen(2)
    for t, (root, size) in _both((0.9, 0.95), 1000, lambda t: (to if t > 200 else 1.0) * torch.randn(N, generator=g), (200, 500, 1000)).items():
        assert abs(root - 1) <= NEAR and abs(size - 1) <= NEAR, (t, root, size)


@pytest.mark.parametrize("b1", [0.9, 0.99])
def test_gradients_that_stay(b1):
    """Nothing but the codes' own rounding moves a mean on: it must not stop half way."""
    for t, (root, size) in _both((b1, 0.999), 500, lambda t: torch.ones(N), (20, 100, 500)).items():
        assert abs(root - 1) <= NEAR and abs(size - 1) <= NEAR, (t, root, size)


def test_rounding_at_random_has_the_value_as_its_mean():
    """Over many steps each value's mean code is the value, whatever its place between two codes, down to the smallest ones; codes are the neighbours of their value."""
    steps = 4096
    x = torch.cat([torch.tensor([448.0, -448.0, 0.0, 3.1, -5.7, 0.011, -2.0 ** -8, 1.3 * 2.0 ** -9, 0.3 * 2.0 ** -9, 2.0 ** -6 * (1 - 2.0 ** -6), 17.001, 447.0]), 448 * torch.rand(244, generator=_gen(3)) ** 4])
    total, near = torch.zeros(256, dtype=torch.float64), adamw.decode(*adamw.encode(x))
    for t in range(1, steps + 1):
        codes, scale = adamw.encode(x, draws=adamw.draws(256, t))
        y = adamw.decode(codes, scale)
        assert scale.item() == 1.0
        total += y.double()
        step = torch.ldexp(torch.ones(256), torch.frexp(x.abs().clamp(min=2.0 ** -6))[1] - 4)
        assert ((y - x).abs() < step).all() and (y[near == x] == x[near == x]).all()
    # the mean of 4096 roundings, each off by less than a step: six standard deviations of half a step at most
    assert ((total / steps - x.double()).abs() <= 6 * 0.5 * step.double() / steps ** 0.5).all()
    roots, _ = adamw.encode(x.abs(), root=True, draws=adamw.draws(256, 7))
    assert torch.equal(roots.float() > 0, x != 0)


def test_draws_are_even_and_unlike_from_step_to_step():
    d = [adamw.draws(40000, t, seed).double() / 2 ** 32 - 0.5 for t, seed in ((1, 0), (2, 0), (3, 0), (1000000, 0), (1, 1), (2, 1), (1, -7))]
    six = 6 / 40000 ** 0.5
    for i, x in enumerate(d):
        assert abs(x.mean()) <= six * 12 ** -0.5 and abs(12 * x.square().mean() - 1) <= six
        for y in d[:i]:
            assert abs(12 * (x * y).mean()) <= six
        for k in (1, 2, 3, 4, 8, 256):
            assert abs(12 * (x[k:] * x[:-k]).mean()) <= 1.01 * six
    assert adamw.draws(40000, 5).max() < 2 ** 32 and torch.equal(adamw.draws(7, 5), adamw.draws(40000, 5)[:7])


def test_what_is_held_twice_stays_the_same():
    """Rounding goes by place and step alone: a tensor that several ranks step stays equal whatever else each of them steps beside it."""
    ps = [torch.nn.Parameter(torch.ones(700)) for _ in range(3)]
    opts = [adamw.AdamW([ps[0]], state_bits=8), adamw.AdamW([ps[1], ps[2]], state_bits=8)]
    for k in range(20):
        ps[0].grad = torch.randn(700, generator=_gen(k))
        ps[2].grad = ps[0].grad.clone()
        ps[1].grad = None if k % 2 else torch.ones(700)
        for o in opts:
            o.step()
    a, b = opts[0].state[ps[0]], opts[1].state[ps[2]]
    assert torch.equal(ps[0], ps[2]) and all(torch.equal(a[n].float(), b[n].float()) for n in a)


def test_a_step_without_a_seed_takes_the_nearest_codes():
    """As it did before there was one; and a state that was saved then goes on with a seed of 0."""
    p, grad = torch.ones(600), torch.randn(600, generator=_gen(4))
    out = []
    for seed in (None, 0, 0, 1):
        (m, ms), (v, vs) = adamw.encode(torch.zeros(600)), adamw.encode(torch.zeros(600), root=True)
        adamw.step([p.clone()], [grad], [m], [v], [torch.tensor(0)], lr=0.1, scales=([ms], [vs]), seed=seed)
        out.append((m.float(), v.float(), ms, vs))
    near = adamw.encode(grad * (1 - 0.9))[0], adamw.encode((grad * grad * (1 - 0.999)).sqrt(), root=True)[0]
    assert torch.equal(out[0][0], near[0].float()) and torch.equal(out[0][1], near[1].float())
    assert all(torch.equal(a, b) for a, b in zip(out[1], out[2])) and not torch.equal(out[1][0], out[0][0]) and not torch.equal(out[1][0], out[3][0])
    q = torch.nn.Parameter(p.clone())
    opt = adamw.AdamW([q], state_bits=8, seed=3)
    old = opt.state_dict()
    del old["param_groups"][0]["seed"]
    opt.load_state_dict(old)
    assert opt.param_groups[0]["seed"] == 0
