"""AdamW's 8-bit moments, rounded at random by place, step and seed or to the nearest code (csrc/kernels/adamw.cu), against the same on the CPU bit by bit over many steps."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
HOW = dict(lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0, seed=5)


def _same(a, b):
    a, nan = a.cpu().float(), b.float().isnan()
    return torch.equal(a.isnan(), nan) and torch.equal(a[~nan], b.float()[~nan])


def _state(shapes, dt, step=0):
    from fuselink_b200.ops import adamw
    s = dict(params=[torch.ones(x).to(dt) for x in shapes], steps=[torch.tensor(step + i) for i in range(len(shapes))])
    for name in ("m", "v"):
        s[name], s[name + "_scale"] = map(list, zip(*(adamw.encode(torch.zeros(x), root=name == "v") for x in shapes)))
    return s


def _step(s, grads, **how):
    from fuselink_b200.ops import adamw
    adamw.step(s["params"], grads, s["m"], s["v"], s["steps"], scales=(s["m_scale"], s["v_scale"]), **{**HOW, **how})


def _on_gpu(s):
    return {k: [t.cuda() for t in v] for k, v in s.items()}


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("seed", [0, 12345, -1, None])
@pytest.mark.parametrize("kind", ["even", "wide", "none", "odd"])
def test_many_steps(dt, kind, seed):
    """Gradients of one size, over the whole range of a code and below it, mostly zeros, and with infinities and NaN: whole blocks, ends of tensors, and no block at all."""
    shapes = [(4096,), (33, 257), (7,), (256,), (1300,)]
    want = _state(shapes, dt)
    got = _on_gpu(want)
    gen = torch.Generator().manual_seed(5)
    for k in range(40):
        grads = []
        for x in shapes:
            g = torch.randn(x, generator=gen)
            if kind == "wide":
                g = g * 2.0 ** (-18 * torch.rand(x, generator=gen))
            if kind == "none":
                g = g * (torch.rand(x, generator=gen) < 0.02)
            if kind == "odd" and k == 20:
                g.view(-1)[[0, -1]] = torch.tensor([math.nan, -math.inf])
            grads.append(g.to(dt))
        _step(want, grads, seed=seed), _step(got, [g.cuda() for g in grads], seed=seed)
        for name in ("m", "v", "m_scale", "v_scale"):
            assert all(_same(a, b) for a, b in zip(got[name], want[name])), (k, name)
        if kind == "odd" and k >= 20:
            assert all(b.float().isnan().sum() == 2 for b in want["m"])


@pytest.mark.parametrize("step", [2 ** 31 - 2, 2 ** 32 - 2, 2 ** 39])
def test_counts_of_steps_that_are_large(step):
    want = _state([(512,), (100,)], torch.float32, step)
    got = _on_gpu(want)
    gen = torch.Generator().manual_seed(6)
    for k in range(3):
        grads = [torch.randn(x.shape, generator=gen) for x in want["params"]]
        _step(want, grads), _step(got, [g.cuda() for g in grads])
        for name in ("m", "v", "m_scale", "v_scale"):
            assert all(_same(a, b) for a, b in zip(got[name], want[name])), (k, name)
    assert [int(t) for t in got["steps"]] == [step + 3, step + 4]


def test_replays_go_on_rounding_anew():
    """Gradients that stay the same, captured: the moments' mean follows the one in 32 bits, which it does only if every replay draws other bits."""
    from fuselink_b200.ops import adamw
    n = 8192
    got = _on_gpu(_state([(n,)], torch.float32))
    grad = torch.ones(n, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _step(got, [grad])
    for k in range(300):
        graph.replay()
    torch.cuda.synchronize()
    m, root = (adamw.decode(got[name][0].cpu(), got[name + "_scale"][0].cpu()).double().mean() for name in ("m", "v"))
    # codes of 1 and of 0.51 are 2^-3 and 2^-4 apart, their variance a quarter of that times the moment, and what that moves means by at most 2^-6 of them
    assert abs(m - 1) <= 2.0 ** -5 and abs(root / math.sqrt(1 - 0.999 ** 300) - 1) <= 2.0 ** -5
