"""Routing of large logits with an offset (csrc/kernels/routing.cu): the sum of both is rounded in fp32, which must change neither the choice nor the weights of 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu
HALF = 2.0 ** -24


def _randn(*shape, seed):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


@pytest.mark.parametrize("shift", [0.0, 200.0, -1000.0, 30000.0])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts,topk,groups,kept,best", [(64, 8, 1, 1, 1), (64, 8, 8, 3, 2), (96, 6, 4, 2, 1), (256, 8, 8, 4, 2), (33, 4, 1, 1, 1)])
def test_large_logits_with_an_offset(experts, topk, groups, kept, best, score, shift):
    from fuselink_b200.ops.routing import route
    x = shift + 1.5 * _randn(20000, experts, seed=1)
    offset = _randn(experts, seed=2) - (shift if score == "sigmoid" else 0.0)      # sigmoids of sums that are near 0
    for bias in (None, 0.05 * _randn(experts, seed=3)):
        for renormalize in (True, False):
            how = dict(score=score, groups=groups, topk_groups=kept, group_best=best, renormalize=renormalize, scale=2.5)
            got = route(x, topk, bias=bias, offset=offset, **how)
            want = route(x.cpu().double(), topk, bias=None if bias is None else bias.cpu(), offset=offset.cpu(), **how)
            assert torch.equal(got.experts.cpu(), want.experts) and torch.equal(got.load.cpu(), want.load)
            # in half steps: exponentials of 4 each, of the sum and of what it lost, their arguments (differences from the largest, up to 16), quotients and a factor 6;
            # a sum over the chosen or a lane's experts, and 5 for the tree
            assert ((got.weights.cpu().double() - want.weights).abs() <= (experts / 32 + topk + 45) * HALF * want.weights.abs() + 1e-44).all()


def test_masked_and_infinite_sums():
    """-inf among logits or offsets stays no probability; sums beyond fp32 are what 64 bits make of them."""
    from fuselink_b200.ops.routing import route
    x, offset = 300 + _randn(500, 40, seed=4), _randn(40, seed=5)
    x[:, 3], offset[7], offset[11] = -torch.inf, -torch.inf, -3e38
    x[5], x[6, 2] = -torch.inf, 3.2e38
    for score in ("softmax", "sigmoid"):
        for renormalize in (True, False):
            got = route(x, 4, score=score, offset=offset, renormalize=renormalize)
            want = route(x.cpu().double(), 4, score=score, offset=offset.cpu(), renormalize=renormalize)
            assert torch.equal(got.experts.cpu(), want.experts)
            assert torch.equal(got.weights.isnan().cpu(), want.weights.isnan())
            assert ((got.weights.cpu().double() - want.weights).abs() <= 60 * HALF * want.weights.abs() + 1e-44).logical_or(want.weights.isnan()).all()
