"""Log-probabilities and the policy loss (csrc/kernels/losses.cu) at their edges: empty batches of any layout, extreme temperatures, logits far from 0, ratios
exactly at a border; against the definition in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DT = [torch.bfloat16, torch.float16, torch.float32]


def _empty(dt):
    full = torch.zeros(4, 5, 12, 7, device="cuda", dtype=dt)
    return [full[:0, :3, ::2], full[0, 0].t()[:0], full[:, :0, ::2, ::3], full[:0].transpose(1, 2), torch.empty(0, 2, 3, 7, device="cuda", dtype=dt).transpose(1, 2),
            full[0, 0].t()[:0, ::2], full[:0].permute(2, 0, 1, 3)[::3], full[:0, :, :, :1], full[:, :, :0, 6:]]


@pytest.mark.parametrize("weighted", [False, True])
@pytest.mark.parametrize("case", range(9))
def test_no_rows_of_any_layout(case, weighted):
    """Nothing to read whatever the sizes and strides are: the loss is 0, and so is the (empty) gradient."""
    from fuselink_b200.ops.losses import policy_loss, token_logprobs
    for dt in DT:
        x = _empty(dt)[case].detach().requires_grad_(True)
        assert x.numel() == 0
        f = torch.zeros(x.shape[:-1], device="cuda")
        t = f.long()
        r = policy_loss(x, t, f, f, weights=f if weighted else None, reference=f, kl=0.1)
        lp = token_logprobs(x, t)
        for got in (*torch.autograd.grad(r.loss, x), *torch.autograd.grad(lp, x, f)):
            assert got.shape == x.shape
        with torch.no_grad():
            again = policy_loss(x, t, f, f, weights=f if weighted else None)
        torch.cuda.synchronize()
        assert [float(v.detach()) for v in (r.loss, r.divergence, r.clipped, again.loss)] == [0.0] * 4 and lp.shape == r.logprobs.shape == t.shape
