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


HALF = 2.0 ** -24


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _off(vocab):
    """How far a row's logarithm may be, in 32 bits.  A thread adds up to vocab / 64 pairs of exponentials, and some 24 sums join threads; the hardware's exponential is off by 4
    half steps; an argument a by 2 half steps of itself (its factor's rounding and its own), and the mean of a over the row is ln(vocab) at most."""
    return (vocab / 64 + 28 + 2 * math.log(vocab)) * HALF


def _check_rows(x, temperature, tokens, shift=0.0):
    """Log-probabilities, their gradient and the policy loss of rows x [n, vocab] against 64 bits; dlp / dx has a factor of 1 / T, so its derivatives come with a factor of T."""
    from fuselink_b200.ops.losses import policy_loss, token_logprobs
    n, V = x.shape
    leaf = x.detach().requires_grad_(True)
    y = x.detach().cpu().double() / temperature
    lp64 = torch.log_softmax(y, 1)
    want = lp64.gather(1, tokens.cpu()[:, None])[:, 0]
    off = _off(V)
    lp = token_logprobs(leaf, tokens, temperature=temperature)
    assert ((lp.detach().cpu().double() - want).abs() <= off + 2 * HALF * want.abs()).all()
    each = torch.randn(n, generator=_gen(7), device="cuda") * temperature
    p, g = lp64.exp(), (each.cpu().double() / temperature)[:, None]
    onehot = torch.zeros_like(p).scatter_(1, tokens.cpu()[:, None], 1.0)

    def near(got, g, rows=slice(None), more=0.0):
        w = (g * (onehot - p))[rows]
        # a probability is off as its row's logarithm is, and by its own argument's steps; a factor and a product round, and `more` is the factor's own
        tol = (g.abs() * p)[rows] * (off + (8 + 4 * lp64[rows].abs().clamp(max=200)) * HALF) + w.abs() * (torch.finfo(got.dtype).eps / 2 + 4 * HALF + more)
        assert ((got.detach().cpu().double()[rows] - w).abs() <= tol + torch.finfo(got.dtype).tiny * (1 + g.abs().max())).all()

    if each.abs().min() > 1e-36 and each.abs().max() < 1e36:
        near(torch.autograd.grad(lp, leaf, each)[0], g)
    # `old` is the kernel's own logarithm, but rounded to 32 bits: a ratio is exp(d) with |d| of at most a half step of it, d + d^2 off from 1 where d is small.  Where |lp| is
    # of the order of 2^24 or more that is any number, so rows below 2^14 are looked at: each row's gradient is its own.
    r = policy_loss(leaf, tokens, lp.detach(), torch.ones(n, device="cuda"), temperature=temperature)
    assert torch.equal(r.logprobs, lp)
    rows = want.abs() < 2.0 ** 14
    more = (HALF * want.abs()[rows, None]) * 1.01 + 4 * HALF             # and exp's own rounding, of a result near 1
    if rows.all():
        assert abs(float(r.loss.detach()) + 1) <= float(more.max()) + 2 * HALF
    if 1e-30 < temperature < 1e36:
        got, = torch.autograd.grad(r.loss * temperature, leaf)
        near(got, torch.full((n, 1), -1.0 / n, dtype=torch.float64), rows, more)


@pytest.mark.parametrize("temperature", [1e-30, 1e-12, 1e-9, 1e-8, 1e-6, 2e-5, 1e-5, 1e-3, 1e3, 1e30, 1e38, 1e44, 1e60, 1e300])
@pytest.mark.parametrize("n,vocab", [(3, 5), (5, 300), (4, 3001), (7, 9001), (3, 40001), (1300, 517), (700, 5003)])
def test_any_temperature_that_is_accepted(n, vocab, temperature):
    """Few rows and many (512 threads a row, 256, 128 and a warp), rows with fewer vectors than threads, and rows of many.  The token is the likeliest, the next or any."""
    for dt in DT:
        x = (2 * torch.randn(n, vocab, generator=_gen(vocab), device="cuda")).to(dt)
        best = x.float().topk(2, dim=1)[1]
        tokens = torch.where(torch.arange(n, device="cuda") % 3 == 0, best[:, 0], best[:, 1])
        if temperature >= 1e-3:
            tokens[1::3] = torch.randint(0, vocab, (len(tokens[1::3]),), generator=_gen(1), device="cuda")
        _check_rows(x, temperature, tokens)


@pytest.mark.parametrize("temperature", [1e-9, 1.0, 1e40, 1e200])
def test_masked_logits_at_any_temperature(temperature):
    from fuselink_b200.ops.losses import token_logprobs
    for dt in DT:
        x = (2 * torch.randn(6, 3000, generator=_gen(4), device="cuda")).to(dt)
        x[:, ::2] = -math.inf
        x[5] = -math.inf
        leaf, t = x.requires_grad_(True), torch.tensor([1, 3, 5, 7, 2, 1], device="cuda")
        lp = token_logprobs(leaf, t, temperature=temperature)
        want = torch.log_softmax(x.detach().cpu().double() / temperature, 1).gather(1, t.cpu()[:, None])[:, 0]
        assert lp[4] == -math.inf and lp[5].isnan()
        assert ((lp.detach().cpu().double() - want)[:4].abs() <= _off(3000) + 2 * HALF * want[:4].abs()).all()
        g, = torch.autograd.grad(lp, leaf, torch.full((6,), min(temperature, 1e30), device="cuda"))
        assert (g[:5, ::2][torch.arange(0, 3000, 2, device="cuda").expand(5, -1) != t[:5, None]] == 0).all() and g[:5].isfinite().all()
        # 1e30 / 1e200 is 0 in 32 bits, and a row whose derivative is 0 has a gradient of 0 unread
        assert (g[5] == 0).all() if temperature == 1e200 else g[5].isnan().all()


def test_logits_at_the_ends_of_their_type():
    """Differences that are beyond the type, at temperatures that bring them back."""
    from fuselink_b200.ops.losses import token_logprobs
    for vocab in (7, 2000):
        x = torch.zeros(2, vocab, device="cuda")
        x[:, 0], x[:, -1] = 3e38, -3e38
        for temperature in (1e38, 3e38, 1e39):
            t = torch.tensor([0, vocab - 1], device="cuda")
            lp = token_logprobs(x, t, temperature=temperature).cpu().double()
            want = torch.log_softmax(x.cpu().double() / temperature, 1).gather(1, t.cpu()[:, None])[:, 0]
            # and a factor of fewer bits where it is below 2^-126: half of 2^-149, times 3e38
            assert ((lp - want).abs() <= _off(vocab) + 2 * HALF * want.abs() + 6e38 * 2.0 ** -150 * 2).all()


@pytest.mark.parametrize("shift", [0.0, 1e3, -1e4, 1e5, -1e6, 5e6, 1e7])
@pytest.mark.parametrize("n,vocab,temperature", [(388, 2048, 1.0), (1300, 1999, 0.7), (700, 5003, 1.3), (5, 32768, 1.0)])
def test_logits_far_from_zero(n, vocab, temperature, shift):
    """A common offset changes nothing but which logits fp32 has: sums stay as exact as without it while a thread's maximum rises."""
    x = 2 * torch.randn(n, vocab, generator=_gen(11), device="cuda")
    x = x.sort(dim=1)[0] if n == 388 else x                             # maxima that rise all the time
    _check_rows(x + shift, temperature, torch.randint(0, vocab, (n,), generator=_gen(12), device="cuda"))


def test_at_a_border_exactly_the_ratio_still_counts():
    """Two equal logits: lp is -ln 2, and rounded to 32 bits it is 1.9e-9 from that, so the ratio rounds to 1, the border of a clip of 0 on either side.  Nothing is clipped, and the
    gradient is that of the open term; one unit away, on the side where the advantage is held, it is 0."""
    from fuselink_b200.ops.losses import policy_loss
    t, A = torch.tensor([0, 1, 0, 1], device="cuda"), torch.tensor([1.0, -1.0, 2.0, -0.5], device="cuda")
    leaf = torch.zeros(4, 2, device="cuda").requires_grad_(True)
    old = torch.full((4,), -math.log(2), device="cuda")
    for dt in (torch.float32, torch.bfloat16):
        x = leaf.to(dt)
        r = policy_loss(x, t, old, A, clip=(0.0, 0.0))
        assert r.clipped == 0 and r.loss == -A.mean()
        g, = torch.autograd.grad(r.loss, leaf)
        onehot = torch.nn.functional.one_hot(t, 2).float()
        assert torch.equal(g, -A[:, None] / 4 * (onehot - 0.5))
        away = policy_loss(x, t, old - torch.where(A > 0, 1e-4, -1e-4), A, clip=(0.0, 0.0))
        assert away.clipped == 1 and (torch.autograd.grad(away.loss, leaf)[0] == 0).all()
    one = policy_loss(torch.full((3, 1), 5.0, device="cuda"), t[:3] * 0, old[:3] * 0, A[:3], clip=(0.0, 0.0))
    assert one.clipped == 0 and one.loss == -A[:3].mean() and (one.logprobs == 0).all()
