"""Sampling (csrc/kernels/sampling.cu) against its definition in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DT = [torch.bfloat16, torch.float16]


def _logits(rows, vocab, dt, seed=1, scale=3.0):
    return (scale * torch.randn(rows, vocab, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")).to(dt)


def _u(rows, seed=2, dtype=torch.float32):
    return torch.rand(rows, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda", dtype=dtype)


def _per_row(rows, values, dtype, seed):
    at = torch.randint(0, len(values), (rows,), generator=torch.Generator().manual_seed(seed))
    return torch.tensor(values, dtype=dtype)[at].cuda()


def _check(got, logits, u, *limits):
    """Tokens and logarithms against the plain form on the CPU, which runs in 64 bits."""
    from fuselink_b200.ops.sampling import sample
    tokens, logprobs = sample(logits.cpu(), u.cpu(), *(t.cpu() if torch.is_tensor(t) else t for t in limits))
    assert got[0].tolist() == tokens.tolist()
    a, b = got[1].cpu(), logprobs
    assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.isinf(), b.isinf())
    ok = b.isfinite()
    assert ((a - b).abs()[ok] <= 2.0 ** -23 * b.abs()[ok] + 1e-12).all()        # each rounded once to fp32, from sums in 64 bits


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("rows,vocab", [(1, 1), (2, 7), (3, 1000), (1, 50257), (5, 50257), (40, 50272), (2, 65528), (2, 65529), (17, 128256), (300, 32000), (1, 524224)])
def test_sample(dt, rows, vocab):
    from fuselink_b200.ops.sampling import sample
    x, u = _logits(rows, vocab, dt), _u(rows)
    limits = (_per_row(rows, [0.5, 0.7, 1.0, 1.5, 0.0], torch.float32, 1), _per_row(rows, [0, 1, 40, 500], torch.int32, 2), _per_row(rows, [1.0, 0.5, 0.9, 0.99], torch.float32, 3),
              _per_row(rows, [0.0, 0.02, 0.3], torch.float32, 4))
    _check(sample(x, u, *limits), x, u, *limits)


@pytest.mark.parametrize("limits", [(1.0, 0, 1.0, 0.0), (0.0, 0, 1.0, 0.0), (0.7, 50, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (1.0, 0, 1.0, 0.05), (0.9, 1000, 0.95, 0.001), (1.0, 1, 1.0, 0.0),
                                    (1.0, 0, 0.0, 0.0), (1.0, 0, 1.0, 1.0), (1.0, 0, 1.0, 7.0), (math.inf, 0, 1.0, 0.0), (1e-30, 0, 1.0, 0.0), (100.0, 0, 0.5, 0.0), (1.0, 10 ** 12, 2.0, -1.0),
                                    (math.nan, 3, 0.5, 0.5), (1.0, -3, math.nan, math.nan), (-1.0, 0, 1.0, 0.0)])
def test_each_limit(limits):
    from fuselink_b200.ops.sampling import sample
    x, u = _logits(24, 5003, torch.bfloat16, seed=5), _u(24, seed=6, dtype=torch.float64)
    u[:4] = torch.tensor([0.0, 1 - 2.0 ** -53, 0.5, 2.0 ** -60], dtype=torch.float64)
    _check(sample(x, u, *limits), x, u, *limits)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("vocab", [1000, 40000, 128256])
def test_rows_that_are_not_ordinary(dt, vocab):
    """Equal logits everywhere, masks by -inf and by the type's lowest value, one token left, none, NaN, +inf; numbers outside [0, 1)."""
    from fuselink_b200.ops.sampling import sample
    x = _logits(16, vocab, dt, seed=7)
    x[0] = 0.0
    x[1] = -0.0
    x[1, ::2] = 0.0                                                    # the same number
    x[2, 1:] = -math.inf
    x[2, 0] = -3.0
    x[3] = -math.inf
    x[4, vocab // 2:] = -math.inf
    x[5, : vocab - 3] = torch.finfo(dt).min
    x[6] = torch.finfo(dt).min
    x[7, vocab - 1] = math.nan
    x[7, 77] = -math.nan
    x[8, 5], x[8, vocab - 2] = math.inf, math.inf
    x[9] = torch.finfo(dt).max
    x[10, :] = x[10, 0]
    x[11, 3:] = x[11, 3:].clamp(max=-200)
    u = _u(16, seed=8, dtype=torch.float64)
    u[12:] = torch.tensor([math.nan, -1.0, 1.0, 5.0], dtype=torch.float64)
    for limits in ((1.0, 0, 1.0, 0.0), (0.8, 7, 0.9, 0.1), (0.0, 0, 1.0, 0.0), (1.0, vocab // 2, 1.0, 0.0)):
        _check(sample(x, u, *limits), x, u, *limits)


def test_equal_logits_are_taken_in_their_order():
    """Uniform rows have sums without rounding: the token is floor(u * left)."""
    from fuselink_b200.ops.sampling import sample
    vocab, rows = 30000, 512
    x = torch.full((rows, vocab), 1.5, dtype=torch.float16, device="cuda")
    u = _u(rows, seed=3, dtype=torch.float64)
    for k in (0, 1, 1000):
        tokens, logprobs = sample(x, u, 1.0, k)
        left = k or vocab
        assert torch.equal(tokens, (u * left).floor().long()) and (logprobs.double() + math.log(left)).abs().max() <= 2.0 ** -23 * math.log(left + 1)


def test_frequencies():
    """Numbers spread evenly over [0, 1) give every token as often as its probability says, to one draw at either end of its stretch."""
    from fuselink_b200.ops.sampling import sample
    n, vocab = 4096, 50
    x = _logits(1, vocab, torch.bfloat16, seed=4, scale=1.0).expand(n, vocab)             # stride 0 between rows
    u = ((torch.arange(n, dtype=torch.float64) + 0.5) / n).cuda()
    tokens, logprobs = sample(x, u, 0.8)
    p = (x[0].double() / 0.8).softmax(0)
    assert (torch.bincount(tokens, minlength=vocab) - n * p).abs().max() <= 1
    assert ((logprobs.double() - p.log()[tokens]).abs() <= 1e-6).all()


def test_rows_anywhere_in_memory():
    from fuselink_b200.ops.sampling import sample
    base = _logits(9, 4001, torch.float16, seed=9)
    for x in (base[:, 1:], base[:, 3: 3998], base[::2, 7:], base[:, ::2], base[3:4].expand(5, -1)):
        u = _u(x.shape[0])
        _check(sample(x, u, 1.0, 100, 0.9, 0.0), x, u, 1.0, 100, 0.9, 0.0)


def test_a_captured_draw_reads_its_numbers_anew():
    from fuselink_b200.ops.sampling import Sampler
    x = _logits(16, 128256, torch.bfloat16)
    s = Sampler(torch.zeros(16, device="cuda"), 0.8, 50, 0.95, logprobs=torch.zeros(16, device="cuda"))
    s(x)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        tokens = s(x)
    for seed in range(3):
        s.u.copy_(_u(16, seed=seed))
        g.replay()
        torch.cuda.synchronize()
        _check((tokens, s.logprobs), x, s.u, 0.8, 50, 0.95, 0.0)


def test_more_rows_than_a_grid_is_high():
    from fuselink_b200.ops.sampling import sample
    x = _logits(1000, 16, torch.bfloat16).repeat(70, 1)
    u = _u(70000, dtype=torch.float64)
    tokens, _ = sample(x, u, 1.0, 0, 1.0, 0.0)
    v, order = torch.sort(x.float(), dim=1, descending=True, stable=True)
    c = (v.double() - v[:, :1].double()).exp().cumsum(1)
    want = order.gather(1, (c <= u[:, None] * c[:, -1:]).sum(1, keepdim=True))[:, 0]
    assert torch.equal(tokens, want)


def test_calls_that_are_refused():
    from fuselink_b200.ops.sampling import sample
    x, u = _logits(3, 100, torch.bfloat16), _u(3)
    for a in ((x.float(), u), (x, u.half()), (x, u[:2]), (x[0], u), (x[:, :0], u), (x, u, torch.ones(2, device="cuda")), (x, u, 1.0, torch.ones(2, device="cuda")),
              (x, u.cpu()), (x, u, torch.ones(3)), (torch.zeros(1, 524225, dtype=torch.bfloat16, device="cuda"), u[:1])):
        with pytest.raises((RuntimeError, ValueError)):
            sample(*a)
    tokens, logprobs = sample(x[:0], u[:0])
    assert tokens.shape == (0,) and logprobs.shape == (0,)


@pytest.mark.parametrize("rows,vocab", [(1, 50257), (5, 32000), (16, 128256)])
def test_draws_behind_a_product_see_all_of_it(rows, vocab):
    """The decoder's last product and the draw, one after the other over and over, the product's output in memory that the last one's held: the draw is
    on the GPU while the product stores."""
    from fuselink_b200 import C
    from fuselink_b200.ops.sampling import sample
    g = torch.Generator(device="cuda").manual_seed(3)
    w = torch.randn(vocab, 256, generator=g, device="cuda").to(torch.bfloat16)
    xs = [torch.randn(rows, 256, generator=g, device="cuda").to(torch.bfloat16) / 4 for _ in range(40)]
    u = _u(rows, seed=4)
    want = []
    for x in xs:
        logits = C.dec_product(x, w, None, 3, True)
        torch.cuda.synchronize()
        want.append(sample(logits, u, 0.8, 0, 0.95))
        torch.cuda.synchronize()
    got = [sample(C.dec_product(x, w, None, 3, True), u, 0.8, 0, 0.95) for x in xs]
    torch.cuda.synchronize()
    for (a, p), (b, q) in zip(got, want):
        assert torch.equal(a, b) and torch.equal(p, q)
