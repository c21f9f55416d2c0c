"""The operators around the expert layers in training (ops/embedding.py, routing.py, losses.py, adamw.py) on the CPU: their plain forms against
independent ones, their gradients against differences, and what they refuse."""
import ctypes
import math
import os

import pytest
import torch

from fuselink_b200.ops import adamw, embedding, losses, routing

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _gen(seed=0):
    return torch.Generator().manual_seed(seed)


def test_lookup():
    table = torch.randn(9, 5, generator=_gen(), dtype=torch.float64, requires_grad=True)
    ids = torch.tensor([[0, 8, 3], [3, -1, -9]])
    assert torch.equal(embedding.lookup(table, ids, 2.5), table[ids] * 2.5)
    assert torch.autograd.gradcheck(lambda t: embedding.lookup(t, ids, 2.5), table)
    half = table.detach().to(torch.bfloat16)
    assert torch.equal(embedding.lookup(half, ids.int(), 1 / 3), (half.float()[ids] * (1 / 3)).to(torch.bfloat16))
    for t in (torch.tensor([9]), torch.tensor([-10])):
        with pytest.raises(IndexError):
            embedding.lookup(table, t)
    for error, args in ((ValueError, (table[0], ids)), (ValueError, (table[:0], ids)), (RuntimeError, (table, ids.float()))):
        with pytest.raises(error):
            embedding.lookup(*args)


def _by_loops(logits, topk, score, bias, groups, kept, best, renormalize, scale):
    """Token by token, in Python's own numbers."""
    weights, experts = [], []
    for row in logits.tolist():
        E = len(row)
        if score == "sigmoid":
            p = [1 / (1 + math.exp(-x)) if x > -700 else 0.0 for x in row]
        else:
            top = max(row)
            e = [math.exp(x - top) for x in row]
            p = [x / math.fsum(e) for x in e]
        c = p if bias is None else [a + b for a, b in zip(p, bias.tolist())]
        size = E // groups
        value = [sum(sorted(c[g * size:(g + 1) * size], reverse=True)[:best]) for g in range(groups)]
        live = sorted(sorted(range(groups), key=lambda g: (-value[g], g))[:kept])
        order = row if bias is None else c
        mine = sorted((e for g in live for e in range(g * size, (g + 1) * size)), key=lambda e: (-order[e], e))[:topk]
        total = math.fsum(p[e] for e in mine) if renormalize else 1.0
        experts.append(mine)
        weights.append([scale * p[e] / total for e in mine])
    return torch.tensor(weights, dtype=torch.float64), torch.tensor(experts, dtype=torch.int32)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,topk,groups,kept,best", [(1, 1, 1, 1, 1), (7, 3, 1, 1, 1), (16, 4, 4, 2, 2), (16, 4, 4, 2, 1), (24, 6, 3, 1, 2), (8, 8, 8, 8, 1)])
@pytest.mark.parametrize("renormalize", [True, False])
def test_route(E, topk, groups, kept, best, score, renormalize):
    x = (2 * torch.randn(30, E, generator=_gen(E), dtype=torch.float64)).mul(4).round().div(4)          # many equal ones
    for bias in (None, torch.randn(E, generator=_gen(1)).mul(2).round().div(8)):
        r = routing.route(x, topk, score=score, bias=bias, groups=groups, topk_groups=kept, group_best=best, renormalize=renormalize, scale=1.5, balance=True)
        w, e = _by_loops(x, topk, score, bias, groups, kept, best, renormalize, 1.5)
        assert torch.equal(r.experts, e) and torch.equal(r.load, torch.bincount(e.reshape(-1), minlength=E).int())
        torch.testing.assert_close(r.weights.double(), w, rtol=2.0 ** -23, atol=1e-30)
        p = torch.sigmoid(x) if score == "sigmoid" else torch.softmax(x, 1)
        balance = (r.load / (30 * topk) * (p / p.sum(1, keepdim=True)).mean(0)).sum() * E
        torch.testing.assert_close(r.balance.double(), balance, rtol=2.0 ** -22, atol=0)


def test_route_without_a_choice():
    x = torch.full((3, 8), -math.inf)
    x[1, 5] = 1.0
    x[2, 4] = math.nan
    for score in ("softmax", "sigmoid"):
        x.requires_grad_(False)
        leaf = x.clone().requires_grad_(True)
        r = routing.route(leaf, 2, score=score)
        assert r.experts[0].tolist() == [0, 1] and r.experts[1].tolist() == [5, 0] and r.experts[2].tolist() == [4, 0]
        assert r.weights[0].tolist() == [0, 0] and r.weights[1].tolist() == [1, 0] and r.weights[2, 0].isnan()
        g, = torch.autograd.grad(r.weights[:2].sum(), leaf)
        assert (g[0] == 0).all()
    assert routing.route(torch.zeros(0, 4), 2, balance=True).load.tolist() == [0, 0, 0, 0]


def test_what_route_refuses():
    x, b = torch.zeros(4, 8), torch.zeros(8)
    for error, args, how in ((ValueError, (x, 9), {}), (ValueError, (x, 0), {}), (ValueError, (x[0], 1), {}), (ValueError, (x[:, :0], 1), {}), (ValueError, (x, 2), dict(score="relu")),
                             (ValueError, (x, 2), dict(groups=3)), (ValueError, (x, 2), dict(groups=0)), (ValueError, (x, 5), dict(groups=2, topk_groups=1)),
                             (ValueError, (x, 2), dict(groups=8)), (ValueError, (x, 2), dict(groups=2, group_best=3)), (ValueError, (x, 2), dict(bias=b[:3])),
                             (ValueError, (x, 2), dict(offset=b.double())), (ValueError, (x, 2), dict(scale=0.0)), (ValueError, (x, 2), dict(scale=math.nan)),
                             (RuntimeError, (x, 2), dict(bias=b.clone().requires_grad_(True)))):
        with pytest.raises(error):
            routing.route(*args, **how)


def test_logprobs_and_policy_loss():
    x = (2 * torch.randn(4, 6, 11, generator=_gen(), dtype=torch.float64)).requires_grad_(True)
    t = torch.randint(0, 11, (4, 6), generator=_gen(1))
    want = torch.log(torch.softmax(x / 0.7, -1)).gather(-1, t[..., None])[..., 0]
    got = losses.token_logprobs(x, t, temperature=0.7)
    torch.testing.assert_close(got.double(), want, rtol=2.0 ** -23, atol=1e-7)
    f = torch.nn.functional.cross_entropy((x / 0.7).view(-1, 11), t.view(-1))
    torch.testing.assert_close(torch.autograd.grad(got.mean(), x)[0], -torch.autograd.grad(f, x)[0], rtol=1e-6, atol=1e-9)
    old, A = want.detach().float() + 0.3 * torch.randn(4, 6, generator=_gen(2)), torch.randn(4, 6, generator=_gen(3))
    ref, w = want.detach().float() + 0.3 * torch.randn(4, 6, generator=_gen(4)), torch.rand(4, 6, generator=_gen(5))
    r = losses.policy_loss(x, t, old, A, weights=w, reference=ref, kl=0.1, clip=(0.1, 0.3), temperature=0.7)
    total, clipped, away = 0.0, 0.0, 0.0
    for lp, o, a, rf, wt in zip(*(v.detach().double().reshape(-1).tolist() for v in (want, old, A, ref, w))):
        q = math.exp(lp - o)
        held = min(max(q, 0.9), 1.3)
        k = math.exp(rf - lp) - (rf - lp) - 1
        total, clipped, away = total + wt * (0.1 * k - min(q * a, held * a)), clipped + wt * (q * a > held * a), away + wt * k
    s = float(w.double().sum())
    assert abs(float(r.loss.detach()) - total / s) < 1e-6 and abs(float(r.clipped) - clipped / s) < 1e-6 and abs(float(r.divergence) - away / s) < 1e-6
    assert r.loss.requires_grad and not r.logprobs.requires_grad and 0 < float(r.clipped) < 1
    g, = torch.autograd.grad(r.loss, x)
    d, h = torch.randn(x.shape, generator=_gen(6), dtype=torch.float64), 2.0 ** -10
    call = lambda y: losses.policy_loss(y, t, old, A, weights=w, reference=ref, kl=0.1, clip=(0.1, 0.3), temperature=0.7)  # noqa: E731
    a, b = call(x + h * d), call(x - h * d)
    # no ratio crosses its border on the way: then only the third derivative (of order 1 along d, per token) and fp32 results part the two
    assert float(a.clipped) == float(b.clipped) == float(r.clipped)
    assert abs(float((g * d).sum()) - (float(a.loss.detach()) - float(b.loss.detach())) / (2 * h)) < 50 * h * h + 2.0 ** -23 * 2 / h
    # rows of weight 0 are not looked at
    y = x.detach().clone()
    y[0], w[0] = math.nan, 0
    assert losses.policy_loss(y, t, old, A, weights=w).loss.isfinite()
    half = losses.policy_loss(x, t, old, A, total=48.0)
    assert abs(float(half.loss.detach()) * 2 - float(losses.policy_loss(x, t, old, A).loss.detach())) < 1e-6
    assert losses.token_logprobs(x, torch.full_like(t, 11)).isnan().all()


def test_what_the_losses_refuse():
    x, t, f = torch.zeros(4, 9), torch.zeros(4, dtype=torch.int64), torch.zeros(4)
    for error, args, how in ((ValueError, (x, t[:3]), {}), (ValueError, (x, t.float()), {}), (ValueError, (x[:, :0], t), {}), (ValueError, (x, t), dict(temperature=0.0)),
                             (ValueError, (x, t), dict(temperature=math.inf)), (ValueError, (x, t), dict(temperature=1e-40))):
        with pytest.raises(error):
            losses.token_logprobs(*args, **how)
    for error, how in ((RuntimeError, dict(advantages=torch.zeros(3))), (RuntimeError, dict(old=f.clone().requires_grad_(True))), (ValueError, dict(clip=(0.2, math.nan))),
                       (ValueError, dict(kl=-0.1)), (ValueError, dict(total=f))):
        with pytest.raises(error):
            losses.policy_loss(x, t, **{**dict(old=f, advantages=f), **how})


def test_adamw_against_the_library():
    ps = [torch.nn.Parameter(torch.randn(s, generator=_gen(i))) for i, s in enumerate(((40, 9), (3,), (1000,)))]
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    a, b = adamw.AdamW(ps, lr=1e-2, betas=(0.9, 0.95), weight_decay=0.1), torch.optim.AdamW(qs, lr=1e-2, betas=(0.9, 0.95), weight_decay=0.1)
    for k in range(6):
        for i, (p, q) in enumerate(zip(ps, qs)):
            p.grad = torch.randn(p.shape, generator=_gen(100 * k + i))
            q.grad = p.grad.clone()
        a.step(), b.step()
    for p, q in zip(ps, qs):
        # six steps of at most 1e-2 (1 + 0.1), each with some ten roundings of fp32, and as many of the weight
        assert (p - q).abs().max() <= 6 * (10 * 2.0 ** -24 * 1.1e-2 * 10 + 2.0 ** -24 * 5)


def test_codes():
    x = torch.cat([torch.randn(256, generator=_gen()), torch.zeros(256), torch.full((256,), 1e-35), torch.logspace(-30, 10, 256), torch.tensor([math.inf, -1.0, math.nan])])
    codes, scale = adamw.encode(x)
    assert scale.tolist()[1:3] == [2.0 ** -100] * 2 and (scale.log2() == scale.log2().round()).all()
    top = x[:256].abs().max()
    assert scale[0] * 448 >= top > scale[0] * 224
    y = adamw.decode(codes, scale)
    assert (y - x)[:256].abs().max() <= 2.0 ** -4 * top and y[-3].isnan() and y[-1].isnan() and y[-2] == -1
    assert (y[:256] - x[:256]).abs().le(2.0 ** -4 * x[:256].abs() + 2.0 ** -10 * scale[0]).all()
    roots, scale = adamw.encode(x[768:1024].abs(), root=True)
    assert (roots.float() > 0).all() and (adamw.encode(x[768:1024])[0].float() == 0).any()


def test_adamw_in_eight_bits_follows_thirty_two():
    """On gradients of one scale, 20 steps: moments are off by a code's half step at most at each step, so the direction stays and its size nearly."""
    p, q = (torch.nn.Parameter(torch.zeros(2048)) for _ in range(2))
    a, b = adamw.AdamW([p], lr=1e-3, state_bits=8, weight_decay=0.0), adamw.AdamW([q], lr=1e-3, weight_decay=0.0)
    for k in range(20):
        p.grad = 1 + 0.1 * torch.randn(2048, generator=_gen(k))
        q.grad = p.grad.clone()
        a.step(), b.step()
    # each of the two moments carries an error of at most half a step (2^-4) times 1 / (1 - b) of what it gets anew, and all of it in one direction at worst only
    # for the mean, where the roundings' signs differ from weight to weight
    assert abs((p / q - 1).mean()) < 2.0 ** -4


def test_what_adamw_refuses():
    p = torch.nn.Parameter(torch.zeros(8))
    for how in (dict(lr=-1.0), dict(betas=(0.9, 1.0)), dict(eps=-1.0), dict(weight_decay=-0.1), dict(state_bits=16), dict(lr=math.nan)):
        with pytest.raises(ValueError):
            adamw.AdamW([p], **how)
    opt = adamw.AdamW([p])
    p.grad = torch.zeros(8).to_sparse()
    with pytest.raises(RuntimeError):
        opt.step()
    z = lambda: torch.zeros(8)  # noqa: E731
    with pytest.raises(RuntimeError):
        adamw.step([z()], [z()], [z()], [], [torch.tensor(0)], lr=0.1)
    with pytest.raises(RuntimeError):
        adamw.step([z()], [z().half()], [z()], [z()], [torch.tensor(0)], lr=0.1)


def test_c_entries_refuse_what_the_kernels_do_not_take():
    """The C interface says -1 before it launches anything."""
    lib = os.path.join(ROOT, "fuselink_b200", "lib", "libfuselink.so")
    if not os.path.exists(lib):
        pytest.skip("libfuselink.so not built")
    c = ctypes.CDLL(lib)
    zeros = ctypes.create_string_buffer(512)                             # every field 0
    for name in ("fl_embed", "fl_embed_grad", "fl_route", "fl_route_grad", "fl_token_logprobs", "fl_policy_loss", "fl_logprobs_grad"):
        f = getattr(c, name)
        f.argtypes = [ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p]
        assert f(0, zeros, None) == -1, name
    c.fl_embed_scratch.argtypes, c.fl_embed_scratch.restype = [ctypes.c_longlong] * 3, ctypes.c_longlong
    for sizes in ((-1, 8, 8), (2 ** 31, 8, 8), (8, 0, 8), (8, 2 ** 31, 8), (8, 8, 0)):
        assert c.fl_embed_scratch(*sizes) == -1
    need = [c.fl_embed_scratch(n, 1000, 64) for n in (0, 1, 1024, 1025, 10 ** 6)]
    assert need == sorted(need) and need[0] >= 4004
    c.fl_adamw.argtypes = [ctypes.c_int, ctypes.c_void_p, ctypes.c_longlong, ctypes.c_void_p, ctypes.c_void_p]
    assert c.fl_adamw(0, None, -1, zeros, None) == -1 and c.fl_adamw(7, None, 0, zeros, None) == -1 and c.fl_adamw(0, None, 0, zeros, None) == 0


def test_masters_start_anew_from_parameters_that_were_written():
    p = torch.nn.Parameter(torch.ones(4, dtype=torch.bfloat16))
    opt = adamw.AdamW([p], lr=1e-3, master=True, weight_decay=0.0)
    p.grad = torch.ones_like(p)
    opt.step()
    with torch.no_grad():
        p.fill_(5.0)
    opt.refresh_masters()
    opt.step()
    assert (opt.state[p]["master"] - 5).abs().max() <= 2e-3 and (p == 5).all()


def _net(**how):
    import dataclasses

    from fuselink_b200.models.moe import Gate
    from fuselink_b200.models.moe_transformer import MOE_ZOO, MoETransformer
    cfg = dataclasses.replace(MOE_ZOO["tiny_moe"], **{**dict(embed_scale=2.0, gate=Gate(groups=2, topk_groups=1, scale=1.5, balance_bias=True)), **how})
    return MoETransformer(cfg, 2 * 12, None, 0, 1, device="cpu", seed=2)


def test_gated_layers_route_as_the_operator_does():
    from fuselink_b200.models.moe import Gate, MoELayer
    from fuselink_b200.ops.moe import MoEConfig
    layer = MoELayer(MoEConfig(hidden=32, ffn=128, num_experts=8, topk=2, tokens=50), None, 0, 1, device="cpu", gate=Gate(score="softmax", balance_bias=True))
    x = torch.randn(50, 32, generator=_gen()).to(torch.bfloat16)
    w, idx = layer.route(x)
    r = routing.route(x @ layer.router.t(), 2, bias=layer.balance_bias, offset=layer.router_bias, balance=True)
    assert torch.equal(w, r.weights) and torch.equal(idx, r.experts) and torch.equal(layer.l_aux, r.balance) and torch.equal(layer.last_load, r.load)
    before = layer.balance_bias.clone()
    layer.update_balance(0.5)
    assert torch.equal(layer.balance_bias - before, 0.5 * torch.sign(50 * 2 / 8 - r.load.float()))
    assert "balance_bias" in layer.state_dict()
    layer.eval()
    layer.route(x)
    assert layer.l_aux == 0
    plain = MoELayer(MoEConfig(hidden=32, ffn=128, num_experts=8, topk=2, tokens=50), None, 0, 1, device="cpu")
    assert "balance_bias" not in plain.state_dict()
    with pytest.raises(RuntimeError):
        plain.update_balance(0.1)
    with pytest.raises(ValueError):
        MoELayer(MoEConfig(hidden=32, ffn=128, num_experts=8, topk=2, tokens=50), None, 0, 1, device="cpu", gate=Gate(), noisy_gate="rsample")


def test_a_transformer_around_its_experts():
    net = _net()
    tokens = torch.randint(0, 512, (2, 12), generator=_gen(4))
    lp = net.token_logprobs(tokens)
    want = torch.log_softmax(net(tokens).detach(), -1)[:, :-1].gather(-1, tokens[:, 1:, None])[..., 0]
    # the same logits in fp32 on either side; logarithms of magnitude 6 rounded to it
    assert lp.shape == (2, 12) and (lp[:, -1] == 0).all() and (lp[:, :-1] - want).abs().max() <= 8 * 2.0 ** -22
    old, A = lp + 0.1, torch.randn(2, 1, generator=_gen(5))
    loss, r = net.policy_loss(tokens, old, A, reference=lp, kl=0.1)
    loss.backward()
    # ratios of e^-0.1 lie inside the borders: the mean of -q A, and the divergence of a reference that is the policy itself
    assert abs(float(r.loss.detach()) + math.exp(-0.1) * float(A.mean())) < 1e-4 and float(r.clipped) == 0 and abs(float(r.divergence)) < 1e-9
    assert all(p.grad is not None and p.grad.isfinite().all() for p in net.parameters())
    seen = {}

    def look(module, inputs):
        inputs[0].register_hook(lambda g: seen.update(g=g.detach().clone()))

    net.blocks[0].register_forward_pre_hook(look)
    net.embed.grad = None
    net.policy_loss(tokens, old, A, reference=lp, kl=0.1)[0].backward()
    rows = torch.zeros(net.embed.shape, dtype=torch.float64).index_add_(0, tokens.reshape(-1), seen["g"].reshape(-1, 128).double()) * 2.0
    # bf16 gradients added up row by row by the library, each sum of at most 24 rounded to bf16
    assert ((net.embed.grad.double() - rows).abs() <= 24 * 2.0 ** -8 * rows.abs().amax(1, keepdim=True) + 1e-30).all()
    from fuselink_b200.ops.adamw import AdamW
    opt = AdamW(net.parameters(), lr=1e-3, state_bits=8)
    bias = net.blocks[0].moe.balance_bias.clone()
    r = net.policy_step(tokens, old, A, opt, weights=torch.arange(12) > 3)
    assert r.loss.isfinite() and not r.loss.requires_grad and (r.logprobs[:, :4] == 0).all() and (r.logprobs[:, -1] == 0).all()
    assert not torch.equal(bias, net.blocks[0].moe.balance_bias) and all(p.grad is None for p in net.parameters())
    assert net.train_step(tokens, torch.roll(tokens, -1, 1), opt).isfinite()


def test_the_training_command_with_every_choice():
    import subprocess
    import sys
    script = os.path.join(ROOT, "experiments", "run_moe_training.py")
    small = ["--model", "tiny_moe", "--device", "cpu", "--steps", "2", "--batch", "2", "--seq", "32", "--log-every", "1", "--lr", "0.001"]
    r = subprocess.run([sys.executable, script, *small, "--optimizer", "adamw8", "--objective", "policy", "--gate", "sigmoid", "--embed-scale", "11.3"], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.count('"loss"') == 2, r.stderr[-2000:]
    r = subprocess.run([sys.executable, script, *small, "--optimizer", "adamw", "--reshadow-every", "1"], capture_output=True, text=True, timeout=300)
    assert r.returncode == 2 and "copy slots" in r.stderr
