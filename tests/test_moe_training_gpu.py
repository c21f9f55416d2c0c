"""What surrounds the expert layers of a training step, together on one GPU: embedding, routing, policy loss and AdamW in the transformer that has them."""
import dataclasses

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture
def net():
    from fuselink_b200.models.moe import Gate
    from fuselink_b200.models.moe_transformer import MoEModelConfig, MoETransformer
    from fuselink_b200.parallel.symm import SymmetricHeap
    cfg = MoEModelConfig(layers=2, hidden=256, heads=4, kv_heads=2, head_dim=64, ffn=512, num_experts=16, topk=4, vocab=1000, embed_scale=16.0,
                         gate=Gate(groups=4, topk_groups=2, scale=2.0, balance_bias=True))
    heap = SymmetricHeap.create(256 << 20, device=torch.cuda.current_device())
    yield MoETransformer(cfg, 4 * 128, heap, 0, 1, device="cuda", seed=1)
    torch.cuda.synchronize()
    heap.check_status("training")
    heap.close()


def _batch(net, seed=3):
    g = torch.Generator(device="cuda").manual_seed(seed)
    tokens = torch.randint(0, net.cfg.vocab, (4, 128), device="cuda", generator=g)
    A = torch.randn(4, 1, device="cuda", generator=g)
    weights = (torch.arange(128, device="cuda") >= torch.tensor([[5], [40], [100], [127]], device="cuda")).float()
    return tokens, A, weights


def test_step_against_the_frameworks_operations(net, monkeypatch):
    """Loss and gradients with the kernels, and with their plain forms in their places; all else is the same code on the same GPU."""
    from fuselink_b200.ops import embedding, losses, routing
    tokens, A, weights = _batch(net)
    old = net.token_logprobs(tokens) + 0.1
    ref = old - 0.3
    sides = []
    for plain in (False, True):
        if plain:
            for module in (embedding, losses, routing):
                monkeypatch.setattr(module, "ordinary", lambda t: False)
        for p in net.parameters():
            p.grad = None
        loss, r = net.policy_loss(tokens, old, A, weights=weights, reference=ref, kl=0.05)
        loss.backward()
        sides.append((float(loss.detach()), r, {n: p.grad.double() for n, p in net.named_parameters() if p.grad is not None}, [b.moe.last_topk_idx.clone() for b in net.blocks]))
    (la, ra, ga, ia), (lb, rb, gb, ib) = sides
    assert all(torch.equal(x, y) for x, y in zip(ia, ib))                 # the same experts, in the same order
    # the logits differ only where a weight of an expert rounds to another bf16 product: a few half steps of 2^-9 of a logit's spread, averaged over many
    assert abs(la - lb) <= 2.0 ** -8 * (1 + abs(lb)) and abs(float(ra.clipped) - float(rb.clipped)) <= 0.01
    assert ga.keys() == gb.keys()
    for n in ga:
        norm = gb[n].norm()
        # each value between logits and weights is rounded to bf16 on either side, a step of 2^-8 apart where the two do not agree; chains of some ten of them
        assert (ga[n] - gb[n]).norm() <= 10 * 2.0 ** -8 * norm + 1e-9, n


@pytest.mark.parametrize("bits", [8, 32])
def test_steps(net, bits):
    from fuselink_b200.ops.adamw import AdamW
    opt = AdamW(net.parameters(), lr=1e-4, state_bits=bits, master=True)
    before = {n: p.detach().clone() for n, p in net.named_parameters()}
    for k in range(3):
        tokens, A, weights = _batch(net, 10 + k)
        r = net.policy_step(tokens, net.token_logprobs(tokens), A, opt, weights=weights, kl=0.0)
        assert r.loss.isfinite() and r.clipped == 0                       # of a policy that is its own
    for n, p in net.named_parameters():
        s = opt.state[p]
        assert int(s["step"]) == 3 and torch.equal(p, s["master"].to(p.dtype)) and p.isfinite().all(), n
        assert (s["master"] != before[n].float()).any(), n
    assert all((b.moe.balance_bias != 0).any() for b in net.blocks)
    tokens[0, 0] = net.cfg.vocab
    net(tokens)
    torch.cuda.synchronize()
    with pytest.raises(IndexError):
        net(tokens)


def test_a_step_captured_and_replayed(net):
    """Forward and backward of the operators between given hidden states, with the optimizer, as one graph: what replays give is what calls give."""
    from fuselink_b200.ops import adamw, embedding, losses, routing
    cfg = net.cfg
    g = torch.Generator(device="cuda").manual_seed(5)
    table = (0.02 * torch.randn(cfg.vocab, cfg.hidden, generator=g, device="cuda")).to(torch.bfloat16)
    router = (0.2 * torch.randn(16, cfg.hidden, generator=g, device="cuda")).to(torch.bfloat16)
    tokens, A, weights = _batch(net)
    old = torch.full((4, 128), -6.9, device="cuda")

    def state():
        ps = [table.clone(), router.clone()]
        return ps, [torch.zeros_like(p, dtype=torch.float32) for p in ps], [torch.zeros_like(p, dtype=torch.float32) for p in ps], [torch.zeros((), dtype=torch.int64, device="cuda") for _ in ps]

    def step(ps, m, v, steps):
        t, w = (p.detach().requires_grad_(True) for p in ps)
        x = embedding.lookup(t, tokens, 16.0)
        r = routing.route(x.view(-1, cfg.hidden) @ w.t(), 4, score="sigmoid", groups=4, topk_groups=2, balance=True)
        y = x * r.weights.sum(1).view(4, 128, 1).to(x.dtype) * r.weights[:, 0].view(4, 128, 1).to(x.dtype)
        loss = losses.policy_loss(y @ t.t(), torch.roll(tokens, -1, 1), old, A, weights=weights)
        grads = torch.autograd.grad(loss.loss + 0.01 * r.balance, [t, w])
        adamw.step(ps, list(grads), m, v, steps, lr=1e-3)
        return loss.loss.detach()

    eager, replayed = state(), state()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*state())
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*replayed)
    for s in replayed[1] + replayed[2]:
        s.zero_()
    for k in range(3):
        new, A2, _ = _batch(net, 20 + k)
        tokens.copy_(new), A.copy_(A2)
        want = step(*eager)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        for a, b in zip(eager, replayed):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
