"""What surrounds the training operators, on the CPU: waits between launches as the sources have them, states that are saved and go on, gates on several ranks."""
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _body(source, function):
    text = open(os.path.join(ROOT, "fuselink_b200", "csrc", "kernels", source)).read()
    text = text[text.index("{", text.index(" " + function + "(const")):]
    depth = 0
    for i, c in enumerate(text):
        depth += (c == "{") - (c == "}")
        if depth == 0:
            return text[:i]


def test_every_cta_of_a_kernel_that_starts_early_waits():
    """A CTA that ended without a wait could let what follows begin, and reuse memory, while the kernel in front still works on it."""
    body = _body("losses.cu", "loss_kernel")
    loop, end = body.split("if (policy && threadIdx.x == 0) {")
    assert re.search(r"if \(!asked\) \{\s*asked = true;\s*grid_dep_wait\(\);", loop) and re.search(r"if \(!asked\) grid_dep_wait\(\);", end)
    body = _body("embedding.cu", "embed_sum_kernel")
    assert "return" not in body[:body.index("grid_dep_wait();")]


def _command():
    import importlib.util
    spec = importlib.util.spec_from_file_location("run_moe_training", os.path.join(ROOT, "experiments", "run_moe_training.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def _training(optimizer, lr=1e-2):
    import dataclasses

    import torch

    from fuselink_b200.models.moe import Gate
    from fuselink_b200.models.moe_transformer import MOE_ZOO, MoETransformer
    from fuselink_b200.ops.adamw import AdamW
    cfg = dataclasses.replace(MOE_ZOO["tiny_moe"], embed_scale=2.0, gate=Gate(balance_bias=True))
    net = MoETransformer(cfg, 2 * 8, None, 0, 1, device="cpu", seed=3, dtype=torch.bfloat16)
    if optimizer == "sgd":
        return net, torch.optim.SGD(net.parameters(), lr=lr)
    return net, AdamW(net.parameters(), lr=lr, state_bits=8 if optimizer == "adamw8" else 32, master=True)


def _steps(net, opt, first, last):
    import torch
    for k in range(first, last):
        tokens = torch.randint(0, net.cfg.vocab, (2, 8), generator=torch.Generator().manual_seed(k))
        net.train_step(tokens, torch.roll(tokens, -1, 1), opt)


@pytest.mark.parametrize("optimizer", ["sgd", "adamw", "adamw8"])
def test_a_resumed_run_goes_on_as_if_it_had_not_stopped(optimizer, tmp_path):
    """Five steps are three, a save, a load into a new program, and two: weights, moments, counts and fp32 copies, bit by bit."""
    import torch
    command = _command()
    whole = _training(optimizer)
    _steps(*whole, 0, 5)
    before = _training(optimizer)
    _steps(*before, 0, 3)
    torch.save(command.last_state(*before), tmp_path / "ck")
    after = _training(optimizer)
    command.go_on_from(torch.load(tmp_path / "ck", map_location="cpu"), *after)
    _steps(*after, 3, 5)
    for (name, a), b in zip(whole[0].state_dict().items(), after[0].state_dict().values()):
        assert torch.equal(a, b), name
    for p, q in zip(whole[0].parameters(), after[0].parameters()):
        s, t = whole[1].state.get(p, {}), after[1].state.get(q, {})
        assert s.keys() == t.keys() and all(s[k] is None or (s[k].dtype == t[k].dtype and torch.equal(s[k].float(), t[k].float())) for k in s)
        assert optimizer == "sgd" or int(t["step"]) == 5


def test_what_resuming_takes_and_refuses():
    import torch
    command = _command()
    net, opt = _training("adamw8")
    _steps(net, opt, 0, 1)
    state = command.last_state(net, opt)
    for optimizer in ("sgd", "adamw8"):                       # a model's state alone, as SGD's runs write it, and AdamW's under SGD
        new = _training(optimizer, lr=0.5)
        command.go_on_from(state["model"], *new)
        assert torch.equal(new[0].embed, net.embed) and not new[1].state
    new = _training("sgd", lr=0.5)
    command.go_on_from(state, *new)
    assert torch.equal(new[0].embed, net.embed)
    new = _training("adamw8", lr=0.5)
    command.go_on_from(state, *new)
    assert new[1].param_groups[0]["lr"] == 0.5 and int(new[1].state[new[0].embed]["step"]) == 1
    with pytest.raises(SystemExit, match="8 bits"):
        command.go_on_from(state, *_training("adamw"))


def _gated_rank(rank, world, port, out):
    import datetime

    import torch
    import torch.distributed as dist

    torch.set_num_threads(2)
    dist.init_process_group("gloo", init_method=f"tcp://127.0.0.1:{port}", rank=rank, world_size=world, timeout=datetime.timedelta(seconds=120))
    import dataclasses

    from fuselink_b200.models.moe import Gate
    from fuselink_b200.models.moe_transformer import MOE_ZOO, MoETransformer
    from fuselink_b200.ops.adamw import AdamW
    cfg = dataclasses.replace(MOE_ZOO["tiny_moe"], embed_scale=2.0, gate=Gate(groups=2, topk_groups=1, balance_bias=True), balance_rate=0.25)
    net = MoETransformer(cfg, 2 * 8, None, rank, world, device="cpu", seed=3)
    opt = AdamW(net.parameters(), lr=1e-2, state_bits=8, master=True)
    loads = []
    for k in range(3):
        tokens = torch.randint(0, cfg.vocab, (2, 8), generator=torch.Generator().manual_seed(10 * k + rank))
        old = net.token_logprobs(tokens)
        net.policy_step(tokens, old, torch.ones(2, 1) * (1 - 2 * rank), opt)
        loads.append([b.moe.last_load.clone() for b in net.blocks])
    state = {n: [opt.state[p][n] for p in net.dense_parameters()] for n in ("exp_avg", "root_avg_sq", "master")}
    torch.save({"loads": loads, "bias": [b.moe.balance_bias for b in net.blocks], "dense": [p.detach() for p in net.dense_parameters()], "state": state}, f"{out}.{rank}")
    dist.barrier()
    dist.destroy_process_group()


def test_gates_and_policy_steps_on_two_ranks(tmp_path):
    """Replicated parameters, their 8-bit moments and fp32 copies, and the balance biases are equal on both ranks; the biases moved by the loads of both."""
    import socket

    import torch
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    torch.multiprocessing.spawn(_gated_rank, args=(2, port, str(tmp_path / "out")), nprocs=2)
    a, b = (torch.load(tmp_path / f"out.{r}") for r in (0, 1))
    for x, y in zip(a["dense"], b["dense"]):
        assert torch.equal(x, y)
    for name in a["state"]:
        for x, y in zip(a["state"][name], b["state"][name]):
            assert (x is None and y is None) or torch.equal(x.float(), y.float()), name
    assert any(not torch.equal(x, y) for k in range(3) for x, y in zip(a["loads"][k], b["loads"][k]))
    for layer, bias in enumerate(a["bias"]):
        want = torch.zeros_like(bias)
        for k in range(3):
            load = (a["loads"][k][layer] + b["loads"][k][layer]).float()
            want += 0.25 * (load.mean() - load).sign()
        assert torch.equal(bias, want) and torch.equal(bias, b["bias"][layer]) and bias.any()
