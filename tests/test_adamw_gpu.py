"""AdamW over many tensors (csrc/kernels/adamw.cu) against the same step on the CPU, whose moments and codes it has bit by bit."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DT = [torch.bfloat16, torch.float16, torch.float32]
HOW = dict(lr=1e-2, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)


def _tensors(shapes, dt, bits, master, seed=1, step=3):
    from fuselink_b200.ops import adamw
    g = torch.Generator().manual_seed(seed)
    s = dict(params=[], grads=[], m=[], v=[], steps=[], m_scale=[], v_scale=[], master=[])
    for i, shape in enumerate(shapes):
        w, grad = 0.1 * torch.randn(shape, generator=g), 10.0 ** (i % 5 - 4) * torch.randn(shape, generator=g) * torch.exp(2 * torch.randn(shape, generator=g))
        m, root = 0.3 * grad * torch.randn(shape, generator=g), grad.abs() * torch.rand(shape, generator=g)
        s["params"].append(w.to(dt)), s["grads"].append(grad.to(dt)), s["steps"].append(torch.tensor(step + i % 3))
        if bits == 8:
            for name, x in (("m", m), ("v", root)):
                codes, scale = adamw.encode(x, root=name == "v")
                s[name].append(codes), s[name + "_scale"].append(scale)
        else:
            s["m"].append(m), s["v"].append(root * root)
        if master:
            s["master"].append(w + 1e-4 * torch.randn(shape, generator=g))
    return s


def _to_gpu(s):
    return {k: [t.cuda() for t in v] for k, v in s.items()}


def _step(s, **how):
    from fuselink_b200.ops import adamw
    adamw.step(s["params"], s["grads"], s["m"], s["v"], s["steps"], scales=(s["m_scale"], s["v_scale"]) if s["m_scale"] else None, master=s["master"] or None, **{**HOW, **how})


def _same_bits(a, b):
    kinds = {torch.float32: torch.int32, torch.float8_e4m3fn: torch.uint8, torch.int64: torch.int64}
    return torch.equal(a.cpu().contiguous().view(kinds[a.dtype]) if a.dim() else a.cpu(), b.contiguous().view(kinds[b.dtype]) if b.dim() else b)


def _check(got, want, before, lr=HOW["lr"]):
    for name in ("m", "v", "m_scale", "v_scale"):
        for a, b in zip(got[name], want[name]):
            nan = b.float().isnan()
            assert torch.equal(a.cpu().float().isnan(), nan) and (_same_bits(a, b) or torch.equal(a.cpu().float()[~nan], b.float()[~nan])), name
    assert [int(t) for t in got["steps"]] == [int(t) for t in want["steps"]]
    for name in ("params", "master"):
        for a, b, w in zip(got[name], want[name], before[name]):
            moved = (b.double() - w.double()).abs() + 0.2 * lr * w.double().abs()
            # a root, a factor, a sum, a quotient of 2 units and two more products; then the weight's own rounding on either side
            tol = 16 * 2.0 ** -24 * moved + 2 * 2.0 ** -24 * w.double().abs() + torch.finfo(a.dtype).eps * b.double().abs() + torch.finfo(a.dtype).tiny
            far = (a.cpu().double() - b.double()).abs() <= tol
            assert torch.equal(a.cpu().isnan(), b.isnan()) and (far | b.isnan() | (a.cpu() == b)).all(), name


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("master", [False, True])
def test_step(dt, bits, master):
    if master and dt == torch.float32:
        return
    shapes = [(1,), (3, 5), (256,), (257,), (0, 4), (128, 128), (8191,), (8192,), (8193,), (3, 7, 1001), (70000,), ()]
    want = _tensors(shapes, dt, bits, master)
    got, before = _to_gpu(want), {k: [t.clone() for t in v] for k, v in want.items()}
    for k in range(3):
        _step(got), _step(want)
        _check(got, want, before)
        before = {k: [t.clone() for t in v] for k, v in want.items()}
        for name in ("params", "master"):                              # the two sides may round otherwise: go on from one of them
            for a, b in zip(got[name], want[name]):
                a.copy_(b)


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("count", [32, 33, 400, 401, 1003])
def test_many_tensors(count, bits):
    want = _tensors([(1 + 37 * i % 611,) for i in range(count)], torch.bfloat16, bits, False)
    got, before = _to_gpu(want), {k: [t.clone() for t in v] for k, v in want.items()}
    _step(got), _step(want)
    _check(got, want, before)


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("master", [False, True])
def test_tensors_anywhere_in_memory_and_laid_out_otherwise(master, bits):
    """Views at odd places, a transposed matrix, channels last, gradients with strides of their own and one value for all."""
    want = _tensors([(1000,), (40, 30), (2, 3, 4, 5), (600,), (700,)], torch.bfloat16, bits, master)
    got = _to_gpu(want)

    def at_odd_place(t):
        room = torch.empty(t.numel() + 3, dtype=t.dtype, device="cuda")
        return room[1: 1 + t.numel()].copy_(t)

    for name in ("params", "grads", "m", "v", "master"):
        if got[name]:
            for i in (0, 3):
                got[name][i] = at_odd_place(got[name][i])
            for side in (got, want):
                old = side[name][1]
                side[name][1] = torch.empty(30, 40, dtype=old.dtype, device=old.device).t().copy_(old)
                old = side[name][2]
                side[name][2] = torch.empty(2, 4, 5, 3, dtype=old.dtype, device=old.device).permute(0, 3, 1, 2).copy_(old)
    for side in (got, want):
        side["grads"][1] = side["grads"][1].contiguous()
        side["grads"][4] = torch.full((), 0.01, dtype=torch.bfloat16, device=side["grads"][4].device).expand(700)
    before = {k: [t.clone() for t in v] for k, v in want.items()}
    _step(got), _step(want)
    _check(got, want, before)


@pytest.mark.parametrize("bits", [8, 32])
def test_values_that_are_not_ordinary(bits):
    want = _tensors([(512,), (512,), (300,), (512,)], torch.float32, bits, False)
    g = want["grads"]
    g[0][3], g[0][300], g[1][:256] = math.nan, math.inf, 0.0
    g[2][:] = 1e-30                                                    # squares that are 0, roots that vanish
    g[3][:] = 1e19
    g[3][7] = 1e-25
    for name in ("m", "v"):
        want[name][1] = torch.zeros_like(want[name][1])
    got, before = _to_gpu(want), {k: [t.clone() for t in v] for k, v in want.items()}
    for _ in range(2):
        _step(got), _step(want)
    for name in ("m", "v", "m_scale", "v_scale"):
        for a, b in zip(got[name], want[name]):
            nan = b.float().isnan()
            assert torch.equal(a.cpu().float().isnan(), nan) and torch.equal(a.cpu().float()[~nan], b.float()[~nan]), name
    assert got["params"][0].isnan().sum() == 2 and (got["params"][1][:256].cpu() - before["params"][1][:256] * (1 - 1e-3) ** 2).abs().max() <= 2.0 ** -23
    if bits == 8:
        assert (got["v"][3].float()[:256] > 0).all()                   # small beside the others, and not lost


def test_learning_rate_on_the_device_captured_steps_and_settings():
    want = _tensors([(500,), (9000,)], torch.float32, 8, False, step=0)
    got = _to_gpu(want)
    lr = torch.tensor(1e-2, device="cuda")
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        _step(got, lr=lr, betas=(0.0, 0.999), eps=1e-6, weight_decay=0.0)
    for k in range(3):
        lr.fill_(1e-2 / (k + 1))
        before = {k: [t.clone() for t in v] for k, v in want.items()}
        graph.replay()
        _step(want, lr=1e-2 / (k + 1), betas=(0.0, 0.999), eps=1e-6, weight_decay=0.0)
        torch.cuda.synchronize()
        _check(got, want, before)
    assert [int(t) for t in got["steps"]] == [3, 4]


def test_parameters_count_as_changed():
    s = _to_gpu(_tensors([(64,)], torch.float32, 32, False))
    p = s["params"][0].requires_grad_(True)
    out = (p * p).sum()
    _step(s)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.backward()


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("dt", DT)
def test_optimizer(dt, bits):
    """The class on the GPU and on the CPU: parameters without a gradient, two groups, a state that is saved and loaded."""
    from fuselink_b200.ops.adamw import AdamW
    master = dt != torch.float32
    nets = []
    for device in ("cpu", "cuda"):
        g = torch.Generator().manual_seed(3)
        ps = [torch.nn.Parameter((0.1 * torch.randn(s, generator=g)).to(dt).to(device)) for s in ((300, 7), (11,), (2000,))]
        nets.append((ps, AdamW([dict(params=ps[:2], weight_decay=0.0), dict(params=ps[2:], lr=1e-3)], lr=1e-2, state_bits=bits, master=master)))
    for k in range(4):
        g = torch.Generator().manual_seed(10 + k)
        grads = [torch.randn(s, generator=g) for s in ((300, 7), (11,), (2000,))]
        if k == 2:                                                     # goes on from what was saved
            for i, (ps, opt) in enumerate(nets):
                new = AdamW([dict(params=ps[:2]), dict(params=ps[2:])], state_bits=bits, master=master)
                new.load_state_dict(opt.state_dict())
                nets[i] = (ps, new)
        for ps, opt in nets:
            for p, x in zip(ps, grads):
                p.grad = x.to(dt).to(p.device)
            if k == 1:
                ps[1].grad = None
            opt.step()
    for a, b in zip(nets[0][0], nets[1][0]):
        sa, sb = nets[0][1].state[a], nets[1][1].state[b]
        assert sa.keys() == sb.keys() and int(sa["step"]) == int(sb["step"]) == (3 if a.numel() == 11 else 4)
        for name in sa:
            assert sa[name].dtype == sb[name].dtype and sb[name].is_cuda
            if name not in ("step", "master"):
                assert torch.equal(sa[name].float(), sb[name].float().cpu())
        # four steps, each of them a rounding of the weight (of its fp32 copy, where there is one) on either side
        assert ((a.double() - b.double().cpu()).abs() <= 8 * (2.0 ** -24 if not master else 2.0 ** -24) * (1 + a.double().abs()) + torch.finfo(dt).eps * a.double().abs()).all()


def test_what_is_refused():
    from fuselink_b200.ops import adamw
    ok = lambda **how: _to_gpu(_tensors([(64,), (20, 5)], how.pop("dt", torch.bfloat16), how.pop("bits", 32), how.pop("master", False)))  # noqa: E731

    def bad(s, name, i, t, error=RuntimeError, **how):
        s[name][i] = t
        with pytest.raises(error):
            _step(s, **how)

    f = torch.zeros(64, device="cuda")
    bad(ok(), "grads", 0, f)
    bad(ok(), "grads", 0, f[:5].bfloat16())
    bad(ok(), "grads", 0, f.bfloat16().cpu())
    bad(ok(), "grads", 0, f.bfloat16().to_sparse())
    bad(ok(), "m", 0, f.double())
    bad(ok(), "v", 1, torch.zeros(5, 20, device="cuda").t())
    bad(ok(), "steps", 0, torch.zeros((), device="cuda"))
    bad(ok(), "params", 1, torch.zeros(40, 5, device="cuda", dtype=torch.bfloat16)[::2])
    bad(ok(bits=8), "m_scale", 0, torch.zeros(2, device="cuda"))
    bad(ok(master=True), "master", 0, f.bfloat16())
    s = ok()
    bad(s, "params", 1, s["params"][0])
    s = ok()
    bad(s, "steps", 1, s["steps"][0])
    s = ok(dt=torch.float32)
    s["master"] = [t.clone() for t in s["params"]]
    with pytest.raises(RuntimeError):
        _step(s)
    for how in (dict(lr=-1.0), dict(lr=math.nan), dict(betas=(1.0, 0.9)), dict(eps=-1.0), dict(weight_decay=math.inf)):
        with pytest.raises(ValueError):
            _step(ok(), **how)
    with pytest.raises(RuntimeError):
        _step(ok(), lr=torch.tensor(1e-3))
    s = ok()
    with pytest.raises(RuntimeError):
        adamw.step(s["params"], s["grads"][:1], s["m"], s["v"], s["steps"], lr=1e-3)
    with pytest.raises(ValueError):
        adamw.AdamW([torch.nn.Parameter(f)], state_bits=4)
    p = torch.nn.Parameter(f.clone())
    p.grad = torch.zeros_like(p)
    opt = adamw.AdamW([p])
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()
    adamw.step([], [], [], [], [], lr=1e-3)
