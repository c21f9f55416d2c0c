"""Operators around the expert layers of a training step, one at a time: what a program has them do, and their plain forms.

  embed     embedding.lookup: rows of the embedding times a factor, and on request the table's gradient
  route     routing.route: experts, weights and loads from the router's logits, and on request the logits' gradient
  logprobs  losses.token_logprobs: logarithms of given tokens' probabilities, and on request the logits' gradient
  policy    losses.policy_loss: the clipped policy loss with a KL term, its figures and the logits' gradient
  adamw     adamw.step: one step over many tensors, states in 32 bits or in 8

A case says sizes, types and settings; what follows from them (ragged lengths, shapes of the tensors) is computed here, so that work()
knows it.  States in 8 bits are e4m3 codes with a scale per 256 values of a tensor: the smallest power of two, 2^-100 at least, that
keeps their largest finite magnitude within 448; of the second moment the square root is kept, and a root above 0 is no code of 0.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
F8 = torch.float8_e4m3fn
LEAST = 2.0 ** -100
BLOCK = 256
CLIP = 448.0


def listed():
    return [
        # One decoding step of a batch: the launch is what it costs.
        dict(name="embed 16 new tokens", kind="embed", tokens=16, vocab=32000, hidden=4096, dtype="bf16", scale=64.0, pad=0.0, train=False),
        # A training step of the transformer's default size, 4 sequences of 2048.
        dict(name="embed 4x2048", kind="embed", tokens=8192, vocab=32000, hidden=4096, dtype="bf16", scale=1.0, pad=0.0, train=True),
        # Short sequences in full precision, a vocabulary and rows of odd sizes, a third of the tokens padding.
        dict(name="embed 7x389 padded", kind="embed", tokens=2723, vocab=50257, hidden=1600, dtype="fp32", scale=40.0, pad=0.33, train=True),
        # A decoding step's routing over many small experts in groups: latency.
        dict(name="route 16 of 256", kind="route", tokens=16, experts=256, topk=8, score="sigmoid", bias=True, groups=8, topk_groups=4, dtype="bf16", balance=False, train=False),
        # A training step's routing by softmax, without groups, with the balance term.
        dict(name="route 8192 of 64", kind="route", tokens=8192, experts=64, topk=6, score="softmax", bias=False, groups=1, topk_groups=1, dtype="bf16", balance=True, train=True),
        # A large batch over many experts, chosen with the balance bias within groups; logits in full precision.
        dict(name="route 65536 of 256", kind="route", tokens=65536, experts=256, topk=8, score="sigmoid", bias=True, groups=8, topk_groups=4, dtype="fp32", balance=True, train=True),
        # What an earlier policy made of four answers of 97 tokens; a vocabulary of odd size, so that rows start anywhere.
        dict(name="logprobs 4x97 of 50257", kind="logprobs", batch=4, length=97, vocab=50257, dtype="fp16", temperature=0.7, shifted=False, train=False),
        # A training step on 8 answers of up to 1024 tokens with a reference policy; the logits are a model's without the last position.
        dict(name="policy 8x1024 of 32000", kind="policy", batch=8, length=1024, vocab=32000, dtype="bf16", temperature=1.0, shifted=True, reference=True, high=0.2),
        # Three long answers over a large vocabulary, no reference, an upper border of its own.
        dict(name="policy 3x1365 of 128256", kind="policy", batch=3, length=1365, vocab=128256, dtype="bf16", temperature=1.0, shifted=False, reference=False, high=0.28),
        # All of a model so small that its step is launches: 20 tensors, states in 32 bits.
        dict(name="adamw 20 small tensors", kind="adamw", layers=2, hidden=128, kv=128, ffn=256, vocab=512, dtype="fp32", bits=32, master=False),
        # The replicated and expert weights of a few layers with fp32 copies of the bf16 weights, as training in earnest keeps them.
        dict(name="adamw 2 layers, 32 bits", kind="adamw", layers=2, hidden=4096, kv=1024, ffn=14336, vocab=32000, dtype="bf16", bits=32, master=True),
        # Many layers of odd sizes with states in 8 bits.
        dict(name="adamw 12 layers, 8 bits", kind="adamw", layers=12, hidden=1600, kv=1600, ffn=6400, vocab=50257, dtype="bf16", bits=8, master=False),
    ]


def _log(rng, a, b):
    return max(a, min(b, int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))))


def draw(rng):
    kind, dtype = rng.choice(["embed", "route", "logprobs", "policy", "adamw"]), rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind == "embed":
        vocab = rng.choice([512, 32000, 50257, 50272, 128256, _log(rng, 100, 128256)])
        hidden = rng.choice([4096, 1600, _log(rng, 16, 1024) * 8, _log(rng, 33, 4096)])
        tokens = max(1, min(_log(rng, 1, 65536), 500_000_000 // hidden))
        vocab = max(100, min(vocab, 600_000_000 // hidden))
        return dict(kind=kind, tokens=tokens, vocab=vocab, hidden=hidden, dtype=dtype, scale=rng.choice([1.0, math.sqrt(hidden)]), pad=rng.choice([0.0, 0.0, 0.2, 0.6]), train=rng.random() < 0.7)
    if kind == "route":
        experts, groups = rng.choice([(8, 1), (60, 1), (64, 1), (64, 8), (96, 4), (128, 1), (160, 8), (256, 8), (256, 1), (384, 1), (_log(rng, 4, 512), 1)])
        topk_groups = rng.randint((groups + 1) // 2, groups)
        topk = rng.randint(1, min(8, experts))
        return dict(kind=kind, tokens=_log(rng, 1, 65536), experts=experts, topk=topk, score=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.5,
                    groups=groups, topk_groups=topk_groups, dtype=dtype, balance=rng.random() < 0.6, train=rng.random() < 0.7)
    if kind in ("logprobs", "policy"):
        vocab = rng.choice([1000, 32000, 50257, 50272, 128256, _log(rng, 50, 128256)])
        batch = _log(rng, 1, 16)
        length = max(1, min(_log(rng, 1, 8192), 500_000_000 // (vocab * batch)))
        c = dict(kind=kind, batch=batch, length=length, vocab=vocab, dtype=dtype, temperature=rng.choice([1.0, 1.0, 0.7]), shifted=rng.random() < 0.5)
        return dict(c, train=rng.random() < 0.5) if kind == "logprobs" else dict(c, reference=rng.random() < 0.5, high=rng.choice([0.2, 0.28]))
    hidden = rng.choice([_log(rng, 16, 4096), _log(rng, 4, 512) * 8])
    ffn = rng.choice([4 * hidden, hidden * 7 // 2])
    layer = 2 * hidden * hidden + 3 * hidden * ffn
    layers = max(1, min(_log(rng, 1, 48), 400_000_000 // layer))
    vocab = max(50, min(rng.choice([512, 32000, 50257]), (450_000_000 - layers * layer) // hidden))
    bits = rng.choice([32, 8])
    return dict(kind=kind, layers=layers, hidden=hidden, kv=max(1, hidden // rng.choice([1, 4])), ffn=ffn, vocab=vocab, dtype=dtype, bits=bits,
                master=dtype != "fp32" and rng.random() < 0.5)


# ---- what follows from a case ---------------------------------------------------------------------------------------------------
def _span(tokens, vocab):
    """How many words up to the n-th one take a share of ids drawn as 1 / (rank + 10)."""
    return math.log(vocab / 10 + 1)


def _distinct(c):
    """Expected number of distinct ids."""
    v = np.arange(c["vocab"], dtype=np.float64)
    p = np.log((v + 11) / (v + 10)) / _span(c["tokens"], c["vocab"])
    live = c["tokens"] - int(c["tokens"] * c["pad"])
    return float(np.sum(-np.expm1(live * np.log1p(-np.minimum(p, 1 - 1e-9))))) + (1 if c["pad"] else 0)


def _lengths(c):
    """Answers' lengths, from half of the longest to it, the longest among them."""
    B, L = c["batch"], c["length"]
    return [L if b == B // 2 else L - int((L // 2) * math.modf((b + 0.5) * 0.6180339887498949)[0]) for b in range(B)]


def _counted(c):
    """Rows of the logits that carry a weight, of all."""
    return (sum(_lengths(c)) if c["kind"] == "policy" else c["batch"] * c["length"]), c["batch"] * c["length"]


def _shapes(c):
    """The tensors of a model: per layer the attention's and the feed-forward part's weights and norms, then embedding, head and last norm."""
    h, f, kv = c["hidden"], c["ffn"], c["kv"]
    each = [(h + 2 * kv, h), (h, h), (2 * f, h), (h, f), (h,), (h,), (h + 2 * kv,), (f,)]
    return each * c["layers"] + [(c["vocab"], h), (c["vocab"], h), (h,), (c["vocab"],)]


def _numel(c):
    return [math.prod(s) for s in _shapes(c)]


# ---- inputs -----------------------------------------------------------------------------------------------------------------
def _scale_of(amax):
    """The smallest power of two, 2^-100 at least, that brings amax within 448."""
    m, e = torch.frexp(amax)                               # amax = m 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.where(m <= 0.875, e - 9, e - 8)
    return torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), e), torch.zeros_like(amax)).clamp(min=LEAST)


def _ids(gen, shape, vocab):
    """Tokens as texts have them: a few words often, most seldom, frequent ones anywhere in the vocabulary."""
    u = torch.rand(shape, generator=gen, device=DEV, dtype=torch.float64)
    rank = (10 * torch.expm1(u * math.log(vocab / 10 + 1))).long().clamp(max=vocab - 1)
    return torch.randperm(vocab, generator=gen, device=DEV)[rank]


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device=DEV).manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=DEV)

    if c["kind"] == "embed":
        dt, T, V, H = DTYPES[c["dtype"]], c["tokens"], c["vocab"], c["hidden"]
        ids = _ids(gen, (T,), V)
        if c["pad"]:
            ids[T - int(T * c["pad"]):] = 0                                # the padding token behind the texts
        s = dict(c, table=(0.02 * randn(V, H)).to(dt), ids=ids)
        if c["train"]:
            s["table"].requires_grad_(True)
            s["dout"] = (randn(T, H) * torch.exp(randn(T, 1))).to(dt)
        return s
    if c["kind"] == "route":
        T, E = c["tokens"], c["experts"]
        logits = 1.5 * randn(T, E) + 0.7 * randn(E)                        # some experts are liked by all tokens
        s = dict(c, logits=logits.to(DTYPES[c["dtype"]]), bias_row=0.05 * randn(E) if c["bias"] else None)
        if c["train"]:
            s["logits"].requires_grad_(True)
            s["dw"], s["dbalance"] = randn(T, c["topk"]), torch.full((), 0.01, device=DEV)
        return s
    if c["kind"] in ("logprobs", "policy"):
        B, L, V = c["batch"], c["length"], c["vocab"]
        full = torch.empty(B, L + c["shifted"], V, dtype=DTYPES[c["dtype"]], device=DEV)
        for b in range(B):
            x = 2.0 * randn(L + c["shifted"], V)
            x.scatter_add_(1, torch.randint(0, V, (L + c["shifted"], 24), generator=gen, device=DEV), 6.0 + 2.5 * randn(L + c["shifted"], 24))
            full[b] = x
        logits = full[:, :L]
        # tokens that such a model would have drawn
        tokens = torch.empty(B, L, dtype=torch.int64, device=DEV)
        lp = torch.empty(B, L, device=DEV)
        for b in range(B):
            p = torch.log_softmax(logits[b].float() / c["temperature"], -1)
            gumbel = -torch.log(-torch.log(torch.rand(L, V, generator=gen, device=DEV).clamp(1e-7, 1 - 1e-7)))
            tokens[b] = (p + gumbel).argmax(-1)
            lp[b] = p.gather(1, tokens[b][:, None])[:, 0]
        s = dict(c, logits=logits, tokens=tokens)
        if c["kind"] == "logprobs":
            if c["train"]:
                s["logits"].requires_grad_(True)
                s["dlogprobs"] = randn(B, L)
            return s
        drift = 0.15 * randn(B, L)
        for border in (math.log(0.8), math.log(1 + c["high"])):            # none so near a border that a rounding decides
            drift = torch.where((drift - border).abs() < 1e-3, drift + 0.01, drift)
        s["logits"].requires_grad_(True)
        s["old"] = lp - drift
        s["advantages"] = randn(B, 1).expand(B, L) + 0.1 * randn(B, L)
        s["weights"] = (torch.arange(L, device=DEV) < torch.tensor(_lengths(c), device=DEV)[:, None]).float()
        s["ref"] = lp + 0.3 * randn(B, L) if c["reference"] else None
        s["kl"] = 0.05 if c["reference"] else 0.0
        return s
    dt, sizes = DTYPES[c["dtype"]], _numel(c)
    starts = np.concatenate([[0], np.cumsum([-(-n // BLOCK) * BLOCK for n in sizes])])
    total = int(starts[-1])
    used = torch.zeros(total, dtype=torch.bool, device=DEV)                # tensors start at multiples of 256 values; zeros in between
    spread = torch.empty(total, device=DEV)
    for a, n in zip(starts, sizes):
        used[a: a + n] = True
        spread[a: a + n] = 10.0 ** (-4.5 + math.modf(a * 0.6180339887498949)[0] * 2)
    w = torch.where(used, 0.02 * randn(total), 0.0)
    noise = torch.where(used, spread * torch.exp(0.5 * randn(total)), 0.0)  # a gradient's size, weight by weight
    g, m = noise * randn(total), 0.3 * noise * randn(total)
    s = dict(c, w=w.to(dt), g=g.to(dt), steps=torch.arange(len(sizes), device=DEV) % 3 + 99, lr=3e-4, betas=(0.9, 0.95), eps=1e-8, decay=0.1)
    root = noise * (0.5 + torch.rand(total, generator=gen, device=DEV))
    if c["bits"] == 32:
        s["m"], s["v"] = m, root * root
    else:
        for name, x in (("m", m), ("v", root)):
            scale = _scale_of(x.view(-1, BLOCK).abs().amax(1))
            codes = (x.view(-1, BLOCK) / scale[:, None]).to(F8).view(-1)
            if name == "v":
                codes = torch.where((x > 0) & (codes.view(torch.uint8) == 0), torch.ones_like(codes.view(torch.uint8)), codes.view(torch.uint8)).view(F8)
            s[name], s[name + "_scale"] = codes, scale
    if c["master"]:
        s["master"] = w
    shapes = _shapes(c)

    def tensors(name):
        return [s[name][a: a + n].view(shape) for a, n, shape in zip(starts, sizes, shapes)]

    def scales(name):
        return [s[name + "_scale"][a // BLOCK: -(-(a + n) // BLOCK)] for a, n in zip(starts, sizes)]

    s["lists"] = dict(params=tensors("w"), grads=tensors("g"), m=tensors("m"), v=tensors("v"), steps=list(s["steps"].unbind()),
                      scales=(scales("m"), scales("v")) if c["bits"] == 8 else None, master=tensors("master") if c["master"] else None)
    s["each"] = torch.repeat_interleave(torch.arange(len(sizes), device=DEV), torch.tensor(np.diff(starts) // BLOCK, device=DEV))
    return s


# ---- plain forms --------------------------------------------------------------------------------------------------------------
def _plain_embed(s):
    table, ids = s["table"], s["ids"]
    out = (table.float()[ids] * s["scale"]).to(table.dtype)
    if not s["train"]:
        return out
    wide = torch.float64 if table.dtype == torch.float32 else torch.float32          # the padding token's sum is long
    grad = torch.zeros(table.shape, dtype=wide, device=DEV).index_add_(0, ids, s["dout"].to(wide))
    return out, (grad * s["scale"]).to(table.dtype)


def _plain_route(s):
    """In 64 bits: which expert is chosen lies between values next to one another."""
    T, E, k, G = s["tokens"], s["experts"], s["topk"], s["groups"]
    x = s["logits"].double()
    p = torch.exp(x - x.amax(1, keepdim=True)) if s["score"] == "softmax" else 1 / (1 + torch.exp(-x))
    if s["score"] == "softmax":
        p = p / p.sum(1, keepdim=True)
    c = p if s["bias_row"] is None else p + s["bias_row"].double()
    left = torch.ones(T, E, dtype=torch.bool, device=DEV)
    if G > 1:
        value = torch.sort(c.view(T, G, E // G), dim=2, descending=True)[0][:, :, :2].sum(2)
        best = torch.sort(value, dim=1, descending=True, stable=True)[1][:, : s["topk_groups"]]
        left = torch.zeros(T, G, dtype=torch.bool, device=DEV).scatter_(1, best, True).repeat_interleave(E // G, 1)
    order = x if s["bias_row"] is None else c                              # without a bias the order is the logits'
    idx = torch.sort(torch.where(left, order, -math.inf), dim=1, descending=True, stable=True)[1][:, :k]
    chosen = p.gather(1, idx)
    w = chosen / chosen.sum(1, keepdim=True)
    load = torch.zeros(E, dtype=torch.int64, device=DEV).index_add_(0, idx.reshape(-1), torch.ones(T * k, dtype=torch.int64, device=DEV))
    share = p / p.sum(1, keepdim=True)
    balance = (load * share.mean(0)).sum() * (E / (T * k))
    said = [2.5 * w.float(), idx.int(), load.int()] if not s["balance"] else [2.5 * w.float(), idx.int(), load.int(), balance.float()]
    if not s["train"]:
        return said
    dw = 2.5 * s["dw"].double()
    dp = torch.zeros_like(p).scatter_(1, idx, (dw - (dw * w).sum(1, keepdim=True)) / chosen.sum(1, keepdim=True))
    if s["balance"]:
        a = s["dbalance"].double() * load * (E / (T * T * k))
        dp = dp + (a - (a * share).sum(1, keepdim=True)) / p.sum(1, keepdim=True)
    dx = p * (dp - (p * dp).sum(1, keepdim=True)) if s["score"] == "softmax" else dp * p * (1 - p)
    return said + [dx.to(s["logits"].dtype)]


def _plain_rows(s):
    """Probabilities of all tokens, and the logarithm of the given one's."""
    x = s["logits"].float() / s["temperature"]
    x = x - x.amax(-1, keepdim=True)
    e = torch.exp(x)
    z = e.sum(-1, keepdim=True)
    lp = x.gather(-1, s["tokens"][..., None])[..., 0].double() - torch.log(z[..., 0].double())
    return e.div_(z), lp


def _plain_back(s, p, g):
    d = p.mul_(-(g / s["temperature"]).float()[..., None])
    return d.scatter_add_(-1, s["tokens"][..., None], (g / s["temperature"]).float()[..., None]).to(s["logits"].dtype)


def _plain_logprobs(s):
    p, lp = _plain_rows(s)
    return (lp.float(), _plain_back(s, p, s["dlogprobs"])) if s["train"] else lp.float()


def _plain_policy(s):
    p, lp = _plain_rows(s)
    w = s["weights"].double() / s["weights"].double().sum()
    r, A = torch.exp(lp - s["old"].double()), s["advantages"].double()
    free, held = r * A, r.clamp(0.8, 1 + s["high"]) * A
    loss, g = -torch.minimum(free, held), torch.where(free <= held, -r * A, 0.0)
    kl = torch.zeros_like(lp)
    if s["ref"] is not None:
        d = s["ref"].double() - lp
        kl = torch.exp(d) - d - 1
        g = g + s["kl"] * (1 - torch.exp(d))
    loss = (w * (loss + s["kl"] * kl)).sum()
    lp = torch.where(s["weights"] > 0, lp, 0.0)
    return loss.float(), lp.float(), (w * kl).sum().float(), (w * (free > held)).sum().float(), _plain_back(s, p, g * w)


def _plain_adamw(s):
    (b1, b2), lr = s["betas"], s["lr"]
    s["steps"] += 1
    t = s["steps"].double()[s["each"]][:, None]
    first, second = (lr / (1 - b1 ** t)).float(), (1 / torch.sqrt(1 - b2 ** t)).float()
    g = s["g"].float().view(-1, BLOCK)
    if s["bits"] == 32:
        m, v = s["m"].view(-1, BLOCK), s["v"].view(-1, BLOCK)
    else:
        m = s["m"].float().view(-1, BLOCK) * s["m_scale"][:, None]
        v = s["v"].float().view(-1, BLOCK) * s["v_scale"][:, None]
        v = v * v
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * g) * (1 - b2)
    root = torch.sqrt(v)
    w = (s["master"] if s["master"] is not False else s["w"].float()).view(-1, BLOCK)
    w = w * (1 - lr * s["decay"]) - first * (m / (root * second + s["eps"]))
    s["w"].copy_(w.view(-1))
    if s["master"] is not False:
        s["master"].copy_(w.view(-1))
    if s["bits"] == 32:
        s["m"].copy_(m.view(-1))
        s["v"].copy_(v.view(-1))
    else:
        ms, vs = _scale_of(m.abs().amax(1)), _scale_of(root.amax(1))
        s["m"].copy_((m / ms[:, None]).to(F8).view(-1))
        code = (root / vs[:, None]).to(F8).view(torch.uint8)
        s["v"].copy_(torch.where((root > 0) & (code == 0), torch.ones_like(code), code).view(F8).view(-1))
        s["m_scale"].copy_(ms)
        s["v_scale"].copy_(vs)
    return _said_adamw(s)


def _said_adamw(s):
    return {name: s[name] for name in ("w", "m", "v", "steps", "m_scale", "v_scale", "master") if s.get(name) is not None and s[name] is not False}


def run(state):
    s = state
    if not own:
        with torch.no_grad():
            return {"embed": _plain_embed, "route": _plain_route, "logprobs": _plain_logprobs, "policy": _plain_policy, "adamw": _plain_adamw}[s["kind"]](s)
    from fuselink_b200.ops import adamw, embedding, losses, routing

    if s["kind"] == "embed":
        out = embedding.lookup(s["table"], s["ids"], s["scale"])
        if not s["train"]:
            return out
        return out.detach(), torch.autograd.grad(out, s["table"], s["dout"])[0]
    if s["kind"] == "route":
        r = routing.route(s["logits"], s["topk"], score=s["score"], bias=s["bias_row"], groups=s["groups"], topk_groups=s["topk_groups"],
                          group_best=2, renormalize=True, scale=2.5, balance=s["balance"])
        said = [r.weights, r.experts, r.load] + ([r.balance] if s["balance"] else [])
        if not s["train"]:
            return said
        outs = [(r.weights, s["dw"])] + ([(r.balance, s["dbalance"])] if s["balance"] else [])
        return said + list(torch.autograd.grad([o for o, _ in outs], s["logits"], [d for _, d in outs]))
    if s["kind"] == "logprobs":
        lp = losses.token_logprobs(s["logits"], s["tokens"], temperature=s["temperature"])
        return (lp, torch.autograd.grad(lp, s["logits"], s["dlogprobs"])[0]) if s["train"] else lp
    if s["kind"] == "policy":
        r = losses.policy_loss(s["logits"], s["tokens"], s["old"], s["advantages"], weights=s["weights"], reference=s["ref"], kl=s["kl"],
                               clip=(0.2, s["high"]), temperature=s["temperature"])
        return r.loss, r.logprobs, r.divergence, r.clipped, torch.autograd.grad(r.loss, s["logits"])[0]
    a = s["lists"]
    adamw.step(a["params"], a["grads"], a["m"], a["v"], a["steps"], lr=s["lr"], betas=s["betas"], eps=s["eps"], weight_decay=s["decay"],
               scales=a["scales"], master=a["master"])
    return _said_adamw(s)


def work(case):
    c = case
    if c["kind"] == "embed":
        T, V, H, z = c["tokens"], c["vocab"], c["hidden"], SIZE[c["dtype"]]
        n = _distinct(c) * H * z + T * (8 + H * z)
        return dict(bytes=n + (T + V) * H * z if c["train"] else n, flops=T * H * (2 if c["train"] else 1))
    if c["kind"] == "route":
        T, E, k, z = c["tokens"], c["experts"], c["topk"], SIZE[c["dtype"]]
        return dict(bytes=T * (E * z + 8 * k) + 8 * E + (T * (E * z + 4 * k) if c["train"] else 0), flops=T * E * (20 if c["train"] else 8))
    if c["kind"] in ("logprobs", "policy"):
        some, rows = _counted(c)
        train = c["kind"] == "policy" or c["train"]
        each = 32 if c["kind"] == "policy" else 12 + 4 * train
        return dict(bytes=c["vocab"] * SIZE[c["dtype"]] * (some + train * rows) + each * rows, flops=some * c["vocab"] * (4 + 3 * train))
    z = SIZE[c["dtype"]]
    each = 3 * z + (16 if c["bits"] == 32 else 4 + 16 / BLOCK) + (8 - z if c["master"] else 0)
    return dict(bytes=sum(_numel(c)) * each, flops=sum(_numel(c)) * 14)


# ---- the same from the definitions, in 64 bits -----------------------------------------------------------------------------------
def _exact_embed(s):
    table, ids, T = s["table"].detach(), s["ids"], s["tokens"]
    out = torch.stack([table[:, h][ids].double() * s["scale"] for h in range(table.shape[1])], 1) if table.shape[1] < 64 else table.double()[ids] * s["scale"]
    if not s["train"]:
        return out
    order = torch.sort(ids, stable=True)[1]
    ends = torch.searchsorted(ids[order].contiguous(), torch.arange(table.shape[0], device=DEV), right=True)
    grad = torch.empty(table.shape, dtype=torch.float64, device=DEV)
    for a in range(0, table.shape[1], 256):                                # differences of running sums over the sorted tokens
        run_sum = torch.cat([torch.zeros_like(s["dout"][:1, a: a + 256], dtype=torch.float64), s["dout"][order, a: a + 256].double().cumsum(0)])
        upto = run_sum[ends]
        grad[:, a: a + 256] = torch.diff(upto, dim=0, prepend=torch.zeros_like(upto[:1])) * s["scale"]
        grad[:, a: a + 256][torch.diff(ends, prepend=torch.zeros_like(ends[:1])) == 0] = 0
    return out, grad


def _exact_route(s):
    """The weights, the term and the gradient, by automatic differentiation of the definition in 64 bits; the choice is whole numbers."""
    T, E, k, G = s["tokens"], s["experts"], s["topk"], s["groups"]
    x = s["logits"].detach().double().requires_grad_(True)
    p = torch.softmax(x, 1) if s["score"] == "softmax" else torch.sigmoid(x)
    with torch.no_grad():
        c = p.clone() if s["bias_row"] is None else p + s["bias_row"].double()
        if G > 1:
            value = torch.topk(c.view(T, G, E // G), 2, dim=2)[0].sum(2)
            kept = torch.topk(value, s["topk_groups"], dim=1)[1]
            out_of = torch.ones(T, G, dtype=torch.bool, device=DEV)
            out_of[torch.arange(T, device=DEV)[:, None], kept] = False
            c.view(T, G, E // G)[out_of] = -math.inf
        idx = torch.argsort(c, dim=1, descending=True, stable=True)[:, :k]
        load = torch.bincount(idx.reshape(-1), minlength=E)
    w = torch.take_along_dim(p, idx, 1)
    w = 2.5 * w / w.sum(1, keepdim=True)
    said = [w.detach(), None, None]
    total = 0.0
    if s["balance"]:
        balance = torch.dot(load.double() / (T * k), torch.nn.functional.normalize(p, p=1, dim=1).mean(0)) * E
        said.append(balance.detach())
        total = total + balance * 0.01
    if s["train"]:
        (total + (w * s["dw"].double()).sum()).backward()
        said.append(x.grad)
    return said


def _exact_rows(s):
    """Row by row: ln p of the given token, and a function that gives p - 1[token]."""
    x = s["logits"].detach()
    B, L, V = x.shape
    lp = torch.empty(B, L, dtype=torch.float64, device=DEV)
    for b in range(B):
        for a in range(0, L, 512):
            y = x[b, a: a + 512].double() / s["temperature"]
            lp[b, a: a + 512] = -torch.logsumexp(y - y.gather(1, s["tokens"][b, a: a + 512, None]), 1)
    return lp


def _exact_back(s, g):
    x = s["logits"].detach()
    out = torch.empty(x.shape, dtype=torch.float64, device=DEV)
    for b in range(x.shape[0]):
        for a in range(0, x.shape[1], 512):
            p = torch.softmax(x[b, a: a + 512].double() / s["temperature"], 1)
            p[torch.arange(p.shape[0], device=DEV), s["tokens"][b, a: a + 512]] -= 1
            out[b, a: a + 512] = -p * g[b, a: a + 512, None] / s["temperature"]
    return out


def _exact_logprobs(s):
    lp = _exact_rows(s)
    return (lp, _exact_back(s, s["dlogprobs"].double())) if s["train"] else lp


def _exact_policy(s):
    lp = _exact_rows(s).requires_grad_(True)
    on = s["weights"].double()
    A, r = s["advantages"].double(), torch.exp(lp - s["old"].double())
    border = torch.where(A > 0, torch.full_like(A, 1 + s["high"]), torch.full_like(A, 0.8))
    stopped = torch.where(A > 0, r > border, r < border)
    term = -A * torch.where(stopped, border, r)
    kl = torch.zeros_like(lp)
    if s["ref"] is not None:
        d = s["ref"].double() - lp
        kl = torch.expm1(d) - d
    mean = lambda t: (t * on).sum() / on.sum()  # noqa: E731
    loss = mean(term + s["kl"] * kl)
    loss.backward()
    return loss.detach(), lp.detach() * on, mean(kl.detach()), mean(stopped.double()), _exact_back(s, lp.grad)


def _exact_adamw(s):
    (b1, b2), lr = s["betas"], s["lr"]
    t = (s["steps"] + 1).double()[s["each"]]
    fix1, fix2 = (1 / (1 - b1 ** t)).repeat_interleave(BLOCK), (1 / (1 - b2 ** t)).repeat_interleave(BLOCK)
    said = {"steps": None}
    parts = {"w": [], "m": [], "v": []}
    for a in range(0, s["w"].numel(), 1 << 26):
        at = slice(a, a + (1 << 26))
        g = s["g"][at].double()
        m, v = s["m"][at].double(), s["v"][at].double()
        if s["bits"] == 8:
            blocks = slice(a // BLOCK, (a + g.numel()) // BLOCK)
            m = m * s["m_scale"][blocks].double().repeat_interleave(BLOCK)
            v = (v * s["v_scale"][blocks].double().repeat_interleave(BLOCK)) ** 2
        m += (1 - b1) * (g - m)
        v += (1 - b2) * (g * g - v)
        w = (s["master"] if s["master"] is not False else s["w"])[at].double()
        parts["w"].append(w - lr * (s["decay"] * w + m * fix1[at] / ((v * fix2[at]).sqrt() + s["eps"])))
        if s["bits"] == 8:
            for x, name in ((m, "m"), (v.sqrt(), "v")):
                y = x.view(-1, BLOCK)
                unit = torch.exp2(torch.ceil(torch.log2(y.abs().amax(1).clamp(min=1e-300) / CLIP))).clamp(min=LEAST)
                parts[name].append((y / unit[:, None]).reshape(-1))
        else:
            parts["m"].append(m)
            parts["v"].append(v)
    for name, values in parts.items():
        said[name] = torch.cat(values)
    if s["bits"] == 8:
        said.update(m_scale=None, v_scale=None)                            # powers of two, as the plain form has them
    if s["master"] is not False:
        said["master"] = said["w"]
    return said


def exact(case, seed):
    s = prepare(case, seed)
    return {"embed": _exact_embed, "route": _exact_route, "logprobs": _exact_logprobs, "policy": _exact_policy, "adamw": _exact_adamw}[case["kind"]](s)
