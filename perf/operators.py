"""Operators of decoding from a cache in 8 bits, one at a time: what a serving program has them do, and their plain forms.

  write    kv8.write: bias and rotation of new tokens' queries and keys; keys and values to 8-bit pages, a scale per page and head
  attend   kv8.attention: new tokens' attention over those pages, on request with the weight that every page got
  evict    kv8.evict: the pages of least weight make room
  sample   sampling.sample: the next tokens from given uniform numbers, temperature, top-k, top-p and min-p

A case says the layout (heads, KV heads, head size, page size), the type and the lengths; ragged lengths follow from these, so
that work() knows them.  A page's scale is the smallest power of two that keeps its largest finite magnitude within e4m3's 448.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
F8 = torch.float8_e4m3fn
LEAST = 2.0 ** -100


def listed():
    return [
        # One request of a small model in half precision: a few pages, where the launch is what a token costs.
        dict(name="attend 1x389", kind="attend", batch=1, heads=32, kv_heads=32, dim=64, page=16, length=389, ragged=False, new=1, mass=False, dtype="fp16"),
        # The serving benchmark's decoding batch: 16 requests of 2048 tokens, four query heads per KV head.
        dict(name="attend 16x2048", kind="attend", batch=16, heads=32, kv_heads=8, dim=128, page=16, length=2048, ragged=False, new=1, mass=False, dtype="bf16"),
        # A large ragged batch whose pages are weighed for eviction; eight query heads per KV head.
        dict(name="attend 48 ragged, weighed", kind="attend", batch=48, heads=64, kv_heads=8, dim=128, page=16, length=4099, ragged=True, new=1, mass=True, dtype="bf16"),
        # Four new tokens per request (a guess being verified), no shared heads, an odd head size, pages of 32.
        dict(name="attend 7x4 of 1531", kind="attend", batch=7, heads=32, kv_heads=32, dim=80, page=32, length=1531, ragged=True, new=4, mass=False, dtype="fp16"),
        # Two very long contexts: the work of a request has to be spread over the GPU.
        dict(name="attend 2x131072", kind="attend", batch=2, heads=32, kv_heads=8, dim=128, page=16, length=131072, ragged=False, new=1, mass=False, dtype="bf16"),
        # The page write of one decoding step.
        dict(name="write 16x1", kind="write", batch=16, heads=32, kv_heads=8, dim=128, page=16, start=2048, new=1, ragged=False, rope=True, bias=False, dtype="bf16"),
        # Prompts of different lengths in a padded batch, behind what is cached already; biases instead of a rotation.
        dict(name="write 5x389 ragged", kind="write", batch=5, heads=32, kv_heads=32, dim=64, page=16, start=77, new=389, ragged=True, rope=False, bias=True, dtype="fp16"),
        # The benchmark's prompts, all of them.
        dict(name="write 16x2048", kind="write", batch=16, heads=32, kv_heads=8, dim=128, page=16, start=0, new=2048, ragged=False, rope=True, bias=False, dtype="bf16"),
        # A batch that has outgrown its pages: one page of each request goes.  And long contexts cut by half.
        dict(name="evict 16 of 145", kind="evict", batch=16, pages=145, page=16, keep=144, recent=4, sinks=1),
        dict(name="evict 64 of 8192", kind="evict", batch=64, pages=8192, page=16, keep=4096, recent=8, sinks=1),
        # A few requests of a model whose vocabulary is an odd number; a large batch whose requests ask for different things.
        dict(name="sample 3x50257", kind="sample", batch=3, vocab=50257, dtype="fp16"),
        dict(name="sample 192x128256", kind="sample", batch=192, vocab=128256, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "write", "write", "evict", "sample", "sample"])
    dtype = rng.choice(["bf16", "fp16"])
    if kind == "sample":
        vocab = rng.choice([1000, 32000, 50257, 50272, 128256, _log(rng, 100, 128256)])
        return dict(kind=kind, batch=_log(rng, 1, 256), vocab=vocab, dtype=dtype)
    if kind == "evict":
        pages = _log(rng, 8, 8192)
        recent, sinks = rng.randint(1, 3), rng.randint(0, 2)
        return dict(kind=kind, batch=_log(rng, 1, 64), pages=pages, page=rng.choice([8, 16, 32]), keep=rng.randint(recent + sinks, pages), recent=recent, sinks=sinks)
    kv_heads, group = rng.choice([(8, 4), (32, 1), (8, 8), (1, 8), (4, 5), (25, 1), (2, 2)])
    dim, page = rng.choice([64, 80, 96, 128, 128, 128]), rng.choice([5, 8, 16, 16, 16, 32])
    batch = _log(rng, 1, 64)
    c = dict(kind=kind, batch=batch, heads=kv_heads * group, kv_heads=kv_heads, dim=dim, page=page)
    if kind == "write":
        new = rng.choice([1, 1, 2, _log(rng, 2, 2048)])
        new = max(1, min(new, 120_000_000 // (batch * (c["heads"] + 2 * kv_heads) * dim)))
        bias = rng.random() < 0.4
        return dict(c, start=rng.choice([0, _log(rng, 1, 4096)]), new=new, ragged=rng.random() < 0.5, rope=not bias, bias=bias, dtype=dtype)
    new = rng.choice([1, 1, 1, 2, 5, 8])
    most = 250_000_000 // (batch * kv_heads * dim * max(1, new * group // 8))
    return dict(c, length=max(9, min(_log(rng, 9, 131072), most)), ragged=rng.random() < 0.5, new=new, mass=rng.random() < 0.4, dtype=dtype)


def _spread(most, least, batch, ragged):
    """One length per request: `most`, or lengths from `least` to `most` in no order, the largest among them."""
    if not ragged:
        return [most] * batch
    return [most if b == batch // 2 else least + int((most - least) * math.modf((b + 0.5) * 0.6180339887498949)[0]) for b in range(batch)]


def _lengths(c):
    return _spread(c["length"], c["new"], c["batch"], c["ragged"])


def _starts_counts(c):
    return _spread(c["start"], 0, c["batch"], c["ragged"]), _spread(c["new"], (c["new"] + 1) // 2, c["batch"], c["ragged"])


# ---- inputs -----------------------------------------------------------------------------------------------------------------
def _scale_of(amax):
    """The smallest power of two, 2^-100 at least, that brings amax within 448."""
    m, e = torch.frexp(amax)                               # amax = m 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.where(m <= 0.875, e - 9, e - 8)
    return torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), e), torch.zeros_like(amax)).clamp(min=LEAST)


def _pool(gen, layers, pages, heads, page, dim, spread):
    """Codes [layers, pages, heads, page, dim] and scales [layers, pages, heads] of normally distributed values; `spread`: how far the
    channels' and the pages' magnitudes differ."""
    codes = torch.empty(layers * pages, heads, page, dim, dtype=F8, device=DEV)
    scales = torch.empty(layers * pages, heads, device=DEV)
    channel = torch.exp(spread * torch.randn(heads, 1, dim, generator=gen, device=DEV))
    step = max(1, (1 << 25) // (heads * page * dim))
    for a in range(0, layers * pages, step):
        n = min(step, layers * pages - a)
        x = torch.randn(n, heads, page, dim, generator=gen, device=DEV) * channel
        x = x * torch.exp(spread * torch.randn(n, heads, 1, 1, generator=gen, device=DEV))
        s = _scale_of(x.abs().amax((2, 3)))
        codes[a:a + n] = (x / s[:, :, None, None]).to(F8)
        scales[a:a + n] = s
    return codes.view(layers, pages, heads, page, dim), scales.view(layers, pages, heads)


def _table(gen, batch, each, pages):
    """Block table [batch, each]: pages in no order, every one once."""
    return torch.randperm(pages, generator=gen, device=DEV)[: batch * each].view(batch, each).int()


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    B = c["batch"]

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=DEV)

    def ints(values):
        return torch.tensor(values, dtype=torch.int64, device=DEV)

    if c["kind"] == "sample":
        V = c["vocab"]
        # a model's logits: a broad body and a few likely tokens; every request with what it asks for
        logits = 2.0 * randn(B, V)
        few = torch.randint(0, V, (B, 24), generator=gen, device=DEV)
        logits.scatter_add_(1, few, 6.0 + 2.5 * randn(B, 24))

        def of(values, dtype):
            at = torch.randint(0, len(values), (B,), generator=gen, device=DEV)
            return torch.tensor(values, dtype=dtype, device=DEV)[at].contiguous()

        return dict(c, logits=logits.to(DTYPES[c["dtype"]]), u=torch.rand(B, generator=gen, device=DEV),
                    temperature=of([0.6, 0.7, 0.8, 1.0, 1.0, 1.3], torch.float32), top_k=of([0, 0, 40, 50, 1000], torch.int32),
                    top_p=of([1.0, 0.8, 0.9, 0.95], torch.float32), min_p=of([0.0, 0.0, 0.05, 0.1], torch.float32))
    if c["kind"] == "evict":
        M, page = c["pages"], c["page"]
        lengths = ints([max(1, n * page - (7 * b) % page) for b, n in enumerate(_spread(M, max(1, M * 3 // 4), B, B > 1))])
        mass = torch.exp(2.0 * randn(B, M))                               # a few pages get most of the weight
        mass = torch.where(torch.rand(B, M, generator=gen, device=DEV) < 0.05, torch.zeros_like(mass), mass)      # and some none at all
        return dict(c, mass=mass, table=_table(gen, B, M, B * M), lengths=lengths)
    H, KH, D, page, dt = c["heads"], c["kv_heads"], c["dim"], c["page"], DTYPES[c["dtype"]]
    if c["kind"] == "attend":
        lens = _lengths(c)
        each = (max(lens) + page - 1) // page
        k, ks = _pool(gen, 1, B * each, KH, page, D, 0.4)
        v, vs = _pool(gen, 1, B * each, KH, page, D, 0.3)
        table = _table(gen, B, each, B * each)
        # slots behind a sequence's end hold what is left of earlier ones, or nothing that is a number
        last = torch.tensor([(n - 1) // page for n in lens], device=DEV)
        behind = torch.arange(page, device=DEV)[None] > (ints(lens) - 1 - last * page)[:, None]
        for pool in (k, v):
            rows = pool[0].view(torch.uint8)[table[torch.arange(B, device=DEV), last].long()]      # [B, KH, page, D]
            rows = torch.where(behind[:, None, :, None], torch.full_like(rows, 0x7F), rows)
            pool[0].view(torch.uint8)[table[torch.arange(B, device=DEV), last].long()] = rows
        return dict(c, q=(1.3 * randn(B, c["new"], H, D)).to(dt), k=k, v=v, ks=ks, vs=vs, table=table, start=ints(lens) - c["new"], layer=0)
    starts, counts = _starts_counts(c)
    each = (max(s + n for s, n in zip(starts, counts)) + page - 1) // page
    k, ks = _pool(gen, 1, B * each, KH, page, D, 0.4)
    v, vs = _pool(gen, 1, B * each, KH, page, D, 0.3)
    rope = None
    if c["rope"]:
        inv = 1.0 / (500000.0 ** (torch.arange(0, D, 2, device=DEV, dtype=torch.float64) / D))
        ang = torch.arange(each * page + 512, device=DEV, dtype=torch.float64).unsqueeze(-1) * inv
        rope = torch.cat([ang.cos(), ang.sin()], -1).float().contiguous()
    qkv = randn(B, c["new"], H + 2 * KH, D) * torch.exp(0.4 * randn(1, 1, H + 2 * KH, D))
    return dict(c, qkv=qkv.to(dt), k=k, v=v, ks=ks, vs=vs, table=_table(gen, B, each, B * each), start=ints(starts), counts=ints(counts),
                positions=ints(starts) + 3 * page, rope_table=rope, layer=0,
                bias_row=(0.5 * randn((H + 2 * KH) * D)).to(dt) if c["bias"] else None)


# ---- plain forms --------------------------------------------------------------------------------------------------------------
def _plain_attend(s):
    B, T, H, D = s["q"].shape
    KH, page, table = s["kv_heads"], s["page"], s["table"].long()
    n = table.shape[1] * page

    def dense(codes, scales):
        x = codes[s["layer"]][table].float() * scales[s["layer"]][table][..., None, None]          # [B, pages, KH, page, D]
        return x.permute(0, 2, 1, 3, 4).reshape(B, KH, n, D)

    seen = s["start"][:, None] + torch.arange(T, device=DEV) + 1                                    # [B, T]
    there = torch.arange(n, device=DEV) < seen[..., None]                                           # [B, T, n]
    k, v = dense(s["k"], s["ks"]), dense(s["v"], s["vs"])
    v = torch.where(there[:, -1][:, None, :, None], v, torch.zeros_like(v))
    q = s["q"].float().permute(0, 2, 1, 3).reshape(B, KH, (H // KH) * T, D)
    x = (q @ k.transpose(2, 3)) / math.sqrt(D)
    x = torch.where(there[:, None, None], x.view(B, KH, H // KH, T, n), torch.full((), -math.inf, device=DEV))
    p = torch.exp(x - x.amax(-1, keepdim=True))
    p = (p / p.sum(-1, keepdim=True)).view(B, KH, (H // KH) * T, n)
    out = (p @ v).view(B, H, T, D).permute(0, 2, 1, 3).reshape(B, T, H * D).to(s["q"].dtype)
    if not s["mass"]:
        return out
    return out, p.sum((1, 2)).view(B, -1, page).sum(-1)


def _plain_write(s):
    x, H, KH, page = s["qkv"].float(), s["heads"], s["kv_heads"], s["page"]
    B, T, _, D = x.shape
    at = torch.arange(T, device=DEV)
    if s["bias_row"] is not None:
        x = x + s["bias_row"].float().view(-1, D)
    if s["rope_table"] is not None:
        row = s["rope_table"][(s["positions"][:, None] + at).clamp(max=s["rope_table"].shape[0] - 1)][:, :, None]
        cos, sin = row[..., : D // 2], row[..., D // 2:]
        a, b = x[:, :, : H + KH, : D // 2], x[:, :, : H + KH, D // 2:]
        x = torch.cat([torch.cat([a * cos - b * sin, b * cos + a * sin], -1), x[:, :, H + KH:]], 2)
    out = torch.where((at < s["counts"][:, None])[..., None, None], x.to(s["qkv"].dtype), s["qkv"])
    start, end = s["start"], s["start"] + s["counts"]
    pi = (start // page)[:, None] + torch.arange((T + page - 2) // page + 1, device=DEV)            # pages that the runs can reach
    used = pi * page < end[:, None]
    ids = s["table"].long().gather(1, pi.clamp(max=s["table"].shape[1] - 1))[used]
    tok = (pi[..., None] * page + torch.arange(page, device=DEV) - start[:, None, None])[used]      # [n, page]
    req = torch.arange(B, device=DEV)[:, None].expand_as(pi)[used]
    new = ((tok >= 0) & (tok < s["counts"][req][:, None]))[:, None, :, None]
    old = (tok < 0)[:, None, :, None]
    for codes, scales, first in ((s["k"], s["ks"], H), (s["v"], s["vs"], H + KH)):
        y = out[req[:, None], tok.clamp(0, T - 1), first: first + KH].float().permute(0, 2, 1, 3)   # [n, KH, page, D]
        amax = torch.where(new, y.abs(), torch.zeros_like(y)).amax((2, 3))
        have, was = codes[s["layer"]][ids], scales[s["layer"]][ids]
        was = torch.where(old.any(2)[:, :, 0], was, torch.full_like(was, LEAST))
        scale = torch.maximum(was, _scale_of(amax))
        fresh = (y / scale[..., None, None]).to(F8)
        kept = (have.float() * (was / scale)[..., None, None]).to(F8)
        got = torch.where(new, fresh.view(torch.uint8), torch.where(old, kept.view(torch.uint8), have.view(torch.uint8)))
        codes[s["layer"]].view(torch.uint8)[ids] = got
        scales[s["layer"]][ids] = scale
    return out, s["k"], s["v"], s["ks"], s["vs"]


def _plain_evict(s):
    mass, M, page = s["mass"], s["pages"], s["page"]
    at = torch.arange(M, device=DEV)[None]
    used = ((s["lengths"] + page - 1) // page)[:, None]
    extra = (used - s["keep"]).clamp(min=0)
    free = (at >= s["sinks"]) & (at < used - s["recent"])
    order = torch.sort(mass, dim=1, stable=True)[1]
    order = order.gather(1, torch.sort((~free.gather(1, order)).int(), dim=1, stable=True)[1])          # lightest of those that may go first
    rank = torch.empty_like(order).scatter_(1, order, at.expand_as(order))
    gone = rank < extra
    to = torch.sort(torch.where(at >= used, 2, gone.int()), dim=1, stable=True)[1]
    return (s["table"].gather(1, to), s["lengths"] - extra[:, 0] * page, torch.where(gone, torch.zeros_like(mass), mass).gather(1, to), extra[:, 0].int())


def _plain_sample(s):
    V = s["vocab"]
    v, order = torch.sort(s["logits"].float(), dim=1, descending=True, stable=True)
    d = (v.double() - v[:, :1].double()) / s["temperature"].double()[:, None]
    w = torch.exp(d)
    c = w.cumsum(1)
    k = torch.where((s["top_k"] > 0) & (s["top_k"] < V), s["top_k"].long(), V)[:, None]
    p, m = s["top_p"].double()[:, None], s["min_p"].double()[:, None]
    inside = torch.where(p < 1, (c < p * c.gather(1, k - 1)).sum(1, keepdim=True) + 1, V)
    n = torch.minimum(torch.minimum(k, inside), (w >= m).sum(1, keepdim=True)).clamp(min=1)
    total = c.gather(1, n - 1)
    j = torch.minimum((c <= s["u"].double()[:, None] * total).sum(1, keepdim=True), n - 1)
    return order.gather(1, j)[:, 0], (d.gather(1, j) - total.log())[:, 0].float()


def run(state):
    s = state
    if not own:
        return {"attend": _plain_attend, "write": _plain_write, "evict": _plain_evict, "sample": _plain_sample}[s["kind"]](s)
    from fuselink_b200.ops import kv8, sampling

    if s["kind"] == "sample":
        return sampling.sample(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])
    if s["kind"] == "evict":
        return kv8.evict(s["mass"], s["table"], s["lengths"], s["page"], s["keep"], recent=s["recent"], sinks=s["sinks"])
    cache = kv8.Kv8Cache(s["k"], s["v"], s["ks"], s["vs"])
    if s["kind"] == "write":
        out = kv8.write(cache, s["layer"], s["qkv"], s["table"], s["start"], counts=s["counts"], positions=s["positions"], rope=s["rope_table"], bias=s["bias_row"])
        return out, s["k"], s["v"], s["ks"], s["vs"]
    if not s["mass"]:
        return kv8.attention(cache, s["layer"], s["q"], s["table"], s["start"])
    mass = torch.zeros(s["table"].shape, device=DEV)
    return kv8.attention(cache, s["layer"], s["q"], s["table"], s["start"], mass=mass), mass


def work(case):
    c = case
    if c["kind"] == "sample":
        return dict(bytes=c["batch"] * (2 * c["vocab"] + 32), flops=2 * c["batch"] * c["vocab"])
    if c["kind"] == "evict":
        return dict(bytes=c["batch"] * (16 * c["pages"] + 20), flops=c["batch"] * c["pages"])
    H, KH, D, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    if c["kind"] == "attend":
        lens, T = _lengths(c), c["new"]
        pages = sum((n + page - 1) // page for n in lens)
        seen = sum(sum(n - T + t + 1 for t in range(T)) for n in lens)
        return dict(bytes=2 * sum(lens) * KH * D + pages * (8 * KH + 4 + (4 if c["mass"] else 0)) + 4 * c["batch"] * T * H * D, flops=4 * seen * H * D)
    starts, counts = _starts_counts(c)
    pages = sum((a + n - 1) // page - a // page + 1 for a, n in zip(starts, counts))
    return dict(bytes=sum(counts) * D * (4 * (H + 2 * KH) + 2 * KH) + 8 * pages * KH + (sum(counts) * 4 * D if c["rope"] else 0),
                flops=sum(counts) * D * (3 * (H + KH) + 4 * KH))


# ---- the same from the definitions, in 64 bits -----------------------------------------------------------------------------------
def _exact_attend(s):
    B, T, H, D = s["q"].shape
    KH, page = s["kv_heads"], s["page"]
    out = torch.zeros(B, T, H, D, dtype=torch.float64, device=DEV)
    mass = torch.zeros(s["table"].shape, dtype=torch.float64, device=DEV)
    for b in range(B):
        end = int(s["start"][b]) + T
        ids = s["table"][b, : (end + page - 1) // page].long()
        for h in range(KH):
            k, v = ((codes[s["layer"], ids, h].double() * scales[s["layer"], ids, h].double()[:, None, None]).reshape(-1, D)[:end]
                    for codes, scales in ((s["k"], s["ks"]), (s["v"], s["vs"])))
            heads = slice(h * (H // KH), (h + 1) * (H // KH))
            for t in range(T):
                seen = end - T + t + 1
                p = torch.softmax(s["q"][b, t, heads].double() @ k[:seen].T * D ** -0.5, 1)
                out[b, t, heads] = p @ v[:seen]
                if s["mass"]:
                    mass[b].index_add_(0, torch.arange(seen, device=DEV) // page, p.sum(0))
    out = out.reshape(B, T, H * D)
    return (out, mass) if s["mass"] else out


def _exact_write(s):
    """The rotated rows in 64 bits; codes and scales follow from those rows in the model's type."""
    H, KH, page, D = s["heads"], s["kv_heads"], s["page"], s["dim"]
    x = s["qkv"].cpu().double().numpy()
    rows = x.copy()
    k, v, ks, vs = (s[name].double().cpu().numpy().copy() for name in ("k", "v", "ks", "vs"))
    table = s["table"].cpu().numpy()
    rope = None if s["rope_table"] is None else s["rope_table"].cpu().double().numpy()

    def code(values):
        return torch.from_numpy(values).float().to(F8).double().numpy()

    for b in range(s["batch"]):
        first, n, turn = int(s["start"][b]), int(s["counts"][b]), int(s["positions"][b])
        y = x[b, :n]
        if s["bias_row"] is not None:
            y = y + s["bias_row"].cpu().double().numpy().reshape(-1, D)
        if rope is not None:
            z = (y[:, : H + KH, : D // 2] + 1j * y[:, : H + KH, D // 2:]) * (rope[turn: turn + n, None, : D // 2] + 1j * rope[turn: turn + n, None, D // 2:])
            y = np.concatenate([np.concatenate([z.real, z.imag], -1), y[:, H + KH:]], 1)
        rows[b, :n] = y
        typed = torch.from_numpy(y).to(s["qkv"].dtype).double().numpy()
        for lead in range(first // page, (first + n - 1) // page + 1 if n else first // page):
            lo, hi = max(first - lead * page, 0), min(first + n - lead * page, page)
            at = (s["layer"], table[b, lead])
            for codes, scales, head in ((k, ks, H), (v, vs, H + KH)):
                new = typed[lead * page + lo - first: lead * page + hi - first, head: head + KH].transpose(1, 0, 2)
                scale = np.maximum(2.0 ** np.ceil(np.log2(np.maximum(np.abs(new).max((1, 2)), 1e-300) / 448.0)), LEAST)
                if lo > 0:
                    scale = np.maximum(scale, scales[at])
                codes[at][:, :lo] = code(codes[at][:, :lo] * (scales[at] / scale)[:, None, None])
                codes[at][:, lo:hi] = code(new / scale[:, None, None])
                scales[at] = scale
    return (torch.from_numpy(rows), *(torch.from_numpy(t) for t in (k, v, ks, vs)))


def _exact_sample(s):
    """The logarithm of the chosen token's probability; the tokens themselves are whole numbers."""
    said = []
    for b in range(s["batch"]):
        x = s["logits"][b].cpu().double().numpy()
        x = np.sort(x)[::-1]
        x = (x - x[0]) / float(s["temperature"][b])
        e = np.exp(x)
        k = int(s["top_k"][b])
        n = k if 0 < k < x.size else x.size
        if float(s["min_p"][b]) > 0:
            n = min(n, int(np.searchsorted(-e, -float(s["min_p"][b]), side="right")))
        if float(s["top_p"][b]) < 1:
            kept = e[: k if 0 < k < x.size else x.size]
            n = min(n, int(np.searchsorted(np.cumsum(kept), float(s["top_p"][b]) * math.fsum(kept), side="left")) + 1)
        n = max(n, 1)
        z = math.fsum(e[:n])
        j = min(int(np.searchsorted(np.cumsum(e[:n]), float(s["u"][b]) * z, side="right")), n - 1)
        said.append(x[j] - math.log(z))
    return None, torch.tensor(said, dtype=torch.float64)


def _exact_evict(s):
    """The weights at their new places; the rest are whole numbers."""
    page, said = s["page"], s["mass"].cpu().double().numpy().copy()
    for b, n in enumerate(s["lengths"].tolist()):
        used = -(-n // page)
        free = sorted(range(s["sinks"], used - s["recent"]), key=lambda i: (said[b, i], i))
        gone = sorted(free[: max(0, used - s["keep"])])
        kept = sorted(set(range(used)) - set(gone))
        said[b, :used] = np.concatenate([said[b, kept], np.zeros(len(gone))])
    return None, None, torch.from_numpy(said), None


def exact(case, seed):
    w = work(case)
    if w["bytes"] > 150_000_000 and case["kind"] != "attend":
        return None                                        # minutes
    return {"attend": _exact_attend, "write": _exact_write, "evict": _exact_evict, "sample": _exact_sample}[case["kind"]](prepare(case, seed))
