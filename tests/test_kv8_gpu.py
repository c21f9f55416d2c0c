"""The cache in 8 bits (csrc/kernels/kv8.cu) against the same in 64 bits: page write, attention, weights of pages, eviction."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DT = [torch.bfloat16, torch.float16]
F8 = torch.float8_e4m3fn
BF, HF = DT


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(*shape, seed=0, dt=torch.float32):
    return torch.randn(*shape, generator=_gen(seed), device="cuda").to(dt)


def _ints(values):
    return torch.tensor(values, dtype=torch.int64, device="cuda")


def _scale64(amax):
    """Smallest power of two, 2^-100 at least, that keeps amax within 448; amax in 64 bits."""
    return torch.exp2(torch.ceil(torch.log2(amax.clamp(min=1e-300) / 448.0))).clamp(min=2.0 ** -100)


def _cache(layers, blocks, kv_heads, bs, dim, seed=1, spread=1.0):
    """A cache whose every slot holds something."""
    from fuselink_b200.ops.kv8 import Kv8Cache
    made = []
    for s in (seed, seed + 1):
        x = _randn(layers, blocks, kv_heads, bs, dim, seed=s) * torch.exp(spread * _randn(layers, blocks, kv_heads, 1, 1, seed=s + 10))
        sc = _scale64(x.abs().amax((3, 4)).double()).float()
        made.append(((x / sc[..., None, None]).to(F8), sc))
    (k, ks), (v, vs) = made
    return Kv8Cache(k, v, ks, vs)


def _table(batch, each, blocks, seed=3):
    return torch.randperm(blocks, generator=torch.Generator().manual_seed(seed))[: batch * each].view(batch, each).int().cuda()


def _values(codes, scales):
    return codes.double() * scales.double()[..., None, None]


def _same(a, b):
    """Equal codes, any NaN like any other."""
    a, b = a.float(), b.float()
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num())


def _want_write(cache, layer, rows, table, start, counts, heads):
    """The cache after tokens whose rows (in the model's type) are given, by definition."""
    k, v, ks, vs = (t.double() for t in cache.tensors())
    bs, KH = cache.block_size, cache.k.shape[2]
    for b, (first, n) in enumerate(zip(start, counts)):
        for page in range(first // bs, (first + n - 1) // bs + 1 if n else first // bs):
            lo, hi = max(first, page * bs), min(first + n, (page + 1) * bs)
            at = (layer, int(table[b, page]))
            for codes, scales, head in ((k, ks, heads), (v, vs, heads + KH)):
                x = rows[b, lo - first: hi - first, head: head + KH].double().transpose(0, 1)
                x = torch.where(x.isfinite(), x, torch.full_like(x, math.nan))
                s = _scale64(x.abs().nan_to_num(0.0).amax((1, 2)))
                lead = lo - page * bs
                if lead:
                    s = torch.maximum(s, scales[at])
                    codes[at][:, :lead] = (codes[at][:, :lead] * (scales[at] / s)[:, None, None]).to(F8).double()
                codes[at][:, lead: hi - page * bs] = (x / s[:, None, None]).float().to(F8).double()
                scales[at] = s
    return k, v, ks, vs


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("heads,kv_heads,dim,bs,tokens,start,counts,how", [
    (1, 1, 16, 16, 1, [0], None, "rope"),
    (4, 2, 64, 16, 1, [15, 16, 17], None, "rope"),
    (32, 8, 128, 16, 1, [5 * i for i in range(16)], None, "rope"),
    (3, 3, 80, 8, 40, [0, 7, 100], [40, 0, 33], "bias"),
    (5, 1, 96, 5, 11, [3, 20], [1, 11], "both"),
    (8, 8, 128, 32, 100, [31, 0], None, "none"),
    (2, 2, 128, 100, 230, [50], None, "rope"),
    (16, 4, 48, 24, 37, [0] * 20, [i * 2 for i in range(20)], "rope"),
])
def test_write(dt, heads, kv_heads, dim, bs, tokens, start, counts, how):
    from fuselink_b200.ops import kv8
    batch, A = len(start), heads + 2 * kv_heads
    n = [min(c, tokens) for c in counts or [tokens] * batch]
    each = (max(s + tokens for s in start) + bs - 1) // bs + 1
    cache = _cache(2, batch * each + 3, kv_heads, bs, dim, spread=2.0)
    table = _table(batch, each, batch * each + 3)
    table[0] -= batch * each + 3                                     # negative ids count from the end
    qkv = (_randn(batch, tokens, A, dim, seed=5) * torch.exp(2 * _randn(batch, tokens, A, 1, seed=6))).to(dt)
    ang = torch.arange(each * bs + 64, device="cuda", dtype=torch.float64)[:, None] / 100.0 ** (torch.arange(dim // 2, device="cuda") / (dim // 2))
    rope = torch.cat([ang.cos(), ang.sin()], 1).float() if how in ("rope", "both") else None
    bias = _randn(A * dim, seed=7, dt=dt) if how in ("bias", "both") else None
    turn = [s + 9 for s in start]
    want = qkv.double()
    if bias is not None:
        want = want + bias.double().view(A, dim)
    if rope is not None:
        r = torch.stack([rope[t: t + tokens] for t in turn]).double()[:, :, None]
        lo, hi, c, s = want[..., : dim // 2], want[..., dim // 2:], r[..., : dim // 2], r[..., dim // 2:]
        turned = torch.cat([lo * c - hi * s, hi * c + lo * s], -1)
        want = torch.cat([turned[:, :, : heads + kv_heads], want[:, :, heads + kv_heads:]], 2)
    for b in range(batch):
        want[b, n[b]:] = qkv[b, n[b]:].double()
    args = dict(counts=None if counts is None else _ints(counts), positions=_ints(turn), rope=rope, bias=bias)
    before = [t.clone() for t in cache.tensors()]
    out = kv8.write(cache, 1, qkv, table, _ints(start), **args)
    # one rounding to the type, and fp32's of a sum of three products of magnitudes up to those of the row's pair
    size = qkv.double().abs() + (0 if bias is None else bias.double().view(A, dim).abs())
    size = size + size.roll(dim // 2, -1)
    assert ((out.double() - want).abs() <= torch.finfo(dt).eps / 2 * want.abs() * 1.001 + 2.0 ** -22 * size + torch.finfo(dt).tiny * torch.finfo(dt).eps).all()
    now = [t.clone() for t in cache.tensors()]
    for t, was in zip(cache.tensors(), before):
        t.copy_(was)
    expect = _want_write(cache, 1, out, table, start, n, heads)
    for got, exp in zip(now, expect):
        assert _same(got, exp)
    # in place, the same bits
    inside = qkv.clone()
    assert kv8.write(cache, 1, inside, table, _ints(start), out=inside, **args) is inside
    assert torch.equal(inside, out)
    for got, exp in zip(cache.tensors(), now):
        assert torch.equal(got.view(torch.uint8) if got.dtype == F8 else got, exp.view(torch.uint8) if exp.dtype == F8 else exp)


def test_rows_of_any_order():
    """Rows that are no contiguous tensor are written as their copy; scales other than the heads' own, 0 among them."""
    from fuselink_b200.ops import kv8
    table = _table(2, 2, 5)
    x = _randn(3, 2, 8, 64, seed=3, dt=BF).transpose(0, 1)             # [2, 3, 8, 64]
    a, b = _cache(1, 5, 2, 16, 64), _cache(1, 5, 2, 16, 64)
    out = kv8.write(a, 0, x, table, _ints([4, 15]))
    assert torch.equal(out, kv8.write(b, 0, x.contiguous(), table, _ints([4, 15]))) and torch.equal(out, x)
    for s, t in zip(a.tensors(), b.tensors()):
        assert torch.equal(s.view(torch.uint8), t.view(torch.uint8))
    q = _randn(8, 3, 2, 64, seed=4, dt=BF).permute(2, 1, 0, 3)[:, :, ::2]        # [2, 3, 4, 64], strides of multiples of 64
    for scale in (0.0, 0.01, 1.0):
        want, _, may = _want_attention(a, 0, q, table, [4, 15], [3, 3], scale)
        _check(kv8.attention(a, 0, q, table, _ints([4, 15]), scale=scale), want, may, BF)
    with pytest.raises(ValueError):
        kv8.attention(a, 0, q, table, _ints([4, 15]), scale=-0.1)


def test_a_page_follows_its_scale_token_by_token():
    """Growing magnitudes: every token raises the scale; the earlier codes follow it each time."""
    from fuselink_b200.ops import kv8
    cache = _cache(1, 4, 2, 16, 64)
    table = torch.tensor([[2, 1]], dtype=torch.int32, device="cuda")
    x = _randn(1, 20, 6, 64, seed=8, dt=BF) * (3.0 ** torch.arange(20, device="cuda"))[None, :, None, None].to(BF)
    for t in range(20):
        was = [c.clone() for c in cache.tensors()]
        kv8.write(cache, 0, x[:, t: t + 1].contiguous(), table, _ints([t]))
        from fuselink_b200.ops.kv8 import Kv8Cache
        for got, exp in zip(cache.tensors(), _want_write(Kv8Cache(*was), 0, x[:, t: t + 1], table, [t], [1], 2)):
            assert _same(got, exp)


@pytest.mark.parametrize("dt", DT)
def test_values_that_are_not_finite_become_nan(dt):
    from fuselink_b200.ops import kv8
    cache = _cache(1, 3, 1, 16, 64)
    table = torch.tensor([[1]], dtype=torch.int32, device="cuda")
    x = _randn(1, 16, 3, 64, seed=9, dt=dt)
    x[0, 3, 1, 5], x[0, 4, 1, 6], x[0, 5, 2, 7], x[0, 6] = math.inf, -math.inf, math.nan, 0.0
    was = [t.clone() for t in cache.tensors()]
    kv8.write(cache, 0, x, table, _ints([0]))
    from fuselink_b200.ops.kv8 import Kv8Cache
    for got, exp in zip(cache.tensors(), _want_write(Kv8Cache(*was), 0, x, table, [0], [16], 1)):
        assert _same(got, exp)
    assert cache.k[0, 1].float().isnan().sum() == 2 and cache.v[0, 1].float().isnan().sum() == 1


@pytest.mark.parametrize("most", [0.0, 2.0 ** -133, 2.0 ** -92, 1.75 * 2.0 ** -3, 1.7578125 * 2.0 ** -3, 3.3e38])
def test_scales_at_the_ends(most):
    """A page of zeros, of magnitudes below every scale, at a scale's limit and one step above it, and the type's largest."""
    from fuselink_b200.ops import kv8
    cache = _cache(1, 2, 1, 16, 16)
    table = torch.tensor([[0]], dtype=torch.int32, device="cuda")
    x = torch.zeros(1, 4, 3, 16, dtype=BF, device="cuda")
    x[0, 2, 1:, 3] = torch.tensor([most, -most], dtype=torch.float64).to(BF).cuda()
    kv8.write(cache, 0, x, table, _ints([0]))
    m = x.double().abs().max()
    want = _scale64(m) if m > 0 else torch.tensor(2.0 ** -100, dtype=torch.float64)
    for scale, codes, sign in ((cache.k_scale, cache.k, 1), (cache.v_scale, cache.v, -1)):
        assert scale[0, 0, 0].double().item() == want.item()
        got = codes[0, 0, 0, :4].double() * scale[0, 0, 0].double()
        assert (got - sign * x[0, :, 1].double().abs()).abs().max() <= max(2.0 ** -4 * m.item(), 2.0 ** -110)


@pytest.mark.parametrize("bs", [8, 16, 40])
def test_pack_is_the_write_of_the_pages_tokens(bs):
    from fuselink_b200.ops import kv8
    L, KH, D, blocks, lens = 3, 4, 64, 40, [1, bs, 0, 3 * bs - 1]
    for dt in DT:
        pools = [_randn(L, blocks, bs, KH, D, seed=s, dt=dt) for s in (1, 2)]
        src, dst = _table(4, 3, blocks, seed=5), _table(4, 4, 50, seed=6)
        a, b = _cache(L, 50, KH, bs, D), _cache(L, 50, KH, bs, D)
        kv8.pack(a, pools[0].view(-1), pools[1].view(-1), blocks, src, dst, _ints(lens))
        for layer in range(L):
            k, v = (p[layer][src.long()].reshape(4, 3 * bs, KH, D) for p in pools)
            kv8.write(b, layer, torch.cat([k, v], 2).contiguous(), dst, _ints([0] * 4), counts=_ints(lens))
        for x, y in zip(a.tensors(), b.tensors()):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


# ---- attention -------------------------------------------------------------------------------------------------------------------
def _want_attention(cache, layer, q, table, start, counts, scale=None):
    """Output and weights per slot in 64 bits, and how far an output may be off before it is rounded."""
    B, T, H, D = q.shape
    KH, bs = cache.k.shape[2], cache.block_size
    cap = table.shape[1] * bs
    scale = D ** -0.5 if scale is None else scale
    out, may = (torch.zeros(B, T, H, D, dtype=torch.float64, device="cuda") for _ in range(2))
    mass = torch.zeros(B, cap, dtype=torch.float64, device="cuda")
    for b in range(B):
        for t in range(counts[b]):
            seen = min(start[b] + t + 1, cap)
            if seen <= 0:
                continue
            pages = table[b, : (seen + bs - 1) // bs].long()
            there = ((pages >= -cache.k.shape[1]) & (pages < cache.k.shape[1])).repeat_interleave(bs)[:seen]
            k, v = (_values(c[layer][pages.clamp(-c.shape[1], c.shape[1] - 1)], s[layer][pages.clamp(-c.shape[1], c.shape[1] - 1)]).transpose(0, 1).reshape(KH, -1, D)[:, :seen]
                    .repeat_interleave(H // KH, 0) for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
            qq = q[b, t].double()
            x = torch.einsum("hd,hnd->hn", qq, k) * scale
            x = torch.where(there, x, torch.full_like(x, -math.inf))
            p = x.softmax(-1)
            v = torch.where(there[:, None], v, torch.zeros_like(v))
            out[b, t] = torch.einsum("hn,hnd->hd", p, v)
            mass[b, :seen] += p.sum(0)
            # The weights, at most 1 before they are divided by a sum of at least 1, are rounded to 11 bits (and to steps of 2^-24 below 2^-14); scores are sums
            # of D exact products in fp32, each step a truncation of 2^-23 at most, times a factor and through an exponential, three more roundings each
            # of 2^-23 of the score; the sums over the tokens the same way again.
            size = (torch.einsum("hd,hnd->hn", qq.abs(), k.abs()) * scale).nan_to_num(0, 0, 0).amax(-1)
            big = v.abs().nan_to_num(0, 0, 0).amax((1, 2))
            may[b, t] = ((2.0 ** -11 + seen * 2.0 ** -25 + 2 * (D + 6) * 2.0 ** -23 * size + (seen + 8) * 2.0 ** -23) * big)[:, None]
    return out.view(B, T, H * D), mass.view(B, -1, bs).sum(-1), may.view(B, T, H * D)


def _check(got, want, may, dt):
    assert torch.equal(got.isnan(), want.isnan())
    ok = ~want.isnan()
    off = (got.double() - want).abs()[ok] - (may + torch.finfo(dt).eps / 2 * want.abs() * 1.01 + 2.0 ** -25)[ok]
    assert (off <= 0).all(), off.max().item()


SHAPES = [  # heads, kv_heads, dim, bs, tokens, lengths (slots that the last token sees)
    (1, 1, 16, 16, 1, [1]),
    (4, 2, 64, 16, 1, [1, 15, 16, 17, 100]),
    (32, 8, 128, 16, 1, [2049, 700, 1]),
    (12, 12, 80, 8, 1, [129, 1]),
    (24, 2, 128, 5, 1, [333, 1000]),
    (8, 8, 96, 16, 1, [7 * i + 1 for i in range(17)]),
    (64, 8, 128, 32, 1, [5000]),
    (8, 1, 128, 16, 1, [20000]),
    (5, 1, 64, 24, 1, [500, 31]),
    (4, 4, 64, 16, 1, [40 + i for i in range(150)]),
    (8, 2, 128, 16, 3, [3, 16, 18, 200]),
    (32, 32, 80, 32, 4, [1531, 4]),
    (64, 8, 128, 16, 8, [1000, 8, 33]),
    (10, 2, 112, 7, 5, [5, 50, 613]),
    (3, 1, 32, 16, 40, [40, 111, 2500]),
    (8, 2, 128, 16, 150, [150, 777]),
    (2, 2, 128, 8, 1, [8, 9, 4000, 7]),
    (8, 1, 64, 5, 3, [3, 4, 10, 11, 1201]),
    (16, 2, 96, 20, 2, [2, 20, 21, 44, 999]),
]


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("heads,kv_heads,dim,bs,tokens,lens", SHAPES)
def test_attention(dt, heads, kv_heads, dim, bs, tokens, lens):
    from fuselink_b200.ops import kv8
    batch, each = len(lens), (max(lens) + bs - 1) // bs + 2
    blocks = batch * each + 1
    cache, table = _cache(2, blocks, kv_heads, bs, dim), _table(batch, each, blocks)
    table[0] -= blocks
    for b, n in enumerate(lens):                                      # behind a request's end there is nothing that is a number
        ids = table[b].long()
        for codes in (cache.k, cache.v):
            flat = codes[1].view(torch.uint8)[ids].transpose(1, 2).reshape(each * bs, kv_heads, dim)
            flat[n:] = 0x7F
            codes[1].view(torch.uint8)[ids] = flat.view(each, bs, kv_heads, dim).transpose(1, 2)
        for scales in (cache.k_scale, cache.v_scale):
            scales[1, ids[(n + bs - 1) // bs:]] = math.nan
    rows = _randn(batch, tokens, heads + 2 * kv_heads, dim, seed=4, dt=dt)
    q = rows[:, :, :heads]                                             # as a decoder has them: beside the keys and values
    start = _ints(lens) - tokens
    mass = torch.full((batch, each), 0.5, device="cuda")
    want, weights, may = _want_attention(cache, 1, q, table, start.tolist(), [tokens] * batch)
    out = kv8.attention(cache, 1, q, table, start, out=torch.full((batch, tokens, heads * dim), math.nan, dtype=dt, device="cuda"))
    _check(out, want, may, dt)
    again = kv8.attention(cache, 1, q, table, start, mass=mass)
    assert torch.equal(out, again)
    # a page's weight: a sum over rows and slots of weights off by the scores' errors alone (relative); then the addition to what was there
    size = 2 * (dim + 8) * 2.0 ** -23 * 6 * max(1.0, float(rows.float().abs().max()) * float(dim) ** 0.5) * float(_values(cache.k[1, table.long()], cache.k_scale[1, table.long()]).nan_to_num().abs().max())
    assert ((mass.double() - 0.5 - weights).abs() <= size * weights + 2.0 ** -22 * (weights + 0.5)).all()
    twice = torch.full((batch, each), 0.5, device="cuda")
    kv8.attention(cache, 1, q, table, start, mass=twice)
    assert torch.equal(mass, twice)                                    # the order of the sums is always the same


@pytest.mark.parametrize("dt", DT)
def test_attention_of_a_padded_batch(dt):
    """Requests of fewer new tokens than others, of none, and with nothing to see: zeros there, and no weight."""
    from fuselink_b200.ops import kv8
    bs, each = 16, 12
    cache, table = _cache(1, 60, 2, bs, 64), _table(5, each, 60)
    start, counts = [-1, 0, 100, 30, -3], [1, 6, 3, 0, 6]
    table[3] = 1000                                                   # is not looked at
    q = _randn(5, 6, 8, 64, seed=4, dt=dt)
    mass = torch.zeros(5, each, device="cuda")
    want, weights, may = _want_attention(cache, 0, q, table, start, counts)
    word = torch.zeros(1, dtype=torch.int32).pin_memory()
    out = kv8.attention(cache, 0, q, table, _ints(start), counts=_ints(counts), mass=mass, status=word.data_ptr())
    _check(out, want, may, dt)
    torch.cuda.synchronize()
    assert int(word) == 0
    for b, n in enumerate(counts):
        assert out[b, n:].abs().max() == 0 if n < 6 else True
    assert out[0].abs().max() == 0 and out[4, :3].abs().max() == 0 and out[4, 3].abs().max() > 0
    assert mass[3].abs().max() == 0 and mass[0].abs().max() == 0
    assert ((mass.double() - weights).abs() <= 1e-4 * weights + 1e-12).all()


@pytest.mark.parametrize("kv_heads,group,dim,bs", [(2, 2, 64, 16), (1, 8, 128, 16), (3, 1, 80, 8)])
def test_later_tokens_reach_no_earlier_one(kv_heads, group, dim, bs):
    """A NaN in the last of five new tokens' value and key: the four before it are as without."""
    from fuselink_b200.ops import kv8
    cache, table = _cache(1, 20, kv_heads, bs, dim), _table(2, 10, 20)
    q, start = _randn(2, 5, kv_heads * group, dim, seed=4, dt=BF), [37, 0]
    clean = kv8.attention(cache, 0, q, table, _ints(start))
    for b, s in enumerate(start):
        slot = s + 4
        for codes in (cache.k, cache.v):
            codes.view(torch.uint8)[0, table[b, slot // bs].long(), :, slot % bs] = 0x7F
    out = kv8.attention(cache, 0, q, table, _ints(start))
    assert torch.equal(out[:, :4], clean[:, :4]) and out[:, 4].isnan().all()


@pytest.mark.parametrize("where", ["key", "value"])
@pytest.mark.parametrize("lens", [[40, 5], [2049, 1500]])
def test_nan_stays_with_its_head_and_request(where, lens):
    from fuselink_b200.ops import kv8
    each = max(lens) // 16 + 1
    cache, table = _cache(1, 2 * each, 4, 16, 64), _table(2, each, 2 * each)
    q = _randn(2, 1, 8, 64, seed=4, dt=HF)
    start = _ints(lens) - 1
    clean = kv8.attention(cache, 0, q, table, start).view(2, 8, 64)
    (cache.k if where == "key" else cache.v).view(torch.uint8)[0, table[0, 1].long(), 1, 3, 7] = 0x7F
    out = kv8.attention(cache, 0, q, table, start).view(2, 8, 64)
    hit = torch.zeros_like(out, dtype=torch.bool)
    if where == "key":
        hit[0, 2:4] = True
    else:
        hit[0, 2:4, 7] = True
    assert torch.equal(out.isnan(), hit) and torch.equal(out[~hit], clean[~hit])


def test_queries_of_any_magnitude():
    """bf16 queries far outside fp16's range, beside ordinary ones; infinite ones give NaN as a softmax does."""
    from fuselink_b200.ops import kv8
    cache, table = _cache(1, 8, 2, 16, 64, spread=0.0), _table(1, 8, 8)
    q = _randn(1, 1, 8, 64, seed=4, dt=BF)
    q[0, 0] *= torch.tensor([1e-30, 1e-6, 1.0, 30.0, 1.0, 1e-36, 0.0, 5.0], device="cuda")[:, None].to(BF)
    q[0, 0, 4, 9] = math.inf
    want, _, may = _want_attention(cache, 0, q, table, [120], [1])
    out = kv8.attention(cache, 0, q, table, _ints([120]))
    want[0, 0, 4 * 64: 5 * 64] = math.nan                             # inf - inf among the scores
    _check(out, want, may, BF)
    # scores of one sign only: all of the weight on the largest
    big = torch.zeros(1, 1, 2, 64, dtype=BF, device="cuda")
    big[..., 0] = 1e30
    out = kv8.attention(cache, 0, big, table, _ints([127])).view(2, 64)
    k, v = (_values(c[0][table[0].long()], s[0][table[0].long()]).transpose(0, 1).reshape(2, 128, 64) for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
    for h in range(2):
        top = k[h, :, 0] == k[h, :, 0].max()
        assert ((out[h].double() - v[h, top].mean(0)).abs() <= 2.0 ** -8 * v[h].abs().max()).all()


@pytest.mark.parametrize("tokens", [1, 4])
@pytest.mark.parametrize("bad", [1 << 20, -(1 << 20)])
def test_a_page_outside_the_pool_is_left_out_and_noted(tokens, bad):
    from fuselink_b200.ops import kv8
    cache, table = _cache(1, 30, 2, 16, 64), _table(2, 10, 30)
    table[0, 2] = bad
    q = _randn(2, tokens, 4, 64, seed=4, dt=BF)
    word = torch.zeros(1, dtype=torch.int32).pin_memory()
    mass = torch.zeros(2, 10, device="cuda")
    want, weights, may = _want_attention(cache, 0, q, table, [100, 60], [tokens] * 2)
    out = kv8.attention(cache, 0, q, table, _ints([100, 60]), mass=mass, status=word.data_ptr())
    torch.cuda.synchronize()
    assert int(word) == 3
    _check(out, want, may, BF)
    assert mass[0, 2] == 0 and ((mass.double() - weights).abs() <= 1e-4 * weights).all()
    word.zero_()
    before = [t.clone() for t in cache.tensors()]
    kv8.write(cache, 0, _randn(2, 1, 8, 64, seed=5, dt=BF), table, _ints([35, 160]), status=word.data_ptr())       # that page, and a slot behind the table
    torch.cuda.synchronize()
    assert int(word) in (2, 3)
    for a, b in zip(before, cache.tensors()):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    word.zero_()
    kv8.write(cache, 0, _randn(1, 1, 8, 64, seed=5, dt=BF), table[1:], _ints([-1]), status=word.data_ptr())
    torch.cuda.synchronize()
    assert int(word) == 2
    word.zero_()
    rope = torch.zeros(50, 64, device="cuda")
    x = _randn(1, 1, 8, 64, seed=5, dt=BF)
    y = kv8.write(cache, 0, x, table[1:], _ints([60]), rope=rope, status=word.data_ptr())            # a rotation that is not there
    torch.cuda.synchronize()
    assert int(word) == 2 and torch.equal(x, y)


def test_a_pool_beyond_32_bits():
    """Codes and rows whose offsets 32 bits do not hold."""
    from fuselink_b200.ops import kv8
    L, blocks, KH, bs, D = 3, 50000, 8, 16, 128                        # 2.46 G codes per pool
    cache = kv8.Kv8Cache.empty(L, blocks, KH, bs, D)
    table = torch.tensor([[49999, 49990, 17]], dtype=torch.int32, device="cuda")
    rows = _randn(1, 40, 16 + KH * 2, D, seed=2, dt=BF)
    out = kv8.write(cache, 2, rows, table, _ints([0]))
    want, _, may = _want_attention(cache, 2, rows[:, 39:, :16], table, [39], [1])
    _check(kv8.attention(cache, 2, out[:, 39:, :16], table, _ints([39])), want, may, BF)
    assert (_values(cache.k[2, 49999], cache.k_scale[2, 49999]).transpose(0, 1) - rows[0, :16, 16: 24].double()).abs().max() <= 2.0 ** -4 * rows.abs().max()


def test_more_requests_than_a_grid_is_high():
    """70000 requests of one page of eight slots, of which they have used one to eight, with weights; the last ones as much as the first."""
    from fuselink_b200.ops import kv8
    B, bs = 70000, 8
    cache = _cache(1, 100, 1, bs, 16)
    table = torch.randint(0, 100, (B, 1), generator=_gen(1), device="cuda").int()
    start = torch.arange(B, device="cuda") % bs
    q, mass = _randn(B, 1, 2, 16, seed=4, dt=BF), torch.zeros(B, 1, device="cuda")
    out = kv8.attention(cache, 0, q, table, start, mass=mass).view(B, 2, 16)
    k, v = (_values(c[0, table[:, 0].long(), 0], s[0, table[:, 0].long(), 0]) for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
    x = torch.einsum("bhd,bnd->bhn", q[:, 0].double(), k) / 4
    x = torch.where(torch.arange(bs, device="cuda") <= start[:, None, None], x, torch.full_like(x, -math.inf))
    want = torch.einsum("bhn,bnd->bhd", x.softmax(-1), v)
    # as _want_attention: weights of 11 bits, the result's rounding, scores of sums of 16 products
    assert ((out.double() - want).abs() <= (2.0 ** -11 + 2.0 ** -16) * v.abs().amax((1, 2))[:, None, None] + 2.0 ** -8 * want.abs()).all()
    assert ((mass - 2).abs() <= 2.0 ** -18).all()


# ---- eviction --------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("pages,bs,lens,keep,recent,sinks", [
    (8, 16, [128, 100, 1, 0, 17], 4, 1, 0), (145, 16, [145 * 16 - 3] * 7, 144, 4, 1), (2000, 8, [16000, 9000, 8001], 1000, 3, 2),
    (5000, 32, [160000, 77], 3, 2, 1), (9, 5, [45, 44, 41, 5], 9, 1, 0), (9, 5, [45, 44], 1, 1, 0), (12, 16, [10 ** 6, -5], 6, 1, 5), (1024, 16, [16384, 16369], 1000, 1, 1), (1025, 16, [16400, 9000], 500, 1, 1),
    (20000, 16, [320000, 250007, 131072], 9000, 2, 1),
])
@pytest.mark.parametrize("masses", ["random", "ties", "odd"])
def test_evict(pages, bs, lens, keep, recent, sinks, masses):
    from fuselink_b200.ops import kv8
    B = len(lens)
    mass = torch.exp(2 * _randn(B, pages, seed=1))
    if masses == "ties":
        mass = torch.floor(mass)
    if masses == "odd":
        pick = torch.randint(0, 6, (B, pages), generator=_gen(2), device="cuda")
        mass = torch.where(pick < 5, torch.tensor([0.0, -0.0, math.inf, -3.0, math.nan, 0.0], device="cuda")[pick], mass)
    table = _table(B, pages, B * pages)
    got = kv8.evict(mass, table, _ints(lens), bs, keep, recent=recent, sinks=sinks)
    for b, n in enumerate(lens):
        used = min(-(-max(n, 0) // bs), pages)
        extra = max(0, used - keep)
        m = mass[b].tolist()
        free = sorted(range(sinks, used - recent), key=lambda i: (m[i] != m[i], m[i] if m[i] == m[i] else 0.0, i))
        gone = sorted(free[:extra])
        out = set(gone)
        order = [i for i in range(used) if i not in out] + gone + list(range(used, pages))
        assert got[0][b].tolist() == table[b, order].tolist() and got[1][b] == n - extra * bs and got[3][b] == extra
        want = torch.where(torch.tensor([i in out for i in order], device="cuda"), torch.zeros((), device="cuda"), mass[b, order])
        assert torch.equal(got[2][b].nan_to_num(-7.0), want.nan_to_num(-7.0))


def test_evict_on_the_cpu_is_the_same():
    from fuselink_b200.ops import kv8
    mass, table, lens = torch.floor(4 * _randn(5, 40, seed=3)), _table(5, 40, 200), _ints([640, 639, 400, 0, 200])
    a = kv8.evict(mass, table, lens, 16, 11, recent=2, sinks=1)
    b = kv8.evict(mass.cpu(), table.cpu(), lens.cpu(), 16, 11, recent=2, sinks=1)
    assert all(torch.equal(x.cpu(), y) for x, y in zip(a, b))


def test_evict_of_lengths_beyond_32_bits():
    from fuselink_b200.ops import kv8
    lens = torch.tensor([2 ** 40 + 3, 2 ** 31 - 1, 2 ** 31, 2 ** 31 + 5, 0])
    for pages, bs in ((12, 16), (3, 2 ** 30), (4, 2 ** 29 + 1)):
        mass = torch.rand(5, pages, generator=torch.Generator().manual_seed(3))
        table = torch.arange(5 * pages, dtype=torch.int32).view(5, pages)
        for a, b in zip(kv8.evict(mass.cuda(), table.cuda(), lens.cuda(), bs, 2), kv8.evict(mass, table, lens, bs, 2)):
            assert torch.equal(a.cpu(), b)


# ---- together --------------------------------------------------------------------------------------------------------------------
def test_decoding_over_an_evicted_cache():
    """Prompt, weights, eviction, then new tokens behind the kept pages: what is left is attended to as by definition, and freed pages are used again."""
    from fuselink_b200.ops import kv8
    H, KH, D, bs, n = 8, 2, 64, 16, 100
    cache, table = _cache(1, 16, KH, bs, D), _table(2, 8, 16)
    rows = _randn(2, n, H + 2 * KH, D, seed=1, dt=BF)
    kv8.write(cache, 0, rows, table, _ints([0, 0]))
    mass = torch.zeros(2, 8, device="cuda")
    kv8.attention(cache, 0, rows[:, n - 1:, :H], table, _ints([n - 1] * 2), mass=mass)
    table, length, mass, gone = kv8.evict(mass, table, _ints([n] * 2), bs, 4, recent=1, sinks=1)
    assert gone.tolist() == [3, 3] and length.tolist() == [52, 52] and sorted(table.flatten().tolist()) == list(range(16))
    for step in range(20):                                             # over the end of the fourth page, into one that was given back
        new = _randn(2, 1, H + 2 * KH, D, seed=10 + step, dt=BF)
        kv8.write(cache, 0, new, table, length)
        want, weights, may = _want_attention(cache, 0, new[:, :, :H], table, length.tolist(), [1, 1])
        m = torch.zeros_like(mass)
        _check(kv8.attention(cache, 0, new[:, :, :H], table, length, mass=m), want, may, BF)
        assert ((m.double() - weights).abs() <= 1e-4 * weights + 1e-12).all()
        length = length + 1


def test_captured_calls_read_their_inputs_anew_and_share_nothing():
    """Two graphs of the same calls, replayed on two streams at once, each on a cache and inputs of its own."""
    from fuselink_b200.ops import kv8
    H, KH, D, bs, B = 8, 2, 128, 16, 3
    made = []
    for i in range(2):
        cache, table = _cache(1, 150, KH, bs, D, seed=20 * i), _table(B, 50, 150, seed=i)
        s = dict(cache=cache, table=table, rows=torch.zeros(B, 1, H + 2 * KH, D, dtype=HF, device="cuda"), start=_ints([0] * B), mass=torch.zeros(B, 50, device="cuda"))

        def step(s=s):
            out = kv8.write(s["cache"], 0, s["rows"], s["table"], s["start"])
            o = kv8.attention(s["cache"], 0, out[:, :, :H], s["table"], s["start"], mass=s["mass"])
            return (o, *kv8.evict(s["mass"], s["table"], s["start"] + 1, bs, 20))

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            s["got"] = step()
        made.append((s, g, torch.cuda.Stream()))
    for rnd in range(3):
        for i, (s, g, _) in enumerate(made):
            s["rows"].copy_(_randn(B, 1, H + 2 * KH, D, seed=rnd + 5 * i, dt=HF))
            s["start"].copy_(_ints([700 - 31 * rnd, 16 * (rnd + 1) - 1, 333]))
            s["mass"].zero_()
        torch.cuda.synchronize()
        for s, g, stream in made:
            with torch.cuda.stream(stream):
                g.replay()
        torch.cuda.synchronize()
        for s, g, _ in made:
            want, weights, may = _want_attention(s["cache"], 0, s["rows"][:, :, :H], s["table"], s["start"].tolist(), [1] * B)
            _check(s["got"][0], want, may, HF)
            assert ((s["mass"].double() - weights).abs() <= 1e-4 * weights + 1e-12).all()
            for x, y in zip(s["got"][1:], kv8.evict(s["mass"], s["table"], s["start"] + 1, bs, 20)):
                assert torch.equal(x, y)


def test_calls_that_are_refused():
    from fuselink_b200.ops import kv8
    cache, table = _cache(1, 8, 2, 16, 64), _table(2, 4, 8)
    q, qkv, start = _randn(2, 1, 4, 64, dt=BF), _randn(2, 1, 8, 64, dt=BF), _ints([5, 6])
    good = dict(cache=cache, table=table, q=q, start=start)

    def att(**kw):
        a = {**good, **kw}
        return kv8.attention(a["cache"], a.get("layer", 0), a["q"], a["table"], a["start"], counts=a.get("counts"), mass=a.get("mass"), out=a.get("out"))

    att()
    bad = [dict(q=q.float()), dict(q=_randn(2, 1, 3, 64, dt=BF)), dict(q=_randn(2, 1, 4, 80, dt=BF)), dict(table=table.long()), dict(table=table[:1]), dict(layer=1), dict(layer=-1),
           dict(start=start.int()), dict(start=start[:1]), dict(counts=start.int()), dict(start=start.cpu()), dict(mass=torch.zeros(2, 5, device="cuda")),
           dict(mass=torch.zeros(2, 4, device="cuda", dtype=torch.float64)), dict(out=torch.zeros(2, 1, 255, dtype=BF, device="cuda")), dict(out=torch.zeros(2, 1, 256, device="cuda")),
           dict(q=_randn(2, 1, 4, 128, dt=BF)[..., ::2]), dict(q=_randn(2, 1, 4, 68, dt=BF)[..., 4:]), dict(q=_randn(2, 1, 4, 65, dt=BF)[..., :64]), dict(q=q.cpu()),
           dict(cache=kv8.Kv8Cache(cache.k.float(), cache.v, cache.k_scale, cache.v_scale)), dict(cache=kv8.Kv8Cache(cache.k, cache.v, cache.k_scale.double(), cache.v_scale)),
           dict(cache=kv8.Kv8Cache(cache.k, cache.v[:, :4], cache.k_scale, cache.v_scale)), dict(cache=kv8.Kv8Cache(cache.k, cache.v, cache.k_scale[:, :4], cache.v_scale))]
    for kw in bad:
        with pytest.raises(RuntimeError):
            att(**kw)
    wide = _cache(1, 2, 1, 16, 144)
    with pytest.raises(RuntimeError):
        kv8.attention(wide, 0, _randn(2, 1, 1, 144, dt=BF), table, start)
    for kw in (dict(qkv=_randn(2, 1, 3, 64, dt=BF)), dict(qkv=qkv.float()), dict(bias=torch.zeros(8 * 64 - 8, dtype=BF, device="cuda")), dict(rope=torch.zeros(20, 32, device="cuda")),
               dict(rope=torch.zeros(20, 64, dtype=BF, device="cuda")), dict(positions=start[:1]), dict(out=torch.zeros(2, 1, 8, 32, dtype=BF, device="cuda"))):
        a = dict(qkv=qkv, **{k: v for k, v in kw.items() if k != "qkv"})
        a.update(kw)
        x = a.pop("qkv")
        with pytest.raises(RuntimeError):
            kv8.write(cache, 0, x, table, start, **a)
    for kw in (dict(keep=1, recent=1, sinks=1), dict(keep=2, recent=0), dict(keep=2, sinks=-1)):
        with pytest.raises(ValueError):
            kv8.evict(torch.zeros(2, 4, device="cuda"), table, start, 16, **kw)
    with pytest.raises(RuntimeError):
        kv8.evict(torch.zeros(2, 5, device="cuda"), table, start, 16, 2)
    empty = kv8.attention(cache, 0, q[:0], table[:0], start[:0])
    assert empty.shape == (0, 1, 256) and kv8.attention(cache, 0, q[:, :0], table, start).shape == (2, 0, 256)
    assert [t.shape[0] for t in kv8.evict(torch.zeros(0, 4, device="cuda"), table[:0], start[:0], 16, 2)] == [0, 0, 0, 0]


@pytest.mark.parametrize("where", [2 ** 63 - 1, 2 ** 63 - 3, 2 ** 62, 2 ** 31 - 1, -2 ** 63])
def test_slots_and_positions_at_the_ends_of_64_bits(where):
    """Slots that are none of the table's are written nowhere and noted, rotations that are not there are left out and noted, however far away; an
    attention from behind the table sees all of it."""
    from fuselink_b200.ops import kv8
    cache, table = _cache(1, 8, 2, 16, 64), _table(2, 3, 8)
    x, rope = _randn(2, 20, 8, 64, seed=3, dt=BF), torch.full((90, 64), 2.0, device="cuda")
    before, word = [t.clone() for t in cache.tensors()], torch.zeros(1, dtype=torch.int32).pin_memory()
    out = kv8.write(cache, 0, x, table, _ints([where, 47]), positions=_ints([0, where]), counts=_ints([20, 0]), status=word.data_ptr())
    torch.cuda.synchronize()
    assert int(word) == 2 and torch.equal(out, x)
    for a, b in zip(before, cache.tensors()):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    word.zero_()
    out = kv8.write(cache, 0, x, table, _ints([3, 20]), positions=_ints([where, where]), rope=rope, status=word.data_ptr())
    torch.cuda.synchronize()
    assert int(word) == 2 and torch.equal(out, x)
    q = x[:, :5, :4]
    got = kv8.attention(cache, 0, q, table, _ints([where, 30]), counts=_ints([5, 2]))
    if where < 0:
        assert got[0].abs().max() == 0
    else:
        assert torch.equal(got, kv8.attention(cache, 0, q, table, _ints([48, 30]), counts=_ints([5, 2])))


@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("heads,kv_heads,tokens,lens", [(8, 2, 4, [200, 130]), (4, 1, 9, [3000, 40]), (64, 8, 2, [100, 5])])
def test_what_stands_in_padding_reaches_no_pages_weight(heads, kv_heads, tokens, lens, what):
    """Rows behind a request's count are whatever they are: outputs and weights as with any others, and eviction sees numbers.  So are rows of tokens before slot 0."""
    from fuselink_b200.ops import kv8
    each = max(lens) // 16 + 2
    cache, table = _cache(1, 2 * each, kv_heads, 16, 64), _table(2, each, 2 * each)
    q = _randn(2, tokens, heads, 64, seed=4, dt=BF)
    counts, got = [1, tokens - 1], []
    start = [n - c for n, c in zip(lens, counts)]
    for fill in (0.5, what):
        for b, c in enumerate(counts):
            q[b, c:] = fill
        mass = torch.zeros(2, each, device="cuda")
        got.append((kv8.attention(cache, 0, q, table, _ints(start), counts=_ints(counts), mass=mass), mass))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
    want, weights, may = _want_attention(cache, 0, q, table, start, counts)
    _check(got[1][0], want, may, BF)
    assert ((got[1][1].double() - weights).abs() <= 1e-4 * weights + 1e-12).all()
    q[:] = _randn(2, tokens, heads, 64, seed=5, dt=BF)
    q[:, :tokens - 1] = what                                           # all but the last, which sees slot 0
    mass = torch.zeros(2, each, device="cuda")
    out = kv8.attention(cache, 0, q, table, _ints([1 - tokens] * 2), mass=mass)
    want, weights, may = _want_attention(cache, 0, q, table, [1 - tokens] * 2, [tokens] * 2)
    _check(out, want, may, BF)
    assert (mass[:, 0] - heads).abs().max() <= 1e-4 and mass[:, 1:].abs().max() == 0


@pytest.mark.parametrize("heads,kv_heads,dim,bs,tokens", [(4, 2, 64, 16, 1), (8, 2, 128, 16, 1), (16, 2, 128, 16, 1), (12, 1, 80, 16, 1), (2, 2, 64, 8, 3), (8, 1, 128, 5, 2), (8, 2, 128, 32, 4)])
@pytest.mark.parametrize("apart", [12, 20, 30, -30, 60])
@pytest.mark.parametrize("nats", [0.0, 7.0, 14.0, 40.0])
def test_values_of_different_magnitude(heads, kv_heads, dim, bs, tokens, apart, nats):
    """Every third page has values 2^apart times the others', and scores `nats` below theirs: what such a page has no weight for takes nothing from the others."""
    from fuselink_b200.ops import kv8
    lens = [37 * bs, 5 * bs + 2, 3 * bs]
    batch, each, dt = len(lens), 37, HF
    cache, table = _cache(1, batch * each, kv_heads, bs, dim, spread=0.3), _table(batch, each, batch * each)
    q = _randn(batch, tokens, heads, dim, seed=4).abs().to(dt)
    # in the far pages every key has -nats for a score: -nats / (scale sum q) in all columns, as near as a code comes to it
    far = torch.zeros(batch * each, dtype=torch.bool, device="cuda")
    far[table[:, torch.arange(each, device="cuda") % 3 == 1].flatten().long()] = True
    key = torch.tensor(-nats / (dim ** 0.5 * 0.8), device="cuda").to(F8)
    cache.k[0, far], cache.k_scale[0, far] = key, 1.0
    cache.v_scale[0, far] *= 2.0 ** apart
    start = [n - tokens for n in lens]
    mass = torch.zeros(batch, each, device="cuda")
    out = kv8.attention(cache, 0, q, table, _ints(start), mass=mass)
    assert torch.equal(out, kv8.attention(cache, 0, q, table, _ints(start)))
    for b in range(batch):
        pages = table[b].long()
        k, v = (_values(c[0][pages], s[0][pages]).transpose(0, 1).reshape(kv_heads, -1, dim).repeat_interleave(heads // kv_heads, 0) for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
        scale = cache.v_scale[0][pages].double().transpose(0, 1).repeat_interleave(bs, 1).repeat_interleave(heads // kv_heads, 0)      # [heads, slots]
        for t in range(tokens):
            seen = start[b] + t + 1
            qq = q[b, t].double()
            p = (torch.einsum("hd,hnd->hn", qq, k[:, :seen]) * dim ** -0.5).softmax(-1)
            want = torch.einsum("hn,hnd->hd", p, v[:, :seen])
            # Weights are cut to 11 bits, off by 0 to 2^-10 each: what that has in common cancels against their sum, and 2^-11 to either side of it is left
            # of the differences between values and output, whose weighed magnitudes are at most twice the values'.  As halves they come in steps of 2^-24
            # where the largest product of a weight and its page's scale is 2^2 at least: 2^-26 of that for each code of at most 448.  Scores and sums over the
            # tokens in fp32 as in _want_attention.
            size = (torch.einsum("hd,hnd->hn", qq.abs(), k[:, :seen].abs()) * dim ** -0.5).amax(-1)
            relative = 2.0 ** -10 + 2 * (dim + 6) * 2.0 ** -23 * size + (seen + 8) * 2.0 ** -23
            may = relative[:, None] * torch.einsum("hn,hnd->hd", p, v[:, :seen].abs()) + (seen * 2.0 ** -26 * 448 * (p * scale[:, :seen]).amax(-1))[:, None]
            got = out[b, t].view(heads, dim).double()
            there = want.abs() < 65000.0                               # beyond fp16 there is infinity
            off = (got - want).abs() - may - 2.0 ** -11 * want.abs() * 1.01 - 2.0 ** -25
            assert (off[there] <= 0).all(), (b, t, off[there].max().item())
    assert (mass.sum(1) - heads * tokens).abs().max() <= 1e-4 * heads * tokens


def test_a_batch_that_goes_in_pieces():
    """Weights of 70 requests of 64 heads with tables of 8192 pages: more than one piece's scratch; the last request as much as the first."""
    from fuselink_b200.ops import kv8
    B, H, KH, D, each = 70, 64, 8, 16, 8192
    cache = _cache(1, 400, KH, 16, D)
    table = torch.randint(0, 400, (B, each), generator=_gen(1), device="cuda").int()
    lens = [1 + (37 * b) % 90 for b in range(B)]
    q, mass = _randn(B, 1, H, D, seed=4, dt=HF), torch.zeros(B, each, device="cuda")
    word = torch.zeros(1, dtype=torch.int32).pin_memory()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    out = kv8.attention(cache, 0, q, table, _ints(lens) - 1, mass=mass, status=word.data_ptr())
    assert torch.cuda.max_memory_allocated() - before <= (1 << 28) + 2 * out.nbytes
    want, weights, may = _want_attention(cache, 0, q, table[:, :6], [n - 1 for n in lens], [1] * B)
    _check(out, want, may, HF)
    assert ((mass[:, :6].double() - weights).abs() <= 1e-4 * weights + 1e-12).all() and mass[:, 6:].abs().max() == 0 and int(word) == 0


def test_gradients_are_refused():
    from fuselink_b200.ops import kv8
    cache, table, start = _cache(1, 8, 2, 16, 64), _table(2, 4, 8), _ints([5, 6])
    q, qkv = _randn(2, 1, 4, 64, dt=BF).requires_grad_(), _randn(2, 1, 8, 64, dt=BF).requires_grad_()
    bias = _randn(8 * 64, dt=BF).requires_grad_()
    for call in (lambda: kv8.attention(cache, 0, q, table, start), lambda: kv8.write(cache, 0, qkv, table, start), lambda: kv8.write(cache, 0, qkv.detach(), table, start, bias=bias)):
        with pytest.raises(RuntimeError, match="gradient"):
            call()
        with torch.no_grad():
            call()
