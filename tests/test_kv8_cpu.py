"""The cache in 8 bits and sampling without a GPU: plain forms, the decoder's routes over them, serving stages, refusals of the C entries."""
import ctypes
import math
import os

import pytest
import torch

from fuselink_b200.models import llama
from fuselink_b200.models.llama import MODEL_ZOO, LlamaShard
from fuselink_b200.ops import kv8
from fuselink_b200.ops.sampling import Sampler, sample
from test_decoder_route_cpu import FUSED, PLAIN, _net, _tokens, route  # noqa: F401 - the fixture
from test_kernel_model_cpu import _run_script_on_model

FAMILIES = ["tiny", "tiny_opt", "tiny_gpt2"]


def _cache(cfg, blocks):
    return kv8.Kv8Cache.empty(cfg.layers, blocks, cfg.kv_heads, cfg.block_size, cfg.head_dim, device="cpu")


def _table(batch, each, seed=1):
    return torch.randperm(batch * each, generator=torch.Generator().manual_seed(seed)).view(batch, each).int()


# ---- plain forms ------------------------------------------------------------------------------------------------------------------
def test_a_written_page_holds_its_values_to_half_a_step():
    g = torch.Generator().manual_seed(1)
    cache = kv8.Kv8Cache.empty(1, 3, 2, 16, 64, device="cpu")
    rows = torch.randn(1, 20, 6, 64, generator=g) * 10 ** torch.randn(1, 20, 6, 1, generator=g)
    table = torch.tensor([[2, -3]], dtype=torch.int32)
    assert torch.equal(kv8.write(cache, 0, rows, table, torch.tensor([5])), rows)
    for codes, scales, head in ((cache.k, cache.k_scale, 2), (cache.v, cache.v_scale, 4)):
        got = kv8.dequantize(codes[0, [2, 0]], scales[0, [2, 0]]).transpose(0, 1).reshape(2, 32, 64)[:, 5:25]
        want = rows[0, :, head: head + 2].transpose(0, 1)
        step = scales[0, [2, 0]].repeat_interleave(16, 0)[5:25].t()[..., None]
        assert ((got - want).abs() <= 2.0 ** -4 * want.abs() + 2.0 ** -10 * step).all()
        amax = torch.stack([want[:, :11].abs().amax((1, 2)), want[:, 11:].abs().amax((1, 2))])
        # the first page had five tokens before, whose scale of 1 it keeps or raises
        assert (amax <= 448 * scales[0, [2, 0]]).all() and (amax[1] > 224 * scales[0, 0]).all() and (scales[0, 2] >= 1).all()


def test_one_token_at_a_time_ends_where_a_run_does():
    """Scales of a page grow to what a run of its tokens gives at once; the codes differ by what the smaller scales' roundings did."""
    g = torch.Generator().manual_seed(2)
    rows = torch.randn(1, 16, 3, 32, generator=g) * 1.7 ** torch.arange(16)[None, :, None, None]
    table = torch.zeros(1, 1, dtype=torch.int32)
    a, b = (kv8.Kv8Cache.empty(1, 1, 1, 16, 32, device="cpu") for _ in range(2))
    kv8.write(a, 0, rows, table, torch.tensor([0]))
    for t in range(16):
        kv8.write(b, 0, rows[:, t: t + 1], table, torch.tensor([t]))
    assert torch.equal(a.k_scale, b.k_scale) and torch.equal(a.v_scale, b.v_scale)
    x, y = kv8.dequantize(a.k, a.k_scale), kv8.dequantize(b.k, b.k_scale)
    assert ((x - y).abs() <= 2.0 ** -9 * a.k_scale).all()                # one step of the smallest numbers


def test_evict_refuses_and_keeps_order():
    mass = torch.tensor([[5.0, 1.0, 1.0, 0.5, 9.0, 2.0, 7.0]])
    table = torch.tensor([[10, 11, 12, 13, 14, 15, 16]], dtype=torch.int32)
    t, n, m, gone = kv8.evict(mass, table, torch.tensor([6 * 16 - 3]), 16, 4, recent=1, sinks=0)
    assert t.tolist() == [[10, 12, 14, 15, 11, 13, 16]] and n.tolist() == [61] and m.tolist() == [[5.0, 1.0, 9.0, 2.0, 0.0, 0.0, 7.0]] and gone.tolist() == [2]
    assert table.tolist() == [[10, 11, 12, 13, 14, 15, 16]]              # inputs stay as they are
    for kw in (dict(keep=2, recent=1, sinks=2), dict(keep=2, recent=0), dict(keep=3, sinks=-1)):
        with pytest.raises(ValueError):
            kv8.evict(mass, table, torch.tensor([90]), 16, **kw)


def test_indices_outside_are_errors():
    cache = kv8.Kv8Cache.empty(1, 4, 1, 16, 32, device="cpu")
    rows, table = torch.randn(1, 2, 3, 32), torch.tensor([[0, 4]], dtype=torch.int32)
    for start in (-1, 31, 15):                                         # before the cache, behind it, into a page outside the pool
        with pytest.raises(IndexError):
            kv8.write(cache, 0, rows, table, torch.tensor([start]))
    with pytest.raises(IndexError):
        kv8.write(cache, 0, rows, table, torch.tensor([0]), rope=torch.zeros(1, 32))
    with pytest.raises(IndexError):
        kv8.attention(cache, 0, rows[:, :, :1], table, torch.tensor([20]))
    with pytest.raises(ValueError):
        kv8.attention(cache, 0, rows[:, :, :1], table, torch.tensor([3]), scale=-1.0)
    with pytest.raises(IndexError):
        kv8.pack(cache, torch.zeros(4 * 16 * 32), torch.zeros(4 * 16 * 32), 4, table, table, torch.tensor([40]))


@pytest.mark.parametrize("limits,left", [((1.0, 0, 1.0, 0.0), 6), ((1.0, 3, 1.0, 0.0), 3), ((1.0, 0, 0.6, 0.0), 2), ((1.0, 0, 1.0, 0.12), 5), ((1.0, 4, 0.9, 0.3), 2), ((1.0, 0, 0.0, 0.0), 1),
                                         ((0.0, 0, 1.0, 0.0), 1), ((0.5, 0, 1.0, 0.1), 2)])
def test_sample_by_hand(limits, left):
    """Probabilities 0.5, 0.2, 0.1, 0.1, 0.06, 0.04: which tokens are left, and the logarithms over them.  (Limits are fp32: 0.06 / 0.5 is above the
    0.12 that they hold.)"""
    p = torch.tensor([0.1, 0.06, 0.5, 0.04, 0.1, 0.2], dtype=torch.float64)
    order = [2, 5, 0, 4, 1, 3]
    x = p.log().expand(400, 6)
    u = (torch.arange(400, dtype=torch.float64) + 0.5) / 400
    tokens, logprobs = sample(x, u, *limits)
    q = p[order[:left]] ** (1 / limits[0] if limits[0] else 1.0)
    if left == 1:
        q = torch.ones(1, dtype=torch.float64)
    q = q / q.sum()
    assert set(tokens.tolist()) == set(order[:left])
    for i, t in enumerate(order[:left]):
        assert abs(int((tokens == t).sum()) - 400 * float(q[i])) <= 1
        assert (logprobs[tokens == t].double() - q[i].log()).abs().max() <= 1e-6


def test_sample_refuses():
    x, u = torch.randn(3, 10), torch.rand(3)
    for a in ((x[0], u), (x[:, :0], u), (x, u[:2]), (x, u.half()), (x, u, torch.ones(2)), (x, u, 1.0, torch.ones(4))):
        with pytest.raises(ValueError):
            sample(*a)


# ---- the decoder ----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("model", FAMILIES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_routes_over_a_small_cache_agree(model, dtype, route):  # noqa: F811
    """Prompt, single tokens and a piece of several, by the fused passes and by the operations: tokens, codes, weights of pages."""
    net = _net(model, dtype)
    cfg, res = net.cfg, []
    toks = _tokens(net, 3, 48)
    table = _table(3, 6)
    for r in (FUSED, PLAIN):
        if r == FUSED and dtype == torch.float32:
            continue
        route(r)
        cache = _cache(cfg, 18)
        mass = torch.zeros(3, 6)
        first = net.prefill(toks, cache, None, table, last_pos=torch.tensor([47, 20, -1]))
        pos = torch.tensor([48, 21, 48])
        got = [first]
        for _ in range(2):
            got.append(net.extend(got[-1], pos, cache, table, mass=mass))
            pos = pos + 1
        piece = _tokens(net, 3, 5)
        got.append(net.extend(piece, pos, cache, table, counts=torch.tensor([5, 0, 2]), mass=mass))
        res.append((torch.cat([got[0], got[1], got[2], got[3][0], got[3][2, :2]]), cache, mass))
    (a, ca, ma), (b, cb, mb) = res[0], res[-1]
    assert torch.equal(a, b)
    assert torch.allclose(ma.sum(1), torch.tensor([7.0, 2.0, 4.0]) * cfg.layers * cfg.heads, rtol=1e-4)       # a weight of 1 per token, head and layer
    assert (ma - mb).abs().max() <= 0.05 * ma.max()
    for s, t in ((ca.k_scale, cb.k_scale), (ca.v_scale, cb.v_scale)):
        used = table[[0, 0, 0, 0, 1, 1, 2, 2, 2, 2], [0, 1, 2, 3, 0, 1, 0, 1, 2, 3]].long()
        assert (s[:, used] == t[:, used]).float().mean() > 0.95           # a rounding may tip a largest value over


@pytest.mark.parametrize("model", FAMILIES)
def test_a_small_cache_follows_the_dense_model(model):
    """Greedy tokens from 8-bit pages are those of the model without a cache, where the winners win by a margin."""
    net = _net(model, torch.float32)
    toks, table, cache = _tokens(net, 2, 32), _table(2, 4), _cache(net.cfg, 8)
    t = net.prefill(toks, cache, None, table)
    seq = toks
    for i in range(4):
        assert torch.equal(t, net.forward_dense(seq).argmax(-1))
        seq = torch.cat([seq, t[:, None]], 1)
        t = net.extend(t, torch.full((2,), 32 + i), cache, table)


def test_several_tokens_at_once_are_one_after_the_other():
    """Pieces of 7 against single tokens, in slots that are not the positions."""
    net = _net("tiny", torch.float32)
    toks, table = _tokens(net, 2, 16), _table(2, 3)
    piece = _tokens(net, 2, 7)
    res = []
    for step in (7, 1):
        cache = _cache(net.cfg, 6)
        net.prefill(toks, cache, None, table)
        res.append(torch.cat([net.extend(piece[:, i: i + step], torch.full((2,), 40 + i), cache, table, slots=torch.full((2,), 16 + i)) for i in range(0, 7, step)], 1))
    assert torch.equal(res[0], res[1])


@pytest.mark.parametrize("r", [FUSED, PLAIN])
def test_tokens_by_chance(r, route):  # noqa: F811
    """Prompt, 16-bit step and 8-bit step draw from the logits of the greedy choice; a temperature of 0 is that choice."""
    net = _net("tiny")
    route(r)
    bs, D, kl, L = net.cfg.block_size, net.cfg.head_dim, net.cfg.kv_heads, net.cfg.layers
    toks, table = _tokens(net, 3, 32), _table(3, 3)
    n = 9 * L * kl * bs * D
    seen = []

    def spy(logits):
        assert logits.shape == (3, net.cfg.vocab) and logits.dtype == net.embed.dtype
        seen.append(logits)
        return Sampler(torch.full((3,), 0.999), temperature=50.0)(logits)

    def pools():
        return [torch.zeros(n, dtype=net.embed.dtype) for _ in range(2)]

    def small():
        cache = _cache(net.cfg, 9)
        net.prefill(toks, cache, None, table)
        return cache

    new, pos = torch.tensor([1, 2, 3]), torch.full((3,), 32)
    for call in (lambda c: net.prefill(toks, *pools(), table, choose=c), lambda c: net.decode_step(new, pos, *pools(), table, 9, choose=c),
                 lambda c: net.extend(new, pos, small(), table, choose=c)):
        greedy = call(None)
        assert torch.equal(call(Sampler(torch.rand(3), temperature=0.0)), greedy)
        drawn = call(spy)
        assert torch.equal(seen[-1].float().argmax(-1), greedy) and not torch.equal(drawn, greedy)


def test_a_cache_of_another_model_is_an_error():
    net = _net("tiny")
    cache = kv8.Kv8Cache.empty(2, 8, 4, 16, 64, device="cpu")           # four KV heads, the model has two
    with pytest.raises(RuntimeError, match="cache of"):
        net.extend(torch.tensor([1]), torch.tensor([0]), cache, torch.zeros(1, 2, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="cache of"):
        net.prefill(torch.zeros(1, 16, dtype=torch.long), cache, None, torch.zeros(1, 1, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="block table"):
        net.extend(torch.tensor([1]), torch.tensor([0]), _cache(net.cfg, 2), torch.zeros(2, 2, dtype=torch.int32))


# ---- serving --------------------------------------------------------------------------------------------------------------------
def test_options_that_do_not_go_together():
    from fuselink_b200.serving.disagg import ServeParams
    for kw in (dict(kv_bits=4), dict(keep_blocks=8), dict(kv_bits=8, keep_blocks=2)):
        with pytest.raises(ValueError):
            ServeParams(MODEL_ZOO["tiny"], **kw).check()
    p = ServeParams(MODEL_ZOO["tiny"], kv_bits=8, keep_blocks=3, temperature=0.5, top_k=4)
    p.check()
    assert p.sampler(2, "cpu").top_k == 4 and ServeParams(MODEL_ZOO["tiny"]).sampler(2, "cpu") is None


OPTIONS = ["--kv-bits", "8", "--keep-blocks", "4", "--temperature", "0.8", "--top-k", "50", "--top-p", "0.95", "--min-p", "0.01"]


def test_serving_benchmark_over_a_small_cache():
    rows = _run_script_on_model("bench/serving_bench.py", ["--device", "cpu", "--model", "tiny", "--emulate", "--batch", "2", "--input-len", "96", "--decode-steps", "40", "--iters", "1", *OPTIONS])
    assert rows and rows[-1]["decode_tok_s"] > 0


def test_online_serving_over_a_small_cache():
    rows = _run_script_on_model("experiments/run_online_serving.py", ["--device", "cpu", "--model", "tiny", "--requests", "6", "--rate", "300", "--input-len", "96",
                                                                      "--decode-steps", "18", *OPTIONS])
    assert [r for r in rows if "served" in r][0]["served"] == 6


# ---- C entries ------------------------------------------------------------------------------------------------------------------
P, I, LL, F32 = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_float


class Kv8(ctypes.Structure):
    _fields_ = [(n, P) for n in ("k", "v", "k_scale", "v_scale", "block_table")] + [(n, I) for n in ("table_stride", "layer", "layers", "num_blocks", "block_size", "heads", "dim")] + [("status", P)]


class Sample(ctypes.Structure):
    _fields_ = [("logits", P), ("row_stride", LL), ("rows", I), ("vocab", LL), ("u64", P), ("u32", P), ("temperature", P), ("temperature_all", F32), ("top_k", P), ("top_k_all", I),
                ("top_p", P), ("top_p_all", F32), ("min_p", P), ("min_p_all", F32), ("tokens", P), ("logprobs", P)]


def _kv(k=0x100000, v=0x100000, stride=4, layer=0, layers=1, blocks=8, bs=16, heads=2, dim=64):
    return ctypes.byref(Kv8(k, v, 0x2000, 0x3000, 0x4000, stride, layer, layers, blocks, bs, heads, dim, None))


@pytest.fixture(scope="module")
def lib():
    from fuselink_b200 import build
    so = ctypes.CDLL(os.path.join(build.LIB, "libfuselink.so"))
    so.fl_kv8_attention_scratch.restype = LL
    return so


A0 = 0x100000


def test_c_entries_refuse_addresses(lib):
    def write(p):
        return lib.fl_kv8_write(I(0), P(p[0]), P(p[1]), P(p[2]), P(p[3]), LL(9), P(8), P(8), P(8), I(0), I(1), I(4), _kv(p[4], p[5]), P())

    def attend(p):
        return lib.fl_kv8_attention(I(0), P(p[0]), LL(64), LL(64), LL(64), P(8), P(), I(0), I(1), I(4), F32(1), _kv(p[1], p[2]), P(p[3]), P(), P(p[4]), P())

    def pack(p):
        return lib.fl_kv8_pack(I(0), P(p[0]), P(p[1]), I(4), P(8), I(4), P(8), I(0), _kv(p[2], p[3]), P())

    for n, call in ((6, write), (5, attend), (4, pack)):
        assert call([A0] * n) == 0                                       # nothing is launched for an empty batch
        for i in range(n):
            for off in (2, 4, 8):
                assert call([A0 + (off if k == i else 0) for k in range(n)]) == -4


@pytest.mark.parametrize("kw", [dict(dim=8), dict(dim=72), dict(dim=144), dict(heads=0), dict(bs=0), dict(blocks=-1), dict(layer=1), dict(layer=-1), dict(layers=0), dict(stride=-1),
                                dict(stride=1 << 30)])
def test_c_entries_refuse_caches(lib, kw):
    kv = _kv(**kw)
    assert lib.fl_kv8_write(I(0), P(A0), P(A0), P(), P(), LL(0), P(8), P(), P(), I(1), I(1), I(4), kv, P()) == -2
    assert lib.fl_kv8_attention(I(0), P(A0), LL(64), LL(64), LL(64), P(8), P(), I(1), I(1), I(4), F32(1), kv, P(A0), P(), P(A0), P()) == -2
    if "layer" not in kw:
        assert lib.fl_kv8_pack(I(0), P(A0), P(A0), I(4), P(8), I(4), P(8), I(1), kv, P()) == -2
        assert lib.fl_kv8_attention_scratch(I(1), I(1), I(4), kv, I(1)) == 0


def test_c_entries_refuse_sizes(lib):
    def attend(dtype=0, strides=(64, 64, 64), batch=1, tokens=1, heads=4, mass=None, scale=1.0):
        return lib.fl_kv8_attention(I(dtype), P(A0), *map(LL, strides), P(8), P(), I(batch), I(tokens), I(heads), F32(scale), _kv(), P(A0), P(mass), P(A0), P())

    for kw in (dict(strides=(4, 64, 64)), dict(strides=(64, 60, 64)), dict(strides=(64, 64, 65)), dict(batch=-1), dict(tokens=-1), dict(heads=3), dict(heads=0),
               dict(tokens=1 << 30), dict(tokens=4000, mass=8), dict(scale=-1.0), dict(scale=math.inf), dict(scale=math.nan)):
        assert attend(**kw) == -2
    assert attend(dtype=7) == -1 and attend(batch=0) == 0 and attend(tokens=0) == 0
    assert lib.fl_kv8_write(I(7), P(A0), P(A0), P(), P(), LL(0), P(8), P(), P(), I(1), I(1), I(4), _kv(), P()) == -1
    for batch, tokens, heads in ((-1, 1, 4), (1, -1, 4), (1, 1, -1), (1, 1 << 30, 4)):
        assert lib.fl_kv8_write(I(0), P(A0), P(A0), P(), P(), LL(0), P(8), P(), P(), I(batch), I(tokens), I(heads), _kv(), P()) == -2

    def evict(batch=1, pages=4, bs=16, keep=2, recent=1, sinks=1):
        return lib.fl_kv8_evict(P(8), P(8), P(8), I(batch), I(pages), I(bs), I(keep), I(recent), I(sinks), P(8), P(8), P(8), P(8), P())

    for kw in (dict(batch=-1), dict(pages=-1), dict(bs=0), dict(keep=1), dict(recent=0), dict(sinks=-1), dict(recent=2 ** 31 - 1, sinks=2 ** 31 - 1)):
        assert evict(**kw) == -2
    assert evict(batch=0) == 0

    def draw(dtype=0, logits=A0, rows=0, vocab=10, u64=None, u32=8):
        return lib.fl_sample(I(dtype), ctypes.byref(Sample(logits, vocab, rows, vocab, u64, u32, None, 1.0, None, 0, None, 1.0, None, 0.0, 8, 8)), P())

    assert draw() == 0
    for kw in (dict(rows=-1), dict(vocab=0), dict(vocab=8 * 65528 + 1), dict(rows=1, logits=None), dict(u64=8), dict(u32=None)):
        assert draw(**kw) == -2
    assert draw(dtype=3) == -1


def test_scratch_covers_every_part(lib):
    """Outputs and sums of every row and chunk, sums of every unit if weights are asked for."""
    for batch, tokens, heads, stride in ((1, 1, 8, 4), (2, 1, 32, 8192), (3, 5, 16, 100), (64, 1, 8, 512)):
        kv = _kv(stride=stride, heads=8, dim=128)
        plain, mass = (lib.fl_kv8_attention_scratch(I(batch), I(tokens), I(heads), kv, I(m)) for m in (0, 1))
        assert plain % 16 == 0 and mass >= plain + 8 * batch * tokens * heads * stride
    assert math.isfinite(plain)


def test_c_entries_refuse_pages_beyond_32_bits(lib):
    """Places in a page are 32-bit numbers."""
    for dim, bs, stride in ((16, 1 << 27, 1), (128, 1 << 24, 2), (64, (1 << 31) - 1, 0)):
        kv = _kv(bs=bs, dim=dim, stride=stride)
        assert lib.fl_kv8_write(I(0), P(A0), P(A0), P(), P(), LL(0), P(8), P(), P(), I(1), I(1), I(4), kv, P()) == -2
        assert lib.fl_kv8_attention(I(0), P(A0), LL(64), LL(64), LL(64), P(8), P(), I(1), I(1), I(4), F32(1), kv, P(A0), P(), P(A0), P()) == -2
        assert lib.fl_kv8_pack(I(0), P(A0), P(A0), I(4), P(8), I(4), P(8), I(1), kv, P()) == -2
    assert lib.fl_kv8_write(I(0), P(A0), P(A0), P(), P(), LL(0), P(8), P(), P(), I(0), I(1), I(4), _kv(bs=1 << 24, dim=64, stride=2), P()) == 0


@pytest.mark.parametrize("online", [False, True])
@pytest.mark.parametrize("seed", [0, 5, -1, 2 ** 63 - 1])
def test_every_token_is_drawn_by_numbers_of_its_own(online, seed, monkeypatch):
    """First tokens and the following ones come from two stages; what one draws by, the other does not."""
    import cpu_kernel_model
    from fuselink_b200.parallel.symm import SymmetricHeap
    from fuselink_b200.serving.disagg import DecodeStage, KVLink, PrefillStage, ServeParams, make_prompts
    from fuselink_b200.serving.online import OnlineDecode, OnlinePrefill, Request
    p = ServeParams(model=MODEL_ZOO["tiny"], batch_size=3, input_len=32, num_decoding_step=4, temperature=1.0, seed=seed)
    seen, call = [], Sampler.__call__
    monkeypatch.setattr(Sampler, "__call__", lambda self, logits: (seen.append(self.u.clone()), call(self, logits))[1])
    heaps = SymmetricHeap.emulated(2, 32 << 20)
    try:
        with cpu_kernel_model.installed():
            net = LlamaShard(p.model, device="cpu", seed=1)
            if online:
                links = [[KVLink(h, p, net.kvh_local, name=f"kv{i}") for i in range(2)] for h in heaps]
                pre, dec = OnlinePrefill(p, net, links[0], dst_rank=1), OnlineDecode(p, net, links[1], src_rank=0)
                for batch in range(2):
                    pre.serve_batch([Request(0.0, 20, 20, 4) for _ in range(3)])
                    dec.serve_batch(4)
            else:
                links = [KVLink(h, p, net.kvh_local) for h in heaps]
                pre, dec = PrefillStage(p, net, links[0], dst_rank=1), DecodeStage(p, net, links[1])
                for batch in range(2):
                    pre.run(make_prompts(p, "cpu", seed=3))
                    dec.run()
    finally:
        for h in heaps:
            h.close()
    assert len(seen) == 2 * (1 + 4) and torch.cat(seen).unique().numel() == 2 * (1 + 4) * 3


def test_scratch_is_bounded(lib):
    """A large batch with a wide table goes in pieces that share their scratch: what one request needs, or 256 MiB."""
    for batch, tokens, heads, stride in ((64, 8, 64, 8192), (65535, 1, 64, 8192), (70000, 4, 8, 1000), (65535, 1, 64, 65535), (3, 96, 64, 8192)):
        kv = _kv(stride=stride, heads=8, dim=128)
        for mass in (0, 1):
            one, all_ = (lib.fl_kv8_attention_scratch(I(b), I(tokens), I(heads), kv, I(mass)) for b in (1, batch))
            assert 0 <= all_ <= max(1 << 28, one)


def test_options_that_the_gpu_does_not_take():
    """Known before a batch is on its way: types, heads and vocabularies that only the plain forms take."""
    import dataclasses
    from fuselink_b200.serving.disagg import ServeParams
    tiny = MODEL_ZOO["tiny"]
    odd, wide = dataclasses.replace(tiny, head_dim=72), dataclasses.replace(tiny, vocab=600000)
    bad = [(tiny, dict(kv_bits=8, dtype=torch.float32)), (tiny, dict(temperature=0.5, dtype=torch.float32)), (odd, dict(kv_bits=8)), (wide, dict(temperature=1.0))]
    for model, kw in bad:
        p = ServeParams(model, **kw)
        p.check()
        p.check("cpu")
        with pytest.raises(ValueError):
            p.check("cuda")
    for model, kw in ((tiny, dict(dtype=torch.float32)), (odd, dict(temperature=1.0)), (wide, dict(kv_bits=8)), (tiny, dict(kv_bits=8, temperature=1.0, dtype=torch.float16))):
        ServeParams(model, **kw).check(torch.device("cuda", 0))


@pytest.mark.parametrize("model", FAMILIES)
@pytest.mark.parametrize("r", [FUSED, PLAIN])
@pytest.mark.parametrize("shape", [(3,), (3, 1), (3, 2)])
def test_a_padded_row_has_no_position(model, r, shape, route):  # noqa: F811
    """A batch with a request that has no new token: whatever its position says, single tokens and pieces alike, the others go on as without it."""
    net = _net(model)
    route(r)
    toks, table = _tokens(net, 3, 32), _table(3, 4)
    new, got = _tokens(net, 3, 2)[:, :1 if len(shape) == 1 else shape[1]].reshape(shape), []
    for where in (32, 10 ** 7):
        cache = _cache(net.cfg, 12)
        net.prefill(toks, cache, None, table)
        positions = torch.tensor([32, where, 32])
        out = net.extend(new, positions, cache, table, slots=torch.tensor([32, 32, 32]), counts=torch.tensor([len(new[0].reshape(-1)), 0, 1]))
        got.append((out.view(3, -1)[[0, 2], 0], *(scales[:, table[[0, 2], :3].long()] for scales in (cache.k_scale, cache.v_scale))))
    assert all(torch.equal(a, b) for a, b in zip(*got))


@pytest.mark.parametrize("r", [FUSED, PLAIN])
@pytest.mark.parametrize("shape", [(3,), (3, 4)])
def test_what_stands_behind_counts_is_no_token(r, shape, route):  # noqa: F811
    """Padding need not be an entry of the vocabulary."""
    net = _net("tiny")
    route(r)
    toks, table, counts = _tokens(net, 3, 32), _table(3, 4), torch.tensor([1, 0, 1])
    new, got = _tokens(net, 3, 4)[:, :1 if len(shape) == 1 else 4].reshape(shape), []
    for fill in (0, -10 ** 9, net.cfg.vocab):
        cache = _cache(net.cfg, 12)
        net.prefill(toks, cache, None, table)
        new = torch.where(torch.arange(new.numel() // 3) < counts[:, None], new.reshape(3, -1), fill).reshape(shape)
        got.append(net.extend(new, torch.full((3,), 32), cache, table, counts=counts).view(3, -1)[[0, 2], 0])
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])
