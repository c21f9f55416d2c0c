"""Disaggregated serving: a prefill (context) stage and a decode stage on different GPUs, linked by the fused
KV hand-off kernel.

Reference behaviour (experiments/serving/main.cc:184-202, model.hh:253-337,420-529): ranks below world/2 run
the context stage, the rest decode; after the WHOLE prefill the context rank sends first tokens, the whole K
pool, the whole V pool, the block table and the block counts to rank + world/2 in one NCCL group, and the
decoder then generates tokens.  It prints elapsed time, KV send time and their ratio (main.cc:228-239).

Here the pairing (rank -> rank + world/2) and the reports are kept; the transfer is `kv_pack_send`: only the
pages in use move, they are re-laid-out for the decode pool on the fly, the small messages ride along as one
header, and each layer's pages leave as soon as that layer has been computed (a side stream ordered by events),
so the transfer overlaps the rest of the prefill.

``KVLink`` is the transfer object, ``PrefillStage`` / ``DecodeStage`` wrap the model, ``run_offline`` is the
two-stage experiment; all of them also work with both stages as virtual ranks on ONE GPU (emulated heap).
"""
from __future__ import annotations

import time
from dataclasses import dataclass, field
from typing import Optional

import torch

from .._ext import require_native
from ..models.llama import KV_BLHSD, KV_LBSHD, LlamaConfig, LlamaShard
from ..ops import kv8
from ..ops.sampling import Sampler
from ..parallel.symm import SymmetricHeap
from ..utils.timing import device_sync, timing_event

HDR_MAX_BATCH = 32
HDR_TOKENS, HDR_LENS, HDR_OUTS = 4, 4 + HDR_MAX_BATCH, 4 + 2 * HDR_MAX_BATCH
HDR_INTS = 4 + 3 * HDR_MAX_BATCH   # [batch, prompt_len, max_blocks, batch_index] + first tokens + prompt lengths + output lengths


def check_model(model) -> None:
    """Behind a synchronisation: raise what the model's kernels noted (models that note nothing have no ``check_status``)."""
    check = getattr(model, "check_status", None)
    if check is not None:
        check()


def choice(choose) -> dict:
    """How a model is told of a choice other than the greedy one."""
    return {} if choose is None else {"choose": choose}


def decoding_flags(ap) -> None:
    """Command line of ServeParams' decoding options."""
    ap.add_argument("--kv-bits", "--kv_bits", type=int, default=16, choices=[8, 16], help="bits of a cached key or value on the decode side")
    ap.add_argument("--keep-blocks", "--keep_blocks", type=int, default=0, help="pages that a request may keep, of a cache in 8 bits; the least attended ones go (0: all stay)")
    ap.add_argument("--temperature", type=float, default=0.0, help="0: greedy")
    ap.add_argument("--top-k", "--top_k", type=int, default=0)
    ap.add_argument("--top-p", "--top_p", type=float, default=1.0)
    ap.add_argument("--min-p", "--min_p", type=float, default=0.0)
    ap.add_argument("--seed", type=int, default=0)


def decoding_options(args) -> dict:
    """What the flags say, as keyword arguments of ServeParams."""
    return {k: getattr(args, k) for k in ("kv_bits", "keep_blocks", "temperature", "top_k", "top_p", "min_p", "seed")}


@dataclass
class ServeParams:
    """The experiment's knobs (TestParams of the reference, experiments/serving/model.hh:31-49)."""
    model: LlamaConfig
    batch_size: int = 16
    input_len: int = 2048
    num_decoding_step: int = 256
    tp_size: int = 1
    dtype: torch.dtype = torch.bfloat16     # --precision of the reference's binaries (fp16 / fp32 there); KV pools use it too
    # Decoding beyond the reference's: a cache in 8 bits (ops/kv8.py), at most so many pages per request (0: all of them; the lightest go, but not the
    # first and the last two), and tokens drawn by chance (ops/sampling.py; temperature 0: the greedy ones)
    kv_bits: int = 16
    keep_blocks: int = 0
    temperature: float = 0.0
    top_k: int = 0
    top_p: float = 1.0
    min_p: float = 0.0
    seed: int = 0

    EVICT_SINKS, EVICT_RECENT = 1, 2        # pages that are never given back
    PREFILL, DECODE = 0, 1                  # stages

    def check(self, device=None) -> None:
        """``device``: where the stage runs, if that is known; the kernels take less than the plain forms on the CPU."""
        if self.kv_bits not in (8, 16):
            raise ValueError(f"kv_bits {self.kv_bits}: 8 or 16")
        if self.keep_blocks and (self.kv_bits != 8 or self.keep_blocks < self.EVICT_SINKS + self.EVICT_RECENT):
            raise ValueError(f"keep_blocks {self.keep_blocks}: at least {self.EVICT_SINKS + self.EVICT_RECENT}, of a cache in 8 bits")
        if device is None or torch.device(device).type != "cuda":
            return
        small, drawn = self.kv_bits == 8, self.temperature > 0
        if (small or drawn) and self.dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"{'kv_bits 8' if small else f'temperature {self.temperature}'} with {self.dtype}: bf16 or fp16 on the GPU")
        if small and (self.model.head_dim % 16 or self.model.head_dim > 128):
            raise ValueError(f"kv_bits 8 with heads of {self.model.head_dim}: a multiple of 16, at most 128, on the GPU")
        most = require_native().SAMPLE_MAX_VOCAB
        if drawn and self.model.vocab > most:
            raise ValueError(f"temperature {self.temperature} with a vocabulary of {self.model.vocab}: at most {most} on the GPU")

    def sampler(self, batch: int, device) -> Optional[Sampler]:
        """What chooses the tokens of a batch; None: the greedy choice."""
        if not self.temperature > 0:
            return None
        return Sampler(torch.zeros(batch, device=device), self.temperature, self.top_k, self.top_p, self.min_p)

    def numbers(self, device, stage: int = PREFILL) -> torch.Generator:
        """The source of a stage's uniform numbers, the same one on every shard, another one in every stage: with one for both, a request's first and second
        token would be drawn by the same number."""
        return torch.Generator(device=device).manual_seed((self.seed + stage * 0x9E3779B97F4A7C15) % 2 ** 64)

    @property
    def elem_bytes(self) -> int:
        return torch.empty((), dtype=self.dtype).element_size()

    @property
    def kv_dim_units(self) -> int:
        """Head dimension as the KV kernel sees it: the kernel moves 2-byte elements, so a 4-byte type is a head twice
        as wide (the innermost run of a page is one head vector either way)."""
        return self.model.head_dim * self.elem_bytes // 2

    @property
    def block_size(self) -> int:
        return self.model.block_size

    @property
    def max_blocks_per_req(self) -> int:          # ceil((input + decode) / block), model.hh:100-103
        return (self.input_len + self.num_decoding_step + self.block_size - 1) // self.block_size

    @property
    def context_blocks_per_req(self) -> int:
        return (self.input_len + self.block_size - 1) // self.block_size


class KVLink:
    """Decode-side pools inside the symmetric heap + the flags and header of the hand-off.  Collective: both
    stages construct it with the same arguments so that offsets agree."""

    def __init__(self, heap: SymmetricHeap, p: ServeParams, kv_heads_local: int, name: str = "kv"):
        self.heap, self.p, self.kvh = heap, p, kv_heads_local
        m = p.model
        self.pool_blocks = p.batch_size * p.max_blocks_per_req
        self.page_elems = kv_heads_local * m.block_size * m.head_dim
        n = self.pool_blocks * m.layers * self.page_elems
        self.k_pool = heap.alloc_tensor([n], p.dtype)
        self.v_pool = heap.alloc_tensor([n], p.dtype)
        self.hdr = heap.alloc_tensor([HDR_INTS], torch.int64)
        self.layer_flags = heap.signal_slots(f"{name}:layers", m.layers)
        self.final_flag = heap.signal_slots(f"{name}:final", 1)
        self.seq = 0
        self.C = require_native()
        dev = self.k_pool.local.device
        self.cta_counter = torch.zeros(1, dtype=torch.int32, device=dev)

    # ---- prefill side -------------------------------------------------------------------------------------
    def send_layers(self, dst_rank: int, src_k, src_v, src_blocks: int, src_bt, dst_bt, nblocks, l0: int, l1: int,
                    hdr: Optional[torch.Tensor] = None, final: bool = False, num_ctas: int = 0):
        m = self.p.model
        flag = self.heap.sig_addr(self.final_flag if final else self.layer_flags + l0, dst_rank)
        self.C.kv_pack_send(src_k, src_v, self.k_pool.addr(dst_rank), self.v_pool.addr(dst_rank), KV_BLHSD, KV_LBSHD,
                            src_blocks, self.pool_blocks, m.layers, self.kvh, m.block_size, self.p.kv_dim_units, l0, l1, src_bt, dst_bt,
                            nblocks, hdr, self.hdr.addr(dst_rank) if hdr is not None else 0, flag, self.seq, self.cta_counter,
                            num_ctas, self.heap.status_addr)

    # ---- decode side --------------------------------------------------------------------------------------
    def wait_final(self, host_timeout_s: float = 300.0):
        """Wait for the header + all pages of hand-off number ``seq``.  The long part of the wait is a host poll (the
        prefill may take seconds); the device wait that follows only orders later kernels after the flag."""
        if not self.heap.host_wait(self.final_flag, self.seq, host_timeout_s):
            raise TimeoutError(f"KV hand-off {self.seq} did not arrive within {host_timeout_s} s")
        self.C.wait_flags([(self.heap.sig_addr(self.final_flag), self.seq)], self.heap.status_addr)

    def wait_layer(self, l: int):
        self.C.wait_flags([(self.heap.sig_addr(self.layer_flags + l), self.seq)], self.heap.status_addr)


class SmallCache:
    """A decode stage's cache in 8 bits: filled from the pages that the hand-off left, extended by every step, and cut to ``p.keep_blocks`` pages per
    request after every ``block_size`` steps."""

    def __init__(self, p: ServeParams, model: LlamaShard, link: KVLink):
        self.p, self.model, m = p, model, p.model
        dev, B = model.embed.device, p.batch_size
        self.cache = kv8.Kv8Cache.empty(m.layers, link.pool_blocks, model.kvh_local, m.block_size, m.head_dim, device=dev)
        # buffers that a captured step may hold
        self._table = torch.zeros(B, p.max_blocks_per_req, dtype=torch.int32, device=dev)
        self._slots = torch.zeros(B, dtype=torch.long, device=dev)
        self._seen, self._mass = (torch.zeros(B, p.max_blocks_per_req, device=dev) for _ in range(2))     # since the last eviction, and before
        self.begin_empty(B)

    def begin_empty(self, batch: int) -> None:
        self.table, self.slots, self.seen, self.mass = (t[:batch] for t in (self._table, self._slots, self._seen, self._mass))
        self.steps = 0

    def begin(self, link: KVLink, table: torch.Tensor, lengths: torch.Tensor) -> None:
        """A batch whose first ``lengths`` tokens are in ``link``'s pages ``table``."""
        self.begin_empty(table.shape[0])
        self.table.copy_(table)
        self.slots.copy_(lengths)
        self.seen.zero_()
        self.mass.zero_()
        status = self.model._status_or_0()
        kv8.pack(self.cache, link.k_pool.local, link.v_pool.local, link.pool_blocks, table, self.table, self.slots, status=status)

    def step(self, tokens: torch.Tensor, pos: torch.Tensor, choose=None) -> torch.Tensor:
        return self.model.extend(tokens, pos, self.cache, self.table, slots=self.slots, mass=self.seen if self.p.keep_blocks else None, choose=choose,
                                 max_positions=self.p.input_len + self.p.num_decoding_step + self.p.block_size)

    def advance(self) -> None:
        """The step's tokens are in the cache (part of a captured step)."""
        self.slots.add_(1)

    def after_step(self) -> None:
        self.steps += 1
        if self.p.keep_blocks and self.steps % self.p.block_size == 0:
            self.mass += self.model._allreduce(self.seen)                   # every shard's heads
            self.seen.zero_()
            table, slots, mass, _ = kv8.evict(self.mass, self.table, self.slots, self.p.block_size, self.p.keep_blocks,
                                              recent=self.p.EVICT_RECENT, sinks=self.p.EVICT_SINKS)
            for t, new in ((self.table, table), (self.slots, slots), (self.mass, mass)):
                t.copy_(new)


@dataclass
class StageReport:
    role: str
    elapsed_ms: float = 0.0
    compute_ms: float = 0.0
    kv_ms: float = 0.0              # device time of the KV hand-off kernels (prefill) / of the wait (decode)
    kv_bytes: int = 0
    tokens: int = 0
    extra: dict = field(default_factory=dict)


class PrefillStage:
    def __init__(self, p: ServeParams, model: LlamaShard, link: KVLink, dst_rank: int, pipeline_layers: bool = True):
        self.p, self.model, self.link, self.dst = p, model, link, dst_rank
        self.pipeline = pipeline_layers
        m = p.model
        dev = model.embed.device
        self.ctx_blocks = p.batch_size * p.context_blocks_per_req
        n = self.ctx_blocks * m.layers * link.page_elems
        self.k_pool = torch.empty(n, dtype=p.dtype, device=dev)
        self.v_pool = torch.empty(n, dtype=p.dtype, device=dev)
        B, cb, mb = p.batch_size, p.context_blocks_per_req, p.max_blocks_per_req
        # source pages: request-major; destination pages: the decode pool reserves max_blocks_per_req per request
        self.src_bt = torch.arange(B * cb, dtype=torch.int32, device=dev).view(B, cb).contiguous()
        self.dst_bt = (torch.arange(B, dtype=torch.int32, device=dev).unsqueeze(1) * mb +
                       torch.arange(cb, dtype=torch.int32, device=dev).unsqueeze(0)).contiguous()
        self.nblocks = torch.full((B,), cb, dtype=torch.int32, device=dev)
        # the KV hand-off runs on a side stream beside the prefill; on host tensors (tests that model the kernels) in line
        self.side = torch.cuda.Stream(device=dev) if dev.type == "cuda" else None
        self.dev = dev
        self.hdr = torch.zeros(HDR_INTS, dtype=torch.int64, device=dev)
        p.check(dev)
        self.choose, self.numbers = p.sampler(B, dev), p.numbers(dev, p.PREFILL)

    def first_tokens(self, tokens: torch.Tensor, on_layer_done=None) -> torch.Tensor:
        """The prompts through the model, into the stage's own pools."""
        if self.choose is not None:
            self.choose.u.copy_(torch.rand(len(self.choose.u), generator=self.numbers, device=self.dev))
        return self.model.prefill(tokens, self.k_pool, self.v_pool, self.src_bt, on_layer_done, **choice(self.choose))

    def run(self, tokens: torch.Tensor) -> StageReport:
        p, link = self.p, self.link
        link.seq += 1
        cuda = self.side is not None
        main = torch.cuda.current_stream() if cuda else None
        e0, e1, k0, k1 = (timing_event(self.dev) for _ in range(4))
        first_kv = [True]

        def after_main():
            """The side stream continues from what the main stream has enqueued so far."""
            if cuda:
                ev = torch.cuda.Event()
                ev.record(main)
                self.side.wait_event(ev)

        def on_layer(l: int):
            if not self.pipeline:
                return
            with torch.cuda.stream(self.side):
                after_main()
                if first_kv[0]:
                    k0.record(self.side)
                    first_kv[0] = False
                link.send_layers(self.dst, self.k_pool, self.v_pool, self.ctx_blocks, self.src_bt, self.dst_bt, self.nblocks, l, l + 1)

        e0.record(main)
        first = self.first_tokens(tokens, on_layer)
        e1.record(main)
        self.hdr[0], self.hdr[1], self.hdr[2] = p.batch_size, p.input_len, p.max_blocks_per_req
        self.hdr[4:4 + p.batch_size] = first
        with torch.cuda.stream(self.side):
            after_main()
            if not self.pipeline:
                k0.record(self.side)
                link.send_layers(self.dst, self.k_pool, self.v_pool, self.ctx_blocks, self.src_bt, self.dst_bt, self.nblocks, 0,
                                 p.model.layers)
            # header + final flag: a zero-layer-cost launch that only copies the control block
            link.send_layers(self.dst, self.k_pool, self.v_pool, self.ctx_blocks, self.src_bt, self.dst_bt,
                             torch.zeros_like(self.nblocks), 0, 1, hdr=self.hdr, final=True, num_ctas=1)
            k1.record(self.side)
        if cuda:
            main.wait_stream(self.side)
        device_sync(self.dev)
        check_model(self.model)
        kv_bytes = 2 * self.ctx_blocks * p.model.layers * link.page_elems * p.elem_bytes
        return StageReport("prefill", elapsed_ms=e0.elapsed_time(k1), compute_ms=e0.elapsed_time(e1), kv_ms=k0.elapsed_time(k1),
                           kv_bytes=kv_bytes, tokens=p.batch_size * p.input_len)


class DecodeStage:
    """Decoding over the paged pool, or over a cache in 8 bits made from it (``p.kv_bits``); greedy, or by chance (``p.temperature``).  The
    per-token step is launch-bound (hundreds of small kernels), so it is captured once in a CUDA graph and replayed;
    ``use_graph=False`` keeps the eager loop."""

    def __init__(self, p: ServeParams, model: LlamaShard, link: KVLink, use_graph: bool = True):
        self.p, self.model, self.link = p, model, link
        dev = model.embed.device
        B, mb = p.batch_size, p.max_blocks_per_req
        self.bt = (torch.arange(B, dtype=torch.int32, device=dev).unsqueeze(1) * mb +
                   torch.arange(mb, dtype=torch.int32, device=dev).unsqueeze(0)).contiguous()
        self.dev = dev
        self.use_graph = use_graph and dev.type == "cuda"
        self.graph = None
        self.g_tokens = torch.zeros(B, dtype=torch.long, device=dev)
        self.g_pos = torch.zeros(B, dtype=torch.long, device=dev)
        # The captured step feeds itself: it takes g_tokens at g_pos, notes the result in row g_step of g_hist, puts it into
        # g_tokens and advances g_pos and g_step, so decoding is nothing but replays.  Nothing of `p` is in the graph, whose
        # lengths a caller may change; longer runs than the history has rows for are read out in between.
        self.g_hist = torch.zeros(max(1, p.num_decoding_step), B, dtype=torch.long, device=dev)
        self.g_step = torch.zeros(1, dtype=torch.long, device=dev)
        p.check(dev)
        self.small = SmallCache(p, model, link) if p.kv_bits == 8 else None
        self.choose, self.numbers = p.sampler(B, dev), p.numbers(dev, p.DECODE)
        self.g_u = None if self.choose is None else torch.zeros_like(self.g_hist, dtype=torch.float32)      # what every step draws by

    def _step(self, tokens, pos):
        link = self.link
        if self.small is not None:
            return self.small.step(tokens, pos, self.choose)
        return self.model.decode_step(tokens, pos, link.k_pool.local, link.v_pool.local, self.bt, link.pool_blocks, **choice(self.choose))

    def _draw(self, n: int) -> None:
        if self.choose is not None:
            self.g_u[:n].copy_(torch.rand(n, self.p.batch_size, generator=self.numbers, device=self.dev))

    def _capture(self):
        """Capture one decode step on static buffers.  The step writes K/V at g_pos, so the capture (which runs the
        step for real during warm-up) is done at a scratch position that the first real step overwrites anyway."""
        try:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                for _ in range(2):
                    self._step(self.g_tokens, self.g_pos)
            torch.cuda.current_stream().wait_stream(side)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                if self.choose is not None:
                    self.choose.u.copy_(self.g_u.index_select(0, self.g_step)[0])
                out = self._step(self.g_tokens, self.g_pos)
                self.link.C.dec_advance(out, self.g_tokens, self.g_pos, self.g_hist, self.g_step)
                if self.small is not None:
                    self.small.advance()
            self.graph = g
        except Exception as e:  # noqa: BLE001 - capture is an optimisation; the eager loop is always valid
            self.graph = None
            self.use_graph = False
            print(f"[fuselink] decode graph capture failed ({type(e).__name__}: {e}); running eagerly")

    def decode(self, tokens: torch.Tensor):
        """Generate num_decoding_step tokens after `tokens` ([B] first tokens).  Returns (generated [B, 1+steps],
        device ms of the loop)."""
        p = self.p
        d0, d1 = timing_event(self.dev), timing_event(self.dev)
        out = [tokens]
        pos = torch.full((p.batch_size,), p.input_len, dtype=torch.long, device=tokens.device)
        if self.use_graph and self.graph is None:
            self.g_tokens.copy_(tokens)
            self.g_pos.copy_(pos)
            if self.small is not None:
                self.small.begin(self.link, self.bt, pos)
            self._capture()                     # one-off set-up, outside the timed loop
        d0.record()
        if self.small is not None:
            self.small.begin(self.link, self.bt, pos)
        if self.graph is not None:
            self.g_tokens.copy_(tokens)
            self.g_pos.copy_(pos)
            rows = self.g_hist.shape[0]
            for first in range(0, p.num_decoding_step, rows):
                n = min(rows, p.num_decoding_step - first)
                self.g_step.zero_()
                self._draw(n)
                for _ in range(n):
                    self.graph.replay()
                    if self.small is not None:
                        self.small.after_step()
                out.append(self.g_hist[:n].clone() if first + n < p.num_decoding_step else self.g_hist[:n])
            gen = torch.cat([tokens.unsqueeze(1), *(h.t() for h in out[1:])], 1)
        else:
            rows = self.g_hist.shape[0]
            for i in range(p.num_decoding_step):
                if i % rows == 0:
                    self._draw(min(rows, p.num_decoding_step - i))
                if self.choose is not None:
                    self.choose.u.copy_(self.g_u[i % rows])
                tokens = self._step(tokens, pos)
                if self.small is not None:
                    self.small.advance()
                    self.small.after_step()
                out.append(tokens)
                pos = pos + 1
            gen = torch.stack(out, 1)
        d1.record()
        device_sync(self.dev)
        check_model(self.model)
        return gen, d0.elapsed_time(d1)

    def run(self) -> StageReport:
        p, link = self.p, self.link
        link.seq += 1
        w0, w1 = timing_event(self.dev), timing_event(self.dev)
        w0.record()
        link.wait_final()                       # header + every layer's pages have landed
        w1.record()
        tokens = link.hdr.local[4:4 + p.batch_size].clone()
        device_sync(self.dev)
        t_first = time.monotonic()              # first token is on the decode side: time-to-first-token ends here
        gen, ms = self.decode(tokens)
        rep = StageReport("decode", elapsed_ms=w0.elapsed_time(w1) + ms, compute_ms=ms, kv_ms=w0.elapsed_time(w1),
                          tokens=p.batch_size * p.num_decoding_step)
        rep.extra["t_first_token"] = t_first
        rep.extra["generated"] = gen
        rep.extra["graph"] = self.graph is not None
        return rep


def make_prompts(p: ServeParams, device, seed: int = 0) -> torch.Tensor:
    g = torch.Generator(device=device).manual_seed(seed)
    return torch.randint(0, p.model.vocab, (p.batch_size, p.input_len), generator=g, device=device)
