"""A paged cache of keys and values in 8 bits (csrc/kernels/kv8.cu): writing, attention, and giving pages back by their weight.

Codes are e4m3 with one scale per page and KV head, a power of two: the smallest, 2^-100 at least, that keeps the page's largest finite
magnitude within 448.  A page that tokens are added to keeps its scale or takes a larger one, which its earlier codes follow.  Values
that are not finite are stored as NaN.  Half the bytes of a 16-bit cache, which is what a decoding step's attention is bound by.

Tensors on the GPU go to the kernels (bf16 and fp16; heads of a multiple of 16 columns, at most 128); on the CPU the same is computed in plain
PyTorch, in any floating type.  The kernels have no gradient: where one would be recorded, they are refused.  They skip a page id outside the pool
or a position outside table and cache and note it in the word at ``status``, as the decoder's other passes do (models/llama.py); on the CPU it is
an IndexError.
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from .._ext import require_native

FP8 = torch.float8_e4m3fn
LEAST_SCALE = 2.0 ** -100


@dataclass
class Kv8Cache:
    """k, v: [layers, blocks, kv_heads, block_size, dim] e4m3; k_scale, v_scale: [layers, blocks, kv_heads] fp32."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor

    @staticmethod
    def empty(layers: int, blocks: int, kv_heads: int, block_size: int, dim: int, device="cuda") -> "Kv8Cache":
        def codes():
            return torch.empty(layers, blocks, kv_heads, block_size, dim, dtype=torch.uint8, device=device).view(FP8)

        def scales():
            return torch.ones(layers, blocks, kv_heads, device=device)

        return Kv8Cache(codes(), codes(), scales(), scales())

    @property
    def block_size(self) -> int:
        return self.k.shape[3]

    @property
    def nbytes(self) -> int:
        return sum(t.nbytes for t in (self.k, self.v, self.k_scale, self.v_scale))

    def tensors(self):
        return self.k, self.v, self.k_scale, self.v_scale


def _check_like(cache: Kv8Cache, t: torch.Tensor, what: str) -> None:
    if t.device != cache.k.device:
        raise RuntimeError(f"kv8: {what} on {cache.k.device} expected, not on {t.device}")


def write(cache: Kv8Cache, layer: int, qkv: torch.Tensor, block_table: torch.Tensor, start: torch.Tensor, *, counts: Optional[torch.Tensor] = None,
          positions: Optional[torch.Tensor] = None, rope: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
          out: Optional[torch.Tensor] = None, status: int = 0) -> torch.Tensor:
    """The pass between the product that makes queries, keys and values and the attention: bias and rotation of new tokens' rows, and their
    keys and values to their pages.

    qkv: [batch, tokens, heads + 2 kv_heads, dim]; token t of request b is the cache's slot ``start[b] + t`` ([batch] int64) of the pages
    ``block_table[b]`` ([batch, pages] int32).  What the last page written held behind that is no longer valid, and no page is written for two
    requests of a call.  counts ([batch] int64): tokens that a request has, of a padded batch; rows behind them stay as they are.  rope ([positions,
    dim] fp32): cosines, then sines; positions ([batch] int64): what the first token is rotated by, where that is not its slot.  bias: [(heads + 2 kv_heads) * dim].  Returns the rows as the
    attention takes them: ``out``, which may be qkv, or a new tensor."""
    if qkv.is_cuda:
        return require_native().kv8_write(cache.k, cache.v, cache.k_scale, cache.v_scale, block_table, layer, qkv, out, bias, rope, start, positions, counts, status)
    _check_like(cache, qkv, "rows")
    return _plain_write(cache, layer, qkv, torch.empty_like(qkv) if out is None else out, block_table, start, counts, positions, rope, bias)


def pack(cache: Kv8Cache, k_pool: torch.Tensor, v_pool: torch.Tensor, src_blocks: int, src_table: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor, *,
         status: int = 0) -> None:
    """The first ``lengths[b]`` tokens ([batch] int64) of every request, all layers, from 16-bit pages [layers, src_blocks, block_size, kv_heads, dim] (what
    the KV hand-off leaves on the decode side) at ``src_table`` to the cache's at ``block_table``."""
    if k_pool.is_cuda:
        require_native().kv8_pack(cache.k, cache.v, cache.k_scale, cache.v_scale, block_table, k_pool, v_pool, src_blocks, src_table, lengths, status)
        return
    _check_like(cache, k_pool, "pages")
    L, _, KH, bs, D = cache.k.shape
    k, v = (p.view(L, src_blocks, bs, KH, D) for p in (k_pool, v_pool))
    for b, n in enumerate(lengths.tolist()):
        pages = -(-max(n, 0) // bs)
        if pages > min(src_table.shape[1], block_table.shape[1]):
            raise IndexError(f"kv8: {n} tokens, {min(src_table.shape[1], block_table.shape[1])} pages of {bs}")
        for page in range(pages):
            here = min(n - page * bs, bs)
            to, at = _page(cache.k.shape[1], block_table[b, page]), _page(src_blocks, src_table[b, page])
            for codes, scales, src in ((cache.k, cache.k_scale, k), (cache.v, cache.v_scale, v)):
                for layer in range(L):
                    _store(codes, scales, layer, to, 0, src[layer, at, :here].transpose(0, 1))


def attention(cache: Kv8Cache, layer: int, q: torch.Tensor, block_table: torch.Tensor, start: torch.Tensor, *, counts: Optional[torch.Tensor] = None,
              scale: Optional[float] = None, mass: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None, status: int = 0) -> torch.Tensor:
    """Attention of new tokens over the cache, their own keys and values (already written) among it: q [batch, tokens, heads, dim], of any strides that
    are multiples of 8 elements; token t of request b sees slots 0 .. start[b] + t.  Returns [batch, tokens, heads * dim]; zeros for tokens behind
    ``counts`` and for those that see nothing.  scale (finite, not negative): 1 / sqrt(dim) by default.
    mass ([batch, pages] fp32) has the weights' sum over this call's tokens and heads added, page by page of ``block_table``; on the GPU such a call
    takes up to 6144 tokens times heads, and memory while it runs: 8 bytes per request, token, head and 16 slots of the table (at most 256 MiB, or one request's)."""
    if scale is None:
        scale = q.shape[-1] ** -0.5
    elif not 0 <= scale < math.inf:
        raise ValueError(f"kv8: scale {scale}")
    if q.is_cuda:
        return require_native().kv8_attention(cache.k, cache.v, cache.k_scale, cache.v_scale, block_table, layer, q, start, counts, scale, out, mass, status)
    _check_like(cache, q, "queries")
    B, T, H, D = q.shape
    return _plain_attention(cache, layer, q, block_table, start, counts, scale, mass, torch.empty(B, T, H * D, dtype=q.dtype) if out is None else out)


def evict(mass: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor, block_size: int, keep: int, *, recent: int = 1,
          sinks: int = 0) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """Requests that hold more than ``keep`` pages give back the lightest ones: of the ceil(lengths / block_size) pages of each, those of least ``mass`` ([batch,
    pages] fp32, see ``attention``; of equals the earlier one, NaN weighs most), but none of the first ``sinks`` and of the last ``recent``.
    Returns (block_table, lengths, mass, gone): the kept pages first, in their order, then the ``gone`` [batch] int32 ones, with a mass of 0,
    free for the request's next tokens or for others, then the rest of the row; lengths in tokens, block_size less for each page that went.
    Keys were rotated when they were written, so positions are no matter; the next token's slot is the new length."""
    if keep < recent + sinks or recent < 1 or sinks < 0 or block_size < 1:
        raise ValueError(f"kv8: keep ({keep}) at least recent ({recent}) + sinks ({sinks}) pages, recent at least one")
    if mass.is_cuda:
        return require_native().kv8_evict(mass, block_table, lengths, block_size, keep, recent, sinks)
    table, mass, lens, gone = block_table.clone(), mass.clone(), lengths.clone(), torch.zeros(len(lengths), dtype=torch.int32)
    for b, n in enumerate(lengths.tolist()):
        used = min(-(-max(n, 0) // block_size), mass.shape[1])
        extra = max(used - keep, 0)
        free = mass[b, sinks: max(used - recent, sinks)]
        out = set((torch.sort(free, stable=True)[1][:extra] + sinks).tolist())
        order = [i for i in range(used) if i not in out] + sorted(out)
        mass[b, list(out)] = 0.0
        table[b, :used], mass[b, :used] = table[b, order], mass[b, order]
        lens[b] -= extra * block_size
        gone[b] = extra
    return table, lens, mass, gone


# ---- plain forms ------------------------------------------------------------------------------------------------------------------
def scale_of(amax: torch.Tensor) -> torch.Tensor:
    """The scale for a largest finite magnitude."""
    m, e = torch.frexp(amax.float())                      # amax = m 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
    s = torch.ldexp(torch.ones_like(m), torch.where(m <= 0.875, e - 9, e - 8))
    return torch.where(amax > 0, s, torch.zeros_like(s)).clamp(min=LEAST_SCALE)


def dequantize(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """[..., block_size, dim] codes and their [...] scales -> fp32."""
    return codes.float() * scales[..., None, None]


def _page(blocks: int, page) -> int:
    i = int(page)
    i += blocks if i < 0 else 0
    if not 0 <= i < blocks:
        raise IndexError(f"kv8: page {int(page)} of a pool of {blocks}")
    return i


def _store(codes, scales, layer: int, page: int, lead: int, rows: torch.Tensor) -> None:
    """rows: [kv_heads, tokens, dim] to slots lead .. of a page whose slots before that are in use."""
    x = rows.float()
    x = torch.where(x.isfinite(), x, torch.full_like(x, math.nan))
    scale = scale_of(x.abs().nan_to_num(0.0).amax((1, 2)))
    if lead:
        was = scales[layer, page]
        scale = torch.maximum(scale, was)
        codes[layer, page, :, :lead] = (codes[layer, page, :, :lead].float() * (was / scale)[:, None, None]).to(FP8)
    codes[layer, page, :, lead: lead + x.shape[1]] = (x / scale[:, None, None]).to(FP8)
    scales[layer, page] = scale


def _tokens(counts, T: int, b: int) -> int:
    return T if counts is None else min(max(int(counts[b]), 0), T)


def _plain_write(cache, layer, qkv, out, block_table, start, counts, positions, rope, bias):
    B, T, A, D = qkv.shape
    KH, bs = cache.k.shape[2], cache.block_size
    if out is not qkv:
        out.copy_(qkv)
    for b in range(B):
        n, first = _tokens(counts, T, b), int(start[b])
        if n == 0:
            continue
        x = qkv[b, :n].float()
        if bias is not None:
            x = x + bias.float().view(A, D)
        if rope is not None:
            turn = first if positions is None else int(positions[b])
            if turn < 0 or turn + n > rope.shape[0]:
                raise IndexError(f"kv8: positions {turn} .. {turn + n - 1}, {rope.shape[0]} rotations")
            cos, sin = rope[turn: turn + n, None, : D // 2], rope[turn: turn + n, None, D // 2:]
            lo, hi = x[:, : A - KH, : D // 2], x[:, : A - KH, D // 2:]
            x = torch.cat([torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1), x[:, A - KH:]], 1)
        out[b, :n] = x.to(qkv.dtype)
        if first < 0 or first + n > block_table.shape[1] * bs:
            raise IndexError(f"kv8: slots {first} .. {first + n - 1} of {block_table.shape[1]} pages of {bs}")
        for page in range(first // bs, (first + n - 1) // bs + 1):
            lo, hi = max(page * bs, first), min((page + 1) * bs, first + n)
            at = _page(cache.k.shape[1], block_table[b, page])
            for codes, scales, head in ((cache.k, cache.k_scale, A - 2 * KH), (cache.v, cache.v_scale, A - KH)):
                _store(codes, scales, layer, at, lo - page * bs, out[b, lo - first: hi - first, head: head + KH].transpose(0, 1))
    return out


def _plain_attention(cache, layer, q, block_table, start, counts, scale, mass, out):
    B, T, H, D = q.shape
    KH, bs = cache.k.shape[2], cache.block_size
    out.zero_()
    for b in range(B):
        n, first = _tokens(counts, T, b), int(start[b])
        end = min(first + n, block_table.shape[1] * bs) if n else 0
        if end <= 0:
            continue
        pages = [_page(cache.k.shape[1], p) for p in block_table[b, : -(-end // bs)]]
        k, v = (dequantize(codes[layer, pages], scales[layer, pages]).transpose(0, 1).reshape(KH, -1, D)[:, :end].repeat_interleave(H // KH, 0)
                for codes, scales in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
        for t in range(n):
            seen = min(first + t + 1, end)
            if seen <= 0:
                continue
            p = (torch.einsum("hd,hnd->hn", q[b, t].float(), k[:, :seen]) * scale).softmax(-1)
            out[b, t] = torch.einsum("hn,hnd->hd", p, v[:, :seen]).reshape(-1).to(out.dtype)
            if mass is not None:
                mass[b].index_add_(0, torch.arange(seen) // bs, p.sum(0))
    return out
