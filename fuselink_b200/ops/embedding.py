"""Embedding lookup with a factor, and the table's gradient (csrc/kernels/embedding.cu).

The gradient of a row is the sum over the places of its token, in their order and in fp32, rounded once: the same batch gives the same bits.
A negative token counts from the vocabulary's end.  A token outside the vocabulary gives a row of zeros on the GPU, gets no gradient, and is noted in
the word at ``status`` (1), as the decoder's passes do (models/llama.py); on the CPU it is an IndexError.
"""
from __future__ import annotations

import torch

from .._ext import require_native
from .checks import ordinary


def lookup(table: torch.Tensor, tokens: torch.Tensor, scale: float = 1.0, *, status: int = 0) -> torch.Tensor:
    """``table[tokens] * scale``, rounded once to the table's type: [*tokens.shape, hidden].  table [vocab, hidden], bf16, fp16 or fp32 on the GPU, with
    contiguous rows; tokens int64 or int32 of any shape."""
    if table.dim() != 2 or table.shape[0] == 0 or table.shape[1] == 0:
        raise ValueError(f"embedding: table [vocab, hidden] expected, not {tuple(table.shape)}")
    if table.is_cuda and ordinary(table) and ordinary(tokens):
        return require_native().embed_lookup(table, tokens, scale, status)
    return _plain_lookup(table, tokens, scale)


def _plain_lookup(table, tokens, scale):
    if tokens.dtype not in (torch.int64, torch.int32):
        raise RuntimeError("embedding: tokens of int64 or int32 expected")
    if tokens.device != table.device:
        raise RuntimeError(f"embedding: tokens on {table.device} expected, not on {tokens.device}")
    wide = torch.float64 if table.dtype == torch.float64 else torch.float32
    return (table.to(wide)[tokens.long()] * scale).to(table.dtype)
