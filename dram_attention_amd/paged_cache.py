"""Keys and values of a batch of sequences in pages of HBM: storing a step's or a prompt's, and attention of one new
token of every sequence.

Beside ``DRAMAttention``, which keeps one long sequence's pages in host memory: the sequences here are many, ragged and
wholly in HBM, and share one pool of pages through a table of page numbers, with their lengths on the device, so that a
step can be captured in a graph and replayed as they grow.  Dense attention of one token, which the reference does on a
contiguous cache (dram_attention/dram_attention.py:144-238).
"""

from __future__ import annotations

import torch

from . import _lib
from .rotary import layout_code


def kv_pages(n_pages: int, page_size: int, n_kv_heads: int, head_dim: int, *, dtype: torch.dtype = torch.bfloat16,
             device="cuda") -> tuple[torch.Tensor, torch.Tensor]:
    """An empty pool: (k_pages, v_pages), each (n_pages, page_size, n_kv_heads, head_dim), views of one tensor that
    holds what a kv head has in a page in one piece, keys and values of a token side by side (the layout of the page
    cache's slots).  dtype bf16, fp16 or fp32, or float8_e4m3fn under 16-bit queries.  Heads of any size can be stored;
    :func:`paged_decode_attention` takes 64, 96, 128 and 256 channels."""
    if dtype not in (torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn):
        raise TypeError(f"unsupported element type {dtype}")
    if n_pages < 0 or page_size < 1 or n_kv_heads < 1 or head_dim < 1:
        raise ValueError(f"no pool of {n_pages} pages of {page_size} tokens of {n_kv_heads} heads of {head_dim}")
    pool = torch.empty(n_pages, n_kv_heads, page_size, 2, head_dim, dtype=dtype, device=device)
    return pool[:, :, :, 0].transpose(1, 2), pool[:, :, :, 1].transpose(1, 2)


def append_kv_pages_(xk: torch.Tensor, xv: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                     page_table: torch.Tensor, positions: torch.Tensor, *, sequences: torch.Tensor | None = None,
                     xq: torch.Tensor | None = None, freqs: torch.Tensor | None = None, layout: str = "interleaved",
                     factor: float = 1.0, k_scale: torch.Tensor | None = None,
                     v_scale: torch.Tensor | None = None) -> torch.Tensor | None:
    """Store keys, turned by their positions on the way, and values in their sequences' pages; returns the turned
    queries (None without ``xq``).

    xk, xv (tokens, kv heads, head_dim); k_pages, v_pages (pages, page_size, kv heads, head_dim) of the same strides
    that share no memory; page_table (sequences, pages) and positions (tokens,) int32 or int64.  Token t is of row
    sequences[t] of the table, or of row t without ``sequences`` (a decode step), and goes to slot p % page_size of page
    page_table[row, p // page_size], p = positions[t].  Tokens of a call have places of their own, which no operand of
    the call is a view of.  Not stored: a token whose position is negative (padding) or beyond its row of the table,
    whose sequence is none of the table's, or whose page number is none of the pool's; its query is turned all the same.
    xq (tokens, heads, head_dim), ``freqs`` (None: nothing turns), ``layout``, ``factor``: as of :func:`rotate`.
    k_scale, v_scale (kv heads,) float32 above 0: 8-bit pages hold a key or value divided by its head's, clamped to 448
    and rounded to nearest; without them 1.
    """
    return _lib.host().paged_append(xk, xv, k_pages, v_pages, page_table, positions, sequences, xq, freqs,
                                    layout_code(layout), float(factor), k_scale, v_scale)


def paged_decode_attention(xq: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                           lengths: torch.Tensor, *, scale: float | None = None, k_scale: torch.Tensor | None = None,
                           v_scale: torch.Tensor | None = None, out: torch.Tensor | None = None,
                           lse: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(q . k * scale) v of one query token of every sequence over the first lengths[b] tokens in its pages.

    xq (sequences, heads, head_dim), heads a multiple of the kv heads; pages and page_table as of
    :func:`append_kv_pages_`, head_dim 64, 96, 128 or 256; lengths (sequences,) int32 or int64, on the device: they
    include the token itself where its key was stored before.  ``scale``: head_dim ** -0.5 by default.  Returns a tensor
    like xq (``out`` if given, which may be a contiguous xq itself); fills ``lse`` (sequences, heads) fp32, the natural
    logarithm of the softmax denominator.  Neither shares memory with another operand.
    A sequence of no tokens gets zeros (lse -inf), and tokens on pages that are none of the pool's do not count; a query
    whose scores are all -inf gets the definition's NaN (lse -inf).
    16-bit and 8-bit keys and values are multiplied exactly and summed in fp32, by weights of 24 bits (bf16) or ones that
    are kept to 2^-20 of themselves or 2^-40 of the sequence's largest, whichever is more (fp16: an infinite value under a
    weight below 2^-29 of the largest may give NaN); fp32 ones are multiplied in fp32.  The same shapes and lengths give the
    same bits.
    """
    return _lib.host().paged_attention(xq, k_pages, v_pages, page_table, lengths, scale, k_scale, v_scale, out, lse)
