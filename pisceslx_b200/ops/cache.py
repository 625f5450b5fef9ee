"""Operators of the paged cache in 8 bits, and attention of new tokens over pages (serving: no autograd).

A cache in 8 bits holds keys and values as e4m3 codes ``[blocks, block, hk, d]`` with one exponent byte for each token and head
``[blocks, hk, block]``: a number is ``code * 2 ** (byte - 127)``, and the exponent is the smallest at which the largest number of
the row (one head of one token) does not pass 448.  A row with a number that is not finite has the byte 255 and is read as NaN
throughout.  It takes d + 1 bytes a row where bf16 takes 2 d, and a code is within 2^-4 of its number (of numbers below 2^-14 of the
row's largest: within 2^-17 of that one).

CUDA tensors run the kernels of ``csrc/cache.cu``; CPU tensors run the plain math of ``ops.reference``."""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import kernels, reference as ref, status_word


def kv_cache_write_fp8(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                       v_scale: torch.Tensor, slot_map: torch.Tensor) -> None:
    """Append rows k/v [T, hk*d] (they may be column ranges of a projection) to the pages of codes and exponent bytes at flat slots
    ``slot_map`` (int32, -1 = skip; a slot has one row at most: of two, parts of both may stay)."""
    if k.is_cuda:
        kernels().kv_cache_write_fp8(k, v, k_cache, v_cache, k_scale, v_scale, slot_map, status_word(k.device))
        return
    ref.kv_cache_write_fp8(k, v, k_cache, v_cache, k_scale, v_scale, slot_map)


def kv_cache_read_fp8(k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                      slot_map: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Cached keys and values at flat slots ``slot_map`` (int32) as bf16 rows [n, hk*d], exactly what the codes stand for; -1 gives a
    row of zeros."""
    if k_cache.is_cuda:
        return kernels().kv_cache_read_fp8(k_cache, v_cache, k_scale, v_scale, slot_map, status_word(k_cache.device))
    return ref.kv_cache_read_fp8(k_cache, v_cache, k_scale, v_scale, slot_map)


def cache_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
                    cu_q: Optional[torch.Tensor] = None, max_q: Optional[int] = None, scale: Optional[float] = None, window: Optional[int] = None,
                    first_tokens: int = 0, k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None,
                    out: Optional[torch.Tensor] = None, splits: int = 0) -> torch.Tensor:
    """Causal attention of the new tokens of every sequence over its pages, which hold them already: q [T, hq, d] -> [T, hq, d].

    ``block_table`` [B, pages] and ``seq_lens`` [B] (cached tokens, the new ones among them) say where a sequence's tokens lie;
    ``cu_q`` [B + 1] where its new tokens lie in ``q`` (None: one token per sequence, a decode step), at most ``max_q`` each (None: as
    many as ``q`` has; few tokens run as such where it says so).  A sequence with more is refused, on the GPU through the status word
    and with its rows not written.  The last new token sits at ``seq_lens - 1``.  With ``window`` a token sees itself, the
    ``window - 1`` tokens in front of it and the ``first_tokens`` first of the sequence; table entries of pages that none of the new
    tokens sees are not read.  A token that sees nothing (``seq_lens`` smaller than the new tokens) gets zeros, and so does one whose
    every score is below -1e29.

    Pages [blocks, block, hk, d] are bf16, or e4m3 codes with ``k_scale`` and ``v_scale`` as ``kv_cache_write_fp8`` leaves them; a page
    holds a multiple of 16 tokens, heads 64 or 128 numbers, and up to 128 query heads share a key head.  What a page holds
    behind a sequence's end does not matter.  A value that is NaN or infinite may reach all of its sequence's new tokens, those that
    it is hidden from among them; a key only those that see it.  8-bit values of one sequence may differ by up to 2^100 in size:
    beside larger ones, smaller ones may count as zero for few tokens.  Over 8-bit pages a few tokens' queries are held to 2^-22 of the
    largest of their row's numbers (those above 2^-14 of it exactly).

    More than 64 rows (token, query head of a key head) of 8-bit pages take scratch of 4 hk d bytes for each token that the table has
    room for, or that the new tokens can see with ``window``: about a gigabyte of sequences at a time, one at least.

    Rows of ``q`` that belong to no sequence: those of ``out`` are left as they are; without ``out`` they are zero.  ``splits``: ranges
    that the keys of a block of queries are cut in (0: a rule on the sizes); calls with few tokens cut them in a way of their own."""
    d = q.shape[-1]
    scale = d ** -0.5 if scale is None else scale
    if window is not None and window <= 0:
        raise ValueError(f"window {window}: at least the token itself is seen")
    if max_q is None:
        max_q = 1 if cu_q is None else q.shape[0]
    if q.is_cuda:
        return kernels().cache_attention(q, k_cache, v_cache, block_table, seq_lens, cu_q, max_q, scale, window or 0, first_tokens,
                                         k_scale, v_scale, out, splits, status_word(q.device))
    if cu_q is not None and cu_q.numel() > 1 and int(cu_q.diff().max()) > max_q:
        raise ValueError(f"a sequence of {int(cu_q.diff().max())} new tokens: at most {max_q} were announced")
    return ref.cache_attention(q, k_cache, v_cache, block_table, seq_lens, cu_q, scale, window, first_tokens, k_scale, v_scale, out)
