"""Paged KV cache: several streams (requests) in one cache of bf16 or f16 pages, and the two operators around it.

The NVFP4 cache of :mod:`longlive_amd.utils.kv_cache` holds one stream and is written by whole blocks, each of which has one
tensor scale.  Here a stream's keys lie in pages of ``page_size`` rows anywhere in the cache, listed in its row of a page
table, so that streams of any length share the memory and grow by single tokens; pages may be shared between streams (a common
beginning) and taken out (an entry of -1 is a hole).  Which page belongs to whom is the caller's business.

What a step of a batch looks like on the device, all int32 (one launch recorded into a graph follows what they hold at its replay):

* ``q_starts`` [streams + 1]: the new tokens of stream b are rows ``q_starts[b] .. q_starts[b + 1] - 1`` of q, k and v;
* ``kv_lens`` [streams]: keys of each stream, its new tokens included;
* ``page_table`` [streams, pages of the longest stream]: key j of stream b is row ``j % page_size`` of page
  ``page_table[b, j // page_size]``.
"""
from __future__ import annotations

import torch

from .. import _native


def initialize_paged_kv_cache(num_layers: int, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int, device,
                              dtype=torch.bfloat16) -> list[dict]:
    """One dict per layer: ``k_pages`` / ``v_pages`` [num_pages, page_size, num_kv_heads, head_dim], not initialized (no operator
    looks at rows that hold no key)."""
    if dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"a paged KV cache holds bfloat16 or float16, not {dtype}")
    if num_pages < 0 or min(page_size, num_kv_heads) < 1 or head_dim not in (64, 128):
        raise ValueError(f"no cache of {num_pages} pages of {page_size} rows of {num_kv_heads} heads of {head_dim}: head_dim is 64 or 128")
    shape = (num_pages, page_size, num_kv_heads, head_dim)
    return [{name: torch.empty(shape, dtype=dtype, device=device) for name in ("k_pages", "v_pages")} for _ in range(num_layers)]


def paged_slots(page_table: torch.Tensor, kv_lens: torch.Tensor, q_starts: torch.Tensor, num_tokens: int, page_size: int) -> torch.Tensor:
    """Where the new tokens' K and V go: int64 [num_tokens], ``page * page_size + row`` of a token's place in its stream, -1 for rows
    outside every stream, for places before a stream's beginning or behind its table, and for places in holes.  Once per step,
    for all layers; nothing waits for the device."""
    if page_table.ndim != 2 or kv_lens.shape != page_table.shape[:1] or q_starts.shape != (kv_lens.shape[0] + 1,):
        raise ValueError(f"page_table {tuple(page_table.shape)}, kv_lens {tuple(kv_lens.shape)} and q_starts {tuple(q_starts.shape)} are not of one batch")
    if page_size < 1 or num_tokens < 0:
        raise ValueError(f"{num_tokens} tokens, pages of {page_size} rows")
    if 0 in page_table.shape or num_tokens == 0:
        return torch.full((num_tokens,), -1, dtype=torch.int64, device=page_table.device)
    starts = q_starts.long()
    token = torch.arange(num_tokens, device=page_table.device)
    stream = torch.searchsorted(starts, token, right=True) - 1     # the last stream that begins at or before the token
    inside = (stream >= 0) & (stream < kv_lens.shape[0])
    stream = stream.clamp(0, kv_lens.shape[0] - 1)
    place = kv_lens.long()[stream] - starts[stream + 1] + token
    inside &= (place >= 0) & (place < page_table.shape[1] * page_size)
    place = place.clamp(0, page_table.shape[1] * page_size - 1)
    page = page_table.long()[stream, place // page_size]
    return torch.where(inside & (page >= 0), page * page_size + place % page_size, -1)


def head_norm_rope_paged(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cache: dict, slots: torch.Tensor, q_weight: torch.Tensor | None,
                         k_weight: torch.Tensor | None, eps: float, cos_f32: torch.Tensor | None, sin_f32: torch.Tensor | None,
                         positions: torch.Tensor | None = None, interleaved: bool = True, out: torch.Tensor | None = None) -> torch.Tensor:
    """:func:`longlive_amd.utils.rope.head_norm_rope` of q and k whose K, with the V beside it, goes to the cache in the same launch:
    rows ``slots`` (int64 [T], :func:`paged_slots`) of ``k_pages`` / ``v_pages``; a slot outside the cache (-1) is written nowhere,
    and two tokens must not have one slot.  Returns the rotated q, in ``out`` if given, which may be q itself.

    Pages of any head_dim that the norm takes are written (multiples of 8 up to 256); :func:`paged_attention` reads 64 and 128."""
    return _native.head_norm_rope(q, k, v, q_weight, k_weight, eps, cos_f32, sin_f32, positions, interleaved, cache, slots, out)


def paged_attention(q: torch.Tensor, cache: dict, page_table: torch.Tensor, kv_lens: torch.Tensor, q_starts: torch.Tensor, causal: bool = True,
                    window: int | None = None, sink_tokens: int = 0, softmax_scale: float | None = None, max_q_len: int | None = None,
                    max_kv_len: int | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of every stream's new tokens over its keys in the cache, the tokens' own (already written) among them.

    q [T, H, D], D 64 or 128, H a multiple of the cache's heads; head h reads kv head ``h // (H // kv heads)``.  Token i of a stream's n
    sits at position ``p = kv_lens[b] - n + i`` and sees key j where ``j <= p`` (``causal``; else every key: a chunk whose tokens see
    one another) and, with a ``window``, ``j > p - window or j < sink_tokens``.  Keys in holes of the page table and behind its
    width do not exist, but count for the positions.  A token that sees no key gets zeros.  Scores, softmax statistics and sums are fp32; the probabilities enter the
    second product in q's type.  Scores times the scale lie within 2^27 (float16) or 2^30 (bfloat16) of zero.

    ``max_q_len`` / ``max_kv_len``: the longest stream's new tokens and keys, if the caller knows them; any value gives the right result,
    true ones a division of the work that fits.  Returns ``out`` [T, H, D]: rows outside every stream are zeros in a new tensor and
    stay as they were in a given one, which may be q itself."""
    return _native.ragged_attention("paged_attention", q, q_starts, softmax_scale, max_q_len, max_kv_len, out, cache=cache, page_table=page_table,
                                    kv_lens=kv_lens, causal=causal, window=window, sink_tokens=sink_tokens)
