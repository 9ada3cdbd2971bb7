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

:func:`lay_out_step` makes these on the device from the streams' lengths and hands out free pages.  Groups of streams that begin alike (many
answers to one prompt, several continuations of one video) may keep what they share outside their own tables, in a row of a
``prefix_table``: :func:`shared_prefix_attention` reads it once for a whole group.
"""
from __future__ import annotations

from typing import NamedTuple

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


class StepLayout(NamedTuple):
    """What :func:`lay_out_step` makes, on the device."""
    q_starts: torch.Tensor      # int32 [streams + 1]
    kv_lens: torch.Tensor       # int32 [streams], the new tokens included
    positions: torch.Tensor     # int64 [num_tokens]
    slots: torch.Tensor         # int64 [num_tokens]
    pages_wanted: torch.Tensor  # int32 [1]


def lay_out_step(new_lens: torch.Tensor, kv_lens: torch.Tensor, page_table: torch.Tensor, free_pages: torch.Tensor, page_size: int, num_tokens: int, *,
                 prefix_lens: torch.Tensor | None = None, group_starts: torch.Tensor | None = None, cursor: torch.Tensor | None = None,
                 kv_lens_out: torch.Tensor | None = None) -> StepLayout:
    """What the operators of a step read, from ``new_lens`` [streams], the streams' new tokens, and ``kv_lens`` [streams], the keys that they hold
    before them: int32 on the device, where nothing is waited for.  One launch, to be recorded into a graph or not.

    A stream's rows follow those of the stream before; its keys go on where they ended.  Pages that they need are taken from ``free_pages`` (int32 [n])
    in order of streams and keys and written into ``page_table``; where the list has come to its end, -1, a hole.  ``pages_wanted`` says how
    many were to be written: more than the list holds, and some tokens have no place.  With a ``cursor`` (int32 [1]) the list is taken from
    that entry on, and the cursor moves behind what was taken; with ``kv_lens_out``, which may be ``kv_lens``, the new lengths go there: steps
    that a graph replays go on from one another.

    ``positions`` count from the stream's first key, and with ``prefix_lens`` (int32 [groups]) from the beginning that its group shares:
    group g is streams ``group_starts[g] .. group_starts[g + 1] - 1`` (int32 [groups + 1]; all streams are one group without).  ``slots`` is -1 for
    tokens in holes and behind the table's width.  Tokens for which ``num_tokens`` has no row left are not laid out: their streams' lengths do not
    count them.  Rows behind the last stream's have position 0 and slot -1.

    ``page_table``, ``cursor`` and ``kv_lens_out`` are written and share no memory with one another or with what is read, but for ``kv_lens_out``
    in place of ``kv_lens``."""
    return StepLayout(*_native.step_layout(new_lens, kv_lens, page_table, free_pages, page_size, num_tokens, prefix_lens, group_starts, cursor, kv_lens_out))


def head_norm_rope_paged(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cache: dict, slots: torch.Tensor, q_weight: torch.Tensor | None,
                         k_weight: torch.Tensor | None, eps: float, cos_f32: torch.Tensor | None, sin_f32: torch.Tensor | None,
                         positions: torch.Tensor | None = None, interleaved: bool = True, out: torch.Tensor | None = None) -> torch.Tensor:
    """:func:`longlive_amd.utils.rope.head_norm_rope` of q and k whose K, with the V beside it, goes to the cache in the same launch:
    rows ``slots`` (int64 [T], :func:`paged_slots`) of ``k_pages`` / ``v_pages``; a slot outside the cache (-1) is written nowhere,
    and two tokens must not have one slot.  Returns the rotated q, in ``out`` if given, which may be q itself.

    Pages of any head_dim that the norm takes are written (multiples of 8 up to 256); :func:`paged_attention` reads 64 and 128."""
    return _native.head_norm_rope(q, k, v, q_weight, k_weight, eps, cos_f32, sin_f32, positions, interleaved, cache, slots, out)


def rotate_by_position_paged(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cache: dict, slots: torch.Tensor, positions: torch.Tensor | None,
                             frequencies: torch.Tensor, *, interleaved: bool = True, amplitude: float = 1.0, grid: tuple[int, int] | None = None,
                             sections: tuple[int, int, int] | None = None, q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None,
                             eps: float = 1e-6, out: torch.Tensor | None = None) -> torch.Tensor:
    """:func:`longlive_amd.utils.rope.rotate_by_position` of q and k whose K, with the V beside it, goes to the cache in the same launch, as in
    :func:`head_norm_rope_paged`.  Returns the rotated q, in ``out`` if given, which is q itself or memory that nothing else of the call uses."""
    return _native.rotate_by_position(q, k, v, q_weight, k_weight, eps, frequencies, amplitude, positions, interleaved, grid, sections, cache, slots, out)


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
    stay as they were in a given one, which is q itself or memory that nothing else of the call uses."""
    return _native.ragged_attention("paged_attention", q, q_starts, softmax_scale, max_q_len, max_kv_len, out, cache=cache, page_table=page_table,
                                    kv_lens=kv_lens, causal=causal, window=window, sink_tokens=sink_tokens)


def shared_prefix_attention(q: torch.Tensor, cache: dict, prefix_table: torch.Tensor, prefix_lens: torch.Tensor, page_table: torch.Tensor,
                            kv_lens: torch.Tensor, q_starts: torch.Tensor, group_starts: torch.Tensor | None = None, causal: bool = True,
                            softmax_scale: float | None = None, max_q_len: int | None = None, max_kv_len: int | None = None,
                            max_prefix_len: int | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """:func:`paged_attention` of streams in groups that share a beginning, which is read once for a group's rows where that is cheaper.

    Group g is streams ``group_starts[g] .. group_starts[g + 1] - 1`` (int32 [groups + 1], not decreasing; without it all streams are one group;
    streams outside every group share nothing).  The ``prefix_lens[g]`` keys (int32 [groups]) that it shares lie in the pages of ``prefix_table[g]``
    (int32 [groups, pages of the longest]), and every token of its streams sees all of them.  ``page_table`` and ``kv_lens`` are of the keys behind,
    each stream's own: token i of n sees own key j where ``j <= kv_lens[b] - n + i`` (``causal``; else every one).  A common beginning of whole
    pages at the front of every row of one table is handed on as views: ``table[:1, :w]`` and ``table[:, w:]``, with lengths that count from there.

    ``max_prefix_len``: the longest beginning, like ``max_q_len`` and ``max_kv_len`` (the longest stream's own keys).  There is no window: with one,
    streams go over one table whose rows begin with the shared pages, by :func:`paged_attention`.  The rest as there."""
    return _native.ragged_attention("shared_prefix_attention", q, q_starts, softmax_scale, max_q_len, max_kv_len, out, cache=cache, page_table=page_table,
                                    kv_lens=kv_lens, causal=causal, prefix=(prefix_table, prefix_lens, group_starts, max_prefix_len))
