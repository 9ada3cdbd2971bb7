"""Cross attention of a batch of requests, each to encoder states of its own number.

The reference's cross attention (wan_5b/modules/causal_model.py:197-262) and ``_native.attention_bf16`` attend one dense context; here every
request has its own, with padding and masked states left out.
"""
from __future__ import annotations

import torch

from .. import _native


def ragged_cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_starts: torch.Tensor, k_starts: torch.Tensor,
                           k_lens: torch.Tensor | None = None, key_mask: torch.Tensor | None = None, softmax_scale: float | None = None,
                           max_q_len: int | None = None, max_k_len: int | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """``softmax(q k^T * scale) v`` of request b's queries, rows ``q_starts[b] .. q_starts[b + 1] - 1`` of q [T, H, D], over its states:
    rows ``k_starts[b] .. k_starts[b + 1] - 1`` of k and v [n, Hk, D], or ``k_lens[b]`` rows from ``k_starts[b]`` on (a padded batch), except
    those whose entry of ``key_mask`` (bool [n]) is False.  A request without states gets zeros.

    bfloat16 or float16, D 64 or 128, H a multiple of Hk; starts and lengths int32 on the device.  Sums, ``max_q_len`` / ``max_k_len``,
    ``out`` and rows outside every request: as in :func:`longlive_amd.utils.paged_kv.paged_attention`."""
    return _native.ragged_attention("ragged_cross_attention", q, q_starts, softmax_scale, max_q_len, max_k_len, out, k=k, v=v, k_starts=k_starts,
                                    k_lens=k_lens, key_mask=key_mask)
