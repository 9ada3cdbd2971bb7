"""Plain 64-bit forms of the operators for several streams in one batch, and the error their kernels may have."""
import math

import torch

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}   # half a step, relative


def head_norm_rope(x, weight, eps, cos, sin, positions, interleaved):
    """(result, allowed error) of x [T, H, D]."""
    u = UNIT[x.dtype]
    y = x.double()
    if weight is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    size = y.abs()
    if cos is not None:
        R = 2 * cos.shape[1]
        at = torch.arange(x.shape[0]) if positions is None else positions.cpu()
        inside = (at >= 0) & (at < cos.shape[0])
        c, s = (t.cpu().double()[at.clamp(0, cos.shape[0] - 1)] for t in (cos, sin))
        c, s = torch.where(inside[:, None], c, 1.0)[:, None], torch.where(inside[:, None], s, 0.0)[:, None]
        first = torch.arange(R // 2) * (2 if interleaved else 1)
        second = first + (1 if interleaved else R // 2)
        a, b = y[..., first].clone(), y[..., second].clone()
        y[..., first], y[..., second] = a * c - b * s, b * c + a * s
        size = size.clone()
        size[..., first], size[..., second] = a.abs() + b.abs(), a.abs() + b.abs()
    # fp32: the sum of D squares (D / 2 relative steps to its root), the root, three products and a sum per value; then one rounding,
    # whose step is a float16 subnormal's below 2^-14
    steps = x.shape[-1] / 2 + 8
    return y, u * y.abs() + steps * 2.0 ** -24 * size * 2 + (2.0 ** -25 if x.dtype == torch.float16 else 0.0)


def attend(q, k, v, seen, scale):
    """(result, allowed error) of one stream and kv head: q [n, D], k, v [m, D], seen [n, m]."""
    u, n, m, D = UNIT[q.dtype], q.shape[0], k.shape[0], q.shape[-1]
    used = seen.any(0)
    q, k, v = q.double(), k.double(), v.double()
    k, v = (torch.where(used[:, None], t, 0.0) for t in (k, v))   # whatever lies where nobody looks
    s = (q @ k.T * scale).masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True) if m else torch.full((n, 1), -math.inf, dtype=torch.float64)
    w = torch.where(seen, (s - torch.where(top == -math.inf, 0.0, top)).exp(), 0.0)
    total = w.sum(-1, keepdim=True)
    total = torch.where(total == 0, 1.0, total)
    out, size = w @ v / total, w @ v.abs() / total
    # fp32 scores: D products added up, one multiplication by scale * log2 e, the reference point subtracted; exp2 within two steps.
    # The matrix unit's sums are taken to truncate: 2^-23 a step.
    reach = (q.abs() @ k.abs().T * scale).masked_fill(~seen, 0.0)
    reach = reach.amax(-1, keepdim=True) if m else torch.zeros(n, 1, dtype=torch.float64)
    score = ((D + 4) * 2.0 ** -23) * reach + 2.0 ** -22 * 4
    sums = (m + 64) * 2.0 ** -23          # numerator and denominator, each in any order
    error = u * out.abs() + size * (u + 2 * score + 2 * sums)
    if u == UNIT[torch.float16]:          # subnormal probabilities and results
        error = error + 2.0 ** -25 * (m * v.abs().amax(0, keepdim=True) if m else 0.0) + 2.0 ** -25
    return out, error


def ragged_attention(q, q_starts, scale, keys_of, seen_of):
    """(result, allowed error, rows of some stream) of q [T, H, D]; keys_of(b) -> (k, v) [m, Hk, D], seen_of(b, n, m) -> [n, m]; on the CPU."""
    out = torch.zeros(q.shape, dtype=torch.float64)
    error, rows = torch.zeros_like(out), torch.zeros(q.shape[0], dtype=torch.bool)
    starts = q_starts.tolist()
    for b in range(len(starts) - 1):
        at, n = starts[b], starts[b + 1] - starts[b]
        rows[at:at + n] = True
        k, v = keys_of(b)
        seen = seen_of(b, n, k.shape[0])
        group = q.shape[1] // k.shape[1]
        for h in range(q.shape[1]):
            out[at:at + n, h], error[at:at + n, h] = attend(q[at:at + n, h], k[:, h // group], v[:, h // group], seen, scale)
    return out, error, rows


def paged_keys(cache, page_table, kv_lens):
    """keys_of and holes_of for :func:`ragged_attention`; rows in holes are zeros that nobody sees."""
    k_pages, v_pages = (cache[n].cpu() for n in ("k_pages", "v_pages"))
    table, lens, P = page_table.cpu().long(), kv_lens.tolist(), k_pages.shape[1]

    def rows(b):
        j = torch.arange(max(0, min(lens[b], table.shape[1] * P)))
        entry = table[b, j // P]
        return entry, j % P, (entry >= 0) & (entry < k_pages.shape[0])

    def keys_of(b):
        entry, row, ok = rows(b)
        at = torch.where(ok, entry, 0)
        if k_pages.shape[0] == 0:
            zero = torch.zeros(len(row), *k_pages.shape[2:], dtype=k_pages.dtype)
            return zero, zero
        return tuple(torch.where(ok[:, None, None], t[at, row], 0.0) for t in (k_pages, v_pages))

    def seen_of(causal=True, window=None, sink=0):
        def seen(b, n, m):
            j, p = torch.arange(m), (m - n + torch.arange(n))[:, None]
            s = rows(b)[2].expand(n, m).clone()
            if causal:
                s &= j <= p
            if window:
                s &= (j > p - window) | (j < sink)
            return s
        return seen
    return keys_of, seen_of
