"""Plain forms of the operators around a step of several streams: the layout as a loop, the rotation and the attention over a shared beginning in
64 bits with the error that their kernels may have."""
import torch

import streams_reference as ref


def step_layout(new_lens, kv_lens, table, free, page_size, num_tokens, prefix_lens=None, group_starts=None, cursor=0):
    """(q_starts, kv_lens, positions, slots, pages wanted, table, cursor) as lists."""
    table, taken, wanted = [list(r) for r in table], max(cursor, 0), 0
    q_starts, lens, positions, slots = [0], [], [], []
    for b, (n, m) in enumerate(zip(new_lens, kv_lens)):
        m = max(m, 0)
        n = min(max(n, 0), num_tokens - len(positions), 2 ** 31 - 1 - m)
        ahead = 0
        if prefix_lens is not None:
            starts = [0, len(kv_lens)] if group_starts is None else group_starts
            for g, p in enumerate(prefix_lens):
                if starts[g] <= b < starts[g + 1]:
                    ahead = max(p, 0)
        width = len(table[b])
        for key in range(m, m + n):
            entry = key // page_size
            page = -1
            if entry < width:
                if key % page_size == 0:
                    at = taken + wanted
                    table[b][entry] = free[at] if at < len(free) else -1
                    wanted += 1
                page = table[b][entry]
            positions.append(ahead + key)
            slots.append(page * page_size + key % page_size if page >= 0 else -1)
        q_starts.append(len(positions))
        lens.append(m + n)
    positions += [0] * (num_tokens - len(positions))
    slots += [-1] * (num_tokens - len(slots))
    return q_starts, lens, positions, slots, wanted, table, min(taken + wanted, max(len(free), taken))


def rotate(x, weight, eps, frequencies, positions, interleaved, amplitude=1.0, grid=None, sections=None):
    """(result, allowed error) of x [T, H, D]."""
    u, amplitude = ref.UNIT[x.dtype], torch.tensor(amplitude, dtype=torch.float32).double()
    y = x.double()
    steps = 0.0
    if weight is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
        steps = x.shape[-1] / 2 + 8          # of the norm, see streams_reference
    R = 2 * len(frequencies)
    p = (torch.arange(x.shape[0]) if positions is None else positions)[:, None].expand(-1, R // 2)
    if grid:
        pair = torch.arange(R // 2)
        p = torch.where(pair < sections[0], p.div(grid[0] * grid[1], rounding_mode="floor"),
                        torch.where(pair < sections[0] + sections[1], p.remainder(grid[0] * grid[1]).div(grid[1], rounding_mode="floor"), p.remainder(grid[1])))
    angle = p.double() * frequencies
    c, s = (angle.cos() * amplitude)[:, None], (angle.sin() * amplitude)[:, None]
    first = torch.arange(R // 2) * (2 if interleaved else 1)
    second = first + (1 if interleaved else R // 2)
    a, b = y[..., first].clone(), y[..., second].clone()
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    size = y.abs()
    size[..., first] = size[..., second] = (a.abs() + b.abs()) * amplitude.abs()
    # the part of a turn, at most a half, is rounded to 32 bits: 2^-26 turns, 2^-23.3 radians; the hardware's sine and cosine are within 2^-22.9
    # (measured on 2^22 points); together 2^-22.  The angle itself: three products in 64 bits, up to 3 * 2^-53 of it.  Then two products, one with
    # the amplitude, and a sum in 32 bits
    turn = angle.abs().amax(-1)[:, None, None] * (3 * 2.0 ** -53) if len(frequencies) else 0.0
    error = u * y.abs() + size * (2.0 ** -22 + (4 + 2 * steps) * 2.0 ** -24 + turn)
    return y, error + (2.0 ** -25 if x.dtype == torch.float16 else 0.0)


def shared_prefix(q, cache, prefix_table, prefix_lens, table, kv_lens, q_starts, group_starts, causal, scale):
    """(result, allowed error, rows of some stream) of q [T, H, D], all on the CPU."""
    shared, _ = ref.paged_keys(cache, prefix_table, prefix_lens)
    own, _ = ref.paged_keys(cache, table, kv_lens)
    streams = len(kv_lens)
    starts = [0, streams] if group_starts is None else group_starts.tolist()

    def holes(of_table, length, P, n_pages):
        j = torch.arange(max(0, min(length, of_table.numel() * P)))
        entry = of_table.long()[j // P] if len(j) else j
        return (entry >= 0) & (entry < n_pages)

    def group(b):
        return next((g for g in range(len(starts) - 1) if starts[g] <= b < starts[g + 1]), None)

    P, n_pages = cache["k_pages"].shape[1], cache["k_pages"].shape[0]

    def keys_of(b):
        g = group(b)
        return own(b) if g is None else tuple(torch.cat(t) for t in zip(shared(g), own(b)))

    def seen_of(b, n, m):
        g = group(b)
        there = holes(table[b], int(kv_lens[b]), P, n_pages)
        ahead = there[:0] if g is None else holes(prefix_table[g], int(prefix_lens[g]), P, n_pages)
        seen = there.expand(n, -1).clone()
        if causal:
            seen &= torch.arange(len(there)) <= (int(kv_lens[b]) - n + torch.arange(n))[:, None]
        return torch.cat([ahead.expand(n, -1), seen], dim=1)
    return ref.ragged_attention(q, q_starts, scale, keys_of, seen_of)
