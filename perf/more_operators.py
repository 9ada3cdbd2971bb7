"""Operators around a step of several streams that share a beginning, as cases with sizes: what a performance measurement runs.

Three operators that follow one another in a step of a batch over a paged cache:

* ``layout``  the step's lengths turned into what the kernels read: where each stream's rows begin, where its tokens sit, pages
              for new keys out of a list of free ones, the page table with them, and the row of the cache for every token;
* ``rotary``  q and k rotated by angles formed from positions of any size and a few frequencies (stretched for contexts longer than
              a model was trained on; positions on a line, or of a video's frame, row and column), K and V on to the cache's rows;
* ``prefix``  attention of the streams' new tokens over a beginning that a group of them shares, read once for all, and over each
              stream's own keys behind it.

The sizes run from a step of a few single tokens, where a call's own latency counts, to prompts of many streams and to several
continuations, 2640 tokens each, of one video of twelve frames of 880 tokens by 24 heads, the chunks of this package's benchmark.
"""
import math
import random

import torch

own = False
DEVICE = "cuda"
TYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16}
VIDEO = (22, 40)  # tokens of a video frame: rows and columns


def listed():
    return [
        # a decoding step of a few streams: one row each, now and then a new page
        dict(name="layout_step", kind="layout", streams=24, new=1, new_most=1, kv=100, kv_most=8000, page=16, groups=0, idle=0.0, spare=40, spread=1),
        # a step of a thousand streams in groups that share a beginning, a part of them waiting
        dict(name="layout_many", kind="layout", streams=1000, new=1, new_most=4, kv=20, kv_most=4000, page=24, groups=40, idle=0.2, spare=7, spread=2),
        # prompts of a hundred requests of up to 4096 tokens
        dict(name="layout_prompts", kind="layout", streams=100, new=50, new_most=4096, kv=1, kv_most=600, page=16, groups=3, idle=0.0, spare=100, spread=3),
        # a decoding step: q and k as the projections leave them, frequencies divided for a context four times as long
        dict(name="rotary_step", kind="rotary", tokens=24, heads=16, kv_heads=4, dim=128, rotary=128, pairs="halves", axes="line", scaling="positions", factor=4.0,
             longest=32768, page=16, type="bfloat16"),
        # a video chunk, 3 frames of 22 x 40 tokens: frame, row and column each turn their part of the pairs
        dict(name="rotary_video", kind="rotary", tokens=2640, heads=24, kv_heads=24, dim=128, rotary=128, pairs="interleaved", axes="video", scaling="none", factor=1.0,
             longest=200 * 880, page=0, type="bfloat16"),
        # prompts of many streams at far positions, narrow heads of which half is rotated, an odd number of tokens and an odd page
        dict(name="rotary_far_odd", kind="rotary", tokens=16381, heads=40, kv_heads=8, dim=64, rotary=32, pairs="halves", axes="line", scaling="parts", factor=16.0,
             longest=1 << 20, page=24, type="float16"),
        # one long prompt
        dict(name="rotary_long", kind="rotary", tokens=40000, heads=32, kv_heads=8, dim=128, rotary=128, pairs="halves", axes="line", scaling="base", factor=8.0,
             longest=40000, page=64, type="bfloat16"),
        # four answers to one short prompt, a few tokens in
        dict(name="prefix_step_small", kind="prefix", streams=4, groups=1, new=1, new_most=1, kv=1, kv_most=40, prefix=500, prefix_most=500, heads=16, kv_heads=4,
             dim=64, page=16, causal=True, type="float16", spread=4),
        # a decoding step of 64 answers to one long prompt
        dict(name="prefix_step_long", kind="prefix", streams=64, groups=1, new=1, new_most=1, kv=30, kv_most=1000, prefix=16384, prefix_most=16384, heads=32, kv_heads=8,
             dim=128, page=16, causal=True, type="bfloat16", spread=5),
        # drafts, single tokens and pieces of prompts of four groups, odd lengths and pages
        dict(name="prefix_mixed", kind="prefix", streams=41, groups=4, new=1, new_most=200, kv=10, kv_most=900, prefix=300, prefix_most=5000, heads=20, kv_heads=4,
             dim=128, page=24, causal=True, type="float16", spread=6),
        # many short answers over one system prompt, a head of its own for every query
        dict(name="prefix_drafts", kind="prefix", streams=100, groups=1, new=4, new_most=4, kv=8, kv_most=300, prefix=3001, prefix_most=3001, heads=12, kv_heads=12,
             dim=64, page=32, causal=True, type="bfloat16", spread=7),
        # four continuations of a video of twelve frames, 2640 tokens each, every token sees its chunk and all that came before
        dict(name="prefix_video", kind="prefix", streams=4, groups=1, new=2640, new_most=2640, kv=2640, kv_most=2640, prefix=10560, prefix_most=10560, heads=24,
             kv_heads=24, dim=128, page=880, causal=False, type="bfloat16", spread=8),
    ]


# ------------------------------------------------------------------------------------------------- drawn cases
def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    kv = rng.choice([1, 2, 3, 4, 8, 12, 16, 24])
    return kv * rng.choice([g for g in (1, 1, 2, 4, 5, 7, 8) if g * kv <= 48]), kv


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng):
    most = 0.8 * max(_cost(c) for c in listed())
    while True:
        case = _draw(rng)
        # the plain form of the attention holds every product of a group's rows and of a padded batch
        held = 0
        if case["kind"] == "prefix":
            held = case["heads"] * (sum(_queries(case)) * case["prefix_most"] + case["streams"] * case["new_most"] * case["kv_most"])
        if _cost(case) <= most and held <= 1.5e9:
            return case


def _draw(rng):
    kind = rng.choice(["layout", "rotary", "prefix", "prefix"])
    spread = rng.randrange(1 << 16)
    if kind == "layout":
        streams, most = _log(rng, 1, 2000), 1 if rng.random() < 0.4 else _log(rng, 2, 4096)
        if streams * most > 400000:
            most = max(400000 // streams, 1)
        kv_most = _log(rng, 1, 16384)
        return dict(kind=kind, streams=streams, new=max(1, int(most * rng.random())), new_most=most, kv=max(1, int(kv_most * rng.random())), kv_most=kv_most,
                    page=rng.choice([1, 8, 16, 24, 64, 880]), groups=rng.choice([0, 1, min(streams, rng.randrange(1, 60))]), idle=rng.choice([0.0, 0.0, 0.3]),
                    spare=rng.choice([0, 5, 100, -3]), spread=spread)
    heads, kv_heads = _heads(rng)
    dim, typ = rng.choice([64, 128, 128]), rng.choice(["bfloat16", "bfloat16", "float16"])
    if kind == "rotary":
        case = dict(kind=kind, tokens=_log(rng, 1, 40000), heads=heads, kv_heads=kv_heads, dim=dim, rotary=rng.choice([dim, dim, dim // 2, 16]),
                    pairs=rng.choice(["halves", "interleaved"]), axes="line", scaling=rng.choice(["none", "positions", "base", "parts"]),
                    factor=rng.choice([1.5, 4.0, 16.0]), longest=_log(rng, 100, 1 << 22), page=rng.choice([0, 1, 16, 24, 64]), type=typ)
        return dict(case, axes="video", rotary=dim, scaling="none") if rng.random() < 0.3 else case
    groups = rng.choice([1, 1, 2, 5])
    new_most = 1 if rng.random() < 0.4 else _log(rng, 2, 2700)
    kv_most, prefix_most = new_most + _log(rng, 1, 2000), _log(rng, 16, 20000)
    return dict(kind=kind, streams=max(groups, _log(rng, 1, 128)), groups=groups, new=max(1, int(new_most * rng.random())), new_most=new_most,
                kv=max(1, int(kv_most * rng.random())), kv_most=kv_most, prefix=max(1, int(prefix_most * rng.random())), prefix_most=prefix_most, heads=heads,
                kv_heads=kv_heads, dim=dim, page=rng.choice([1, 8, 16, 24, 32, 64, 880]), causal=rng.random() < 0.8, type=typ, spread=spread)


# ------------------------------------------------------------------------------------------------- sizes of a case
def _lengths(case, count, lo, hi, salt):
    """`count` lengths between lo and hi, the longest and, where there are two, the shortest among them."""
    rng = random.Random(case["spread"] * 7 + salt)
    got = [_log(rng, lo, hi) for _ in range(count)]
    at = rng.randrange(count)
    got[at] = hi
    if count > 1:
        got[at - 1] = lo
    return got


def _queries(case):
    got = _lengths(case, case["streams"], case["new"], case["new_most"], 1)
    if case["kind"] == "layout" and case["idle"]:
        rng = random.Random(case["spread"] * 7 + 4)
        got = [0 if rng.random() < case["idle"] else n for n in got]
    return got


def _before(case):  # keys that a stream holds ahead of the step
    return _lengths(case, case["streams"], case["kv"], case["kv_most"], 2)


def _own_keys(case):
    return [max(n, m) for n, m in zip(_queries(case), _before(case))]


def _groups(case):
    """(where the groups begin among the streams, the length of each one's shared beginning)."""
    rng = random.Random(case["spread"] * 7 + 5)
    cuts = sorted(rng.sample(range(1, case["streams"]), case["groups"] - 1)) if case["groups"] > 1 else []
    if case["kind"] == "layout":
        return [0] + cuts + [case["streams"]], _lengths(case, case["groups"], 100, 20000, 3)
    return [0] + cuts + [case["streams"]], _lengths(case, case["groups"], case["prefix"], case["prefix_most"], 3)


def _wanted(case):  # pages that a layout's new keys need
    P = case["page"]
    return sum(-(-(m + n) // P) - -(-m // P) for n, m in zip(_queries(case), _before(case)))


def work(case):
    if case["kind"] == "layout":
        S, T = case["streams"], sum(_queries(case))
        return {"bytes": 4 * (2 * S + (S + 1) + S) + 16 * T + 8 * _wanted(case) + 4 * S + 8 * case["groups"], "flops": 4 * T + 8 * S}
    D, Hq, Hk = case["dim"], case["heads"], case["kv_heads"]
    if case["kind"] == "rotary":
        T, moved = case["tokens"], Hq + (2 if case["page"] else 1) * Hk
        return {"bytes": T * (2 * moved * D * 2 + (16 if case["page"] else 8)) + 4 * case["rotary"], "flops": T * (Hq + Hk) * 3 * case["rotary"]}
    starts, shared = _groups(case)
    new, keys = _queries(case), _own_keys(case)
    pairs = 0
    for g, P in enumerate(shared):
        for n, m in zip(new[starts[g]:starts[g + 1]], keys[starts[g]:starts[g + 1]]):
            pairs += n * P + (n * (m - n) + n * (n + 1) // 2 if case["causal"] else n * m)
    return {"bytes": 2 * 2 * sum(new) * Hq * D + 2 * 2 * (sum(shared) + sum(keys)) * Hk * D, "flops": 4 * D * Hq * pairs}


# ------------------------------------------------------------------------------------------------- inputs
def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEVICE)


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _starts(lengths):
    return torch.tensor([0] + lengths, dtype=torch.int32).cumsum(0, dtype=torch.int32).to(DEVICE)


def _table(held, order, width, rest):
    """Page tables of streams that hold so many pages, out of `order` one behind the other, `rest` in the other entries."""
    at = torch.tensor([0] + held[:-1], device=DEVICE).cumsum(0)[:, None] + torch.arange(width, device=DEVICE)
    inside = torch.arange(width, device=DEVICE) < torch.tensor(held, device=DEVICE)[:, None]
    return torch.where(inside, order[at.clamp(max=len(order) - 1)], rest).contiguous()


def _frequencies(case):
    """Radians per position of every pair, and by how much cosines and sines are multiplied."""
    R, factor, base = case["rotary"], case["factor"], 10000.0
    if case["axes"] == "video":  # of a head's pairs, a third for rows, a third for columns, the rest for frames
        third = R // 2 // 3
        parts = [base ** (-torch.arange(n, dtype=torch.float64) / n) for n in (R // 2 - 2 * third, third, third)]
        return torch.cat(parts).to(DEVICE), 1.0, (len(parts[0]), third, third)
    if case["scaling"] == "base":  # the slowest pair turns `factor` times slower, the fastest as before
        base *= factor ** (R / max(R - 2, 1))
    f = base ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)
    if case["scaling"] == "positions":
        f = f / factor
    if case["scaling"] == "parts":  # pairs that turn 32 times or more over the trained length stay, those below one turn are divided
        turns = f * 4096 / (2 * math.pi)
        keep = ((turns - 1.0) / 31.0).clamp(0.0, 1.0)
        f = f * (keep + (1.0 - keep) / factor)
        return f.to(DEVICE), 0.1 * math.log(factor) + 1.0, None
    return f.to(DEVICE), 1.0, None


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(int(seed))
    if case["kind"] == "layout":
        return _prepare_layout(case, gen)
    typ, D, Hq, Hk = TYPES[case["type"]], case["dim"], case["heads"], case["kv_heads"]
    if case["kind"] == "rotary":
        T = case["tokens"]
        rows = _randn(gen, T, (Hq + 2 * Hk) * D).to(typ)  # what a projection of q, k and v leaves: one row a token
        q, k, v = (x.unflatten(1, (-1, D)) for x in rows.split([Hq * D, Hk * D, Hk * D], dim=1))
        f, amplitude, sections = _frequencies(case)
        state = dict(case=case, q=q, k=k, v=v, frequencies=f, amplitude=amplitude, sections=sections,
                     positions=torch.randint(0, case["longest"], (T,), generator=gen, device=DEVICE))
        if case["page"]:
            pages = -(-T // case["page"]) + 3
            state["cache"] = {name: _randn(gen, pages, case["page"], Hk, D).to(typ) for name in ("k_pages", "v_pages")}
            state["slots"] = torch.randperm(pages * case["page"], generator=gen, device=DEVICE)[:T]
        return state
    new, keys = _queries(case), _own_keys(case)
    first, shared = _groups(case)
    T, page = sum(new), case["page"]
    # behind a norm of every head: some channels larger than others, products of q and k of about two
    channels = 0.5 + _randn(gen, D).abs()
    state = dict(case=case, q=(2 * _randn(gen, T, Hq, D) * channels).to(typ), q_starts=_starts(new), kv_lens=_int32(keys), group_starts=_int32(first),
                 prefix_lens=_int32(shared), new=new, keys=keys, first=first, shared=shared)
    held, held_shared = [-(-n // page) for n in keys], [-(-n // page) for n in shared]
    pages = sum(held) + sum(held_shared) + 2
    order = torch.randperm(pages, generator=gen, device=DEVICE).int()
    state["page_table"] = _table(held, order, max(held) + 1, 0)
    state["prefix_table"] = _table(held_shared, order[sum(held):], max(held_shared), 0)
    state["cache"] = {"k_pages": (_randn(gen, pages, page, Hk, D) / channels).to(typ), "v_pages": _randn(gen, pages, page, Hk, D).to(typ)}
    return state


def _prepare_layout(case, gen):
    # lengths of another seed are the case's, dealt to the streams in another order
    deal = torch.randperm(case["streams"], generator=gen, device=DEVICE).tolist()
    new, before, P = [_queries(case)[i] for i in deal], [_before(case)[i] for i in deal], case["page"]
    held = [-(-m // P) for m in before]
    wanted, width = _wanted(case), max(-(-(n + m) // P) for n, m in zip(new, before)) + 1
    free = max(wanted + case["spare"], 0)  # a spare below zero: fewer than the step needs
    order = torch.randperm(sum(held) + free, generator=gen, device=DEVICE).int()
    state = dict(case=case, new_lens=_int32(new), kv_lens=_int32(before), page_table=_table(held, order, width, -1), free_pages=order[sum(held):].contiguous(),
                 tokens=sum(new) + case["streams"] % 3)  # sometimes with rows behind the last
    if case["groups"]:
        first, shared = _groups(case)
        state.update(group_starts=_int32(first), prefix_lens=_int32(shared))
    return state


# ------------------------------------------------------------------------------------------------- one pass
def run(state):
    kind = state["case"]["kind"]
    if own:
        return _run_own(state)
    return {"layout": _plain_layout, "rotary": _plain_rotary, "prefix": _plain_prefix}[kind](state)


def _run_own(s):
    c = s["case"]
    if c["kind"] == "layout":
        from longlive_amd.utils.paged_kv import lay_out_step
        got = lay_out_step(s["new_lens"], s["kv_lens"], s["page_table"], s["free_pages"], c["page"], s["tokens"], prefix_lens=s.get("prefix_lens"),
                           group_starts=s.get("group_starts"))
        return got.q_starts, got.kv_lens, got.positions, got.slots, s["page_table"], got.pages_wanted
    if c["kind"] == "rotary":
        options = dict(interleaved=c["pairs"] == "interleaved", amplitude=s["amplitude"], sections=s["sections"], grid=VIDEO if s["sections"] else None)
        if "cache" in s:
            from longlive_amd.utils.paged_kv import rotate_by_position_paged
            q = rotate_by_position_paged(s["q"], s["k"], s["v"], s["cache"], s["slots"], s["positions"], s["frequencies"], **options)
            return q, s["cache"]["k_pages"], s["cache"]["v_pages"]
        from longlive_amd.utils.rope import rotate_by_position
        return rotate_by_position(s["q"], s["k"], s["positions"], s["frequencies"], **options)
    from longlive_amd.utils.paged_kv import shared_prefix_attention
    return shared_prefix_attention(s["q"], s["cache"], s["prefix_table"], s["prefix_lens"], s["page_table"], s["kv_lens"], s["q_starts"],
                                   group_starts=s["group_starts"], causal=c["causal"], max_q_len=max(s["new"]), max_kv_len=max(s["keys"]),
                                   max_prefix_len=max(s["shared"]))


def _plain_layout(s):
    P, T, table, dev = s["case"]["page"], s["tokens"], s["page_table"], s["page_table"].device
    S, width = table.shape
    before, ends = s["kv_lens"].long(), s["new_lens"].long().cumsum(0)
    starts = torch.cat([ends.new_zeros(1), ends])
    after = before + s["new_lens"]
    have, need = (before + P - 1) // P, (after + P - 1) // P  # pages ahead of the step and behind it
    upto = (need - have).cumsum(0)
    first = upto - (need - have)                              # of a stream's pages in the list of free ones
    spare = torch.cat([s["free_pages"].long(), torch.full((1,), -1, device=dev)])  # behind the list: none
    entry = torch.arange(width, device=dev)
    at = (first[:, None] + entry - have[:, None]).clamp(0, len(spare) - 1)
    table.copy_(torch.where((entry >= have[:, None]) & (entry < need[:, None]), spare[at].int(), table))
    token = torch.arange(T, device=dev)
    b = torch.searchsorted(starts, token, right=True) - 1
    inside = b < S
    b = b.clamp(max=S - 1)
    key = torch.where(inside, before[b] + token - starts[b], 0)
    page = table[b, key // P].long()
    slots = torch.where(inside & (page >= 0), page * P + key % P, -1)
    if "group_starts" in s:
        group = torch.searchsorted(s["group_starts"].long(), torch.arange(S, device=dev), right=True) - 1
        key = key + torch.where(inside, s["prefix_lens"].long()[group][b], 0)
    return starts.int(), after.int(), key, slots, table, upto[-1:].int()


def _plain_rotary(s):
    c, f, p = s["case"], s["frequencies"], s["positions"]
    if s["sections"]:
        rows, cols = VIDEO
        axes = (p // (rows * cols), p // cols % rows, p % cols)
        angle = torch.cat([a.double()[:, None] * part for a, part in zip(axes, f.split(s["sections"]))], dim=1)
    else:
        angle = p.double()[:, None] * f  # far positions lose their angle in 32 bits
    cos, sin = ((t * s["amplitude"]).float()[:, None] for t in (angle.cos(), angle.sin()))
    q, k = (_plain_rotate(s[n].float(), cos, sin, c["rotary"], c["pairs"] == "halves").to(s[n].dtype) for n in ("q", "k"))
    if "cache" not in s:
        return q, k
    for pages, new in ((s["cache"]["k_pages"], k), (s["cache"]["v_pages"], s["v"])):
        pages.view(-1, *pages.shape[2:])[s["slots"]] = new
    return q, s["cache"]["k_pages"], s["cache"]["v_pages"]


def _plain_rotate(x, cos, sin, R, halves):
    if halves:
        a, b = x[..., :R // 2], x[..., R // 2:R]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., R:]], dim=-1)
    a, b = x[..., 0:R:2], x[..., 1:R:2]
    return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2), x[..., R:]], dim=-1)


def _rows_of_keys(s, table, upto):
    """K and V in 32 bits of `upto` keys of every row of a page table: [rows, kv heads, upto, D]."""
    page = s["case"]["page"]
    key = torch.arange(upto, device=table.device)
    entry = table.long()[:, key // page]
    return tuple(s["cache"][n][entry, key % page].float().transpose(1, 2) for n in ("k_pages", "v_pages"))


def _plain_prefix(s):
    c = s["case"]
    typ, dev, T, B, most, Hk = s["q"].dtype, s["q"].device, s["q"].shape[0], c["streams"], max(s["new"]), c["kv_heads"]
    G, keys, scale = c["heads"] // Hk, max(s["keys"]), c["dim"] ** -0.5
    q = s["q"].float().unflatten(1, (Hk, G))  # [T, kv heads, group, D]
    first, n_new, n_keys = s["q_starts"][:-1].long(), s["q_starts"].diff().long(), s["kv_lens"].long()
    # each stream's own keys, as a padded batch
    at = first[:, None] + torch.arange(most, device=dev)
    mine = q[at.clamp(max=T - 1)].permute(0, 2, 3, 1, 4).flatten(2, 3)  # [B, kv heads, group * most, D]
    k, v = _rows_of_keys(s, s["page_table"], keys)
    score = torch.matmul(mine, k.transpose(2, 3).contiguous()).mul_(scale).unflatten(2, (G, most))
    key = torch.arange(keys, device=dev)
    seen = (key < n_keys[:, None])[:, None].expand(B, most, -1)
    if c["causal"]:
        seen = seen & (key <= ((n_keys - n_new)[:, None] + torch.arange(most, device=dev))[..., None])
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    score.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = score.sum(-1, keepdim=True)
    out = torch.matmul(score.flatten(2, 3), v.contiguous()).unflatten(2, (G, most))
    stream = torch.repeat_interleave(torch.arange(B, device=dev), n_new, output_size=T)
    row = torch.arange(T, device=dev) - first[stream]
    top, total, out = (x[stream, :, :, row] for x in (top, total, out))  # [T, kv heads, group, 1 or D]
    del score, seen
    # the beginnings, each for all rows of its group
    k, v = _rows_of_keys(s, s["prefix_table"], max(s["shared"]))
    for g, P in enumerate(s["shared"]):
        a, b = sum(s["new"][:s["first"][g]]), sum(s["new"][:s["first"][g + 1]])
        rows = q[a:b].permute(1, 0, 2, 3).flatten(1, 2)  # [kv heads, rows * group, D]
        score = torch.matmul(rows, k[g, :, :P].transpose(1, 2).contiguous()).mul_(scale)
        high = score.amax(-1, keepdim=True)
        score.sub_(high).exp_()
        low = score.sum(-1, keepdim=True)
        part = torch.matmul(score, v[g, :, :P].contiguous())
        high, low, part = (x.unflatten(1, (b - a, G)).transpose(0, 1) for x in (high, low, part))
        both = torch.maximum(high, top[a:b])
        x, y = (high - both).exp(), (top[a:b] - both).exp()
        out[a:b] = (part * x + out[a:b] * y) / (low * x + total[a:b] * y)
        del score
    return out.flatten(1, 2).to(typ)


# ------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"layout": _exact_layout, "rotary": _exact_rotary, "prefix": _exact_prefix}[case["kind"]](case, s)


def _exact_layout(case, s):
    P, T = case["page"], s["tokens"]
    table, free, wanted, at = s["page_table"].tolist(), s["free_pages"].tolist(), 0, 0
    starts, after, positions, slots = [0], [], [0] * T, [-1] * T
    ahead = [0] * case["streams"]
    if case["groups"]:
        first, shared = s["group_starts"].tolist(), s["prefix_lens"].tolist()
        for g, n in enumerate(shared):
            ahead[first[g]:first[g + 1]] = [n] * (first[g + 1] - first[g])
    for b, (n, m) in enumerate(zip(s["new_lens"].tolist(), s["kv_lens"].tolist())):
        for key in range(m, m + n):
            if key % P == 0:
                table[b][key // P] = free[wanted] if wanted < len(free) else -1
                wanted += 1
            page = table[b][key // P]
            positions[at] = ahead[b] + key
            slots[at] = page * P + key % P if page >= 0 else -1
            at += 1
        starts.append(at)
        after.append(m + n)
    long = [torch.tensor(x, dtype=torch.int64, device=DEVICE) for x in (positions, slots)]
    return _int32(starts), _int32(after), *long, _int32(table), _int32([wanted])


def _exact_rotary(case, s):
    R, halves, f = case["rotary"], case["pairs"] == "halves", s["frequencies"]
    first = torch.arange(R // 2, device=DEVICE) * (1 if halves else 2)
    second = first + (R // 2 if halves else 1)
    p = s["positions"][:, None].expand(-1, R // 2)
    if s["sections"]:
        a, b, _ = s["sections"]
        pair, rows, cols = torch.arange(R // 2, device=DEVICE), *VIDEO
        p = torch.where(pair < a, p.div(rows * cols, rounding_mode="floor"), torch.where(pair < a + b, p.remainder(rows * cols).div(cols, rounding_mode="floor"), p.remainder(cols)))
    turn = torch.polar(torch.full_like(f, s["amplitude"]).expand(p.shape).contiguous(), p * f)[:, None]
    done = []
    for name in ("q", "k"):
        x = s[name].double()
        y = torch.complex(x[..., first], x[..., second]) * turn
        x[..., first], x[..., second] = y.real, y.imag
        done.append(x)
    if not case["page"]:
        return tuple(done)
    k_pages, v_pages = (s["cache"][n].double() for n in ("k_pages", "v_pages"))
    page, row = s["slots"] // case["page"], s["slots"] % case["page"]
    k_pages[page, row] = done[1]
    v_pages[page, row] = s["v"].double()
    return done[0], k_pages, v_pages


def _exact_prefix(case, s):
    D, Hk, G, page = case["dim"], case["kv_heads"], case["heads"] // case["kv_heads"], case["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE)
    at, group = 0, 0
    for b, (n, keys) in enumerate(zip(s["new"], s["keys"])):
        while b >= s["first"][group + 1]:
            group += 1
        P = s["shared"][group]
        tables = ((s["prefix_table"][group], P), (s["page_table"][b], keys))
        k, v = (torch.cat([s["cache"][name][t[:-(-m // page)].long()].flatten(0, 1)[:m] for t, m in tables]) for name in ("k_pages", "v_pages"))
        hidden = torch.zeros(n, P + keys, dtype=torch.bool, device=DEVICE)
        if case["causal"]:
            hidden |= torch.arange(P + keys, device=DEVICE) > P + keys - n + torch.arange(n, device=DEVICE)[:, None]
        for h in range(Hk):
            kh, vh = k[:, h].double(), v[:, h].double()
            rows = s["q"][at:at + n, h * G:(h + 1) * G].double().transpose(0, 1)
            t = torch.matmul(rows, kh.T / math.sqrt(D)).masked_fill(hidden, -math.inf)
            out[at:at + n, h * G:(h + 1) * G] = torch.matmul(torch.softmax(t, dim=-1), vh).transpose(0, 1)
        at += n
    return out
