"""Operators for several streams served in one batch, as cases with sizes: what a performance measurement runs.

Three operators of one attention layer over a batch of streams (requests), each stream with its own number of new tokens:

* ``norm``   every head of q and k through its RMS norm and its position rotation, K and V into their rows of a paged
             cache in the same pass (or, without a cache, q and k alone);
* ``paged``  attention of the streams' new tokens over that cache: single tokens, chunks and whole prompts, causal or
             not, with a window behind a few kept first keys;
* ``cross``  attention of the streams' queries to encoder states, whose number differs from request to request.

The sizes run from a handful of single tokens, where a call's own latency counts, to the chunks of 2640 tokens by 24 heads
over 13200 keys of this package's benchmark, all with ragged lengths.
"""
import math
import random

import torch

own = False
DEVICE = "cuda"
TYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16}


def listed():
    return [
        # one decoding step of a few streams: 24 rows, what counts is the latency of the call
        dict(name="norm_step", kind="norm", tokens=24, heads=16, kv_heads=4, dim=128, rotary=128, pairs="halves", page=16, type="bfloat16"),
        # q and k of a video chunk, 3 frames of 22 x 40 tokens, rotation by interleaved pairs, keys handed on as they are
        dict(name="norm_chunk", kind="norm", tokens=2640, heads=24, kv_heads=24, dim=128, rotary=128, pairs="interleaved", page=0, type="bfloat16"),
        # prompts of many streams at once, narrow heads of which a part is rotated, an odd number of tokens and an odd page
        dict(name="norm_prompt_odd", kind="norm", tokens=16381, heads=40, kv_heads=8, dim=64, rotary=32, pairs="halves", page=24, type="float16"),
        # a decoding step of three streams that have just begun: a few pages of keys
        dict(name="paged_step_small", kind="paged", streams=3, new=1, new_most=1, kv=40, kv_most=300, heads=16, kv_heads=4, dim=64, page=16,
             causal=True, window=0, sink=0, type="float16", spread=1),
        # a decoding step of 32 streams of any age: the caches are what is read
        dict(name="paged_step_long", kind="paged", streams=32, new=1, new_most=1, kv=500, kv_most=16384, heads=32, kv_heads=8, dim=128, page=16,
             causal=True, window=0, sink=0, type="bfloat16", spread=2),
        # single tokens, drafts of a few and chunks of prompts in one batch, over caches of every length
        dict(name="paged_mixed", kind="paged", streams=12, new=1, new_most=700, kv=300, kv_most=9000, heads=40, kv_heads=8, dim=128, page=32,
             causal=True, window=0, sink=0, type="bfloat16", spread=3),
        # the next piece of long prompts with a window behind four kept keys, narrow heads
        dict(name="paged_window", kind="paged", streams=4, new=900, new_most=2100, kv=4000, kv_most=9000, heads=16, kv_heads=16, dim=64, page=64,
             causal=True, window=1024, sink=4, type="float16", spread=4),
        # a video chunk over its cache: 2640 tokens, 13200 keys, every token sees every key
        dict(name="paged_video_chunk", kind="paged", streams=1, new=2640, new_most=2640, kv=13200, kv_most=13200, heads=24, kv_heads=24, dim=128,
             page=880, causal=False, window=0, sink=0, type="bfloat16", spread=5),
        # single queries to a few hundred encoder states
        dict(name="cross_step", kind="cross", streams=8, new=1, new_most=1, states=30, states_most=500, heads=16, kv_heads=16, dim=64, masked=False,
             type="float16", spread=6),
        # video chunks of three requests and their prompts, up to 512 text tokens
        dict(name="cross_video", kind="cross", streams=3, new=2640, new_most=2640, states=60, states_most=512, heads=24, kv_heads=24, dim=128,
             masked=False, type="bfloat16", spread=7),
        # many requests with as many lengths and states that are masked one by one, shared key heads
        dict(name="cross_masked", kind="cross", streams=17, new=3, new_most=900, states=100, states_most=2400, heads=20, kv_heads=4, dim=128, masked=True,
             type="bfloat16", spread=8),
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
        # the plain form of the attentions holds every product of a padded batch
        padded = case.get("streams", 0) * case["heads"] * case.get("new_most", 0) * case.get("kv_most", case.get("states_most", 0))
        if _cost(case) <= most and padded <= 9e8:
            return case


def _draw(rng):
    kind = rng.choice(["norm", "paged", "paged", "cross"])
    heads, kv_heads = _heads(rng)
    dim, typ = rng.choice([64, 128, 128]), rng.choice(["bfloat16", "bfloat16", "float16"])
    if kind == "norm":
        return dict(kind=kind, tokens=_log(rng, 1, 16384), heads=heads, kv_heads=kv_heads, dim=dim, rotary=rng.choice([dim, dim, dim // 2, 16]),
                    pairs=rng.choice(["halves", "interleaved"]), page=rng.choice([0, 1, 16, 24, 64]), type=typ)
    new_most = 1 if rng.random() < 0.4 else _log(rng, 2, 2700)
    case = dict(kind=kind, streams=_log(rng, 1, 64), new=max(1, int(new_most * rng.uniform(0.0, 1.0))), new_most=new_most, heads=heads,
                kv_heads=kv_heads, dim=dim, type=typ, spread=rng.randrange(1 << 16))
    if kind == "cross":
        most = _log(rng, 2, 4096)
        return dict(case, states=max(1, int(most * rng.uniform(0.0, 1.0))), states_most=most, masked=rng.random() < 0.4)
    most = new_most + _log(rng, 1, 16384)
    case.update(kv=max(new_most, int(most * rng.uniform(0.0, 1.0))), kv_most=most, page=rng.choice([1, 8, 16, 24, 32, 64, 880]),
                causal=rng.random() < 0.75, window=0, sink=0)
    if rng.random() < 0.25:
        case.update(window=_log(rng, 16, 4096), sink=rng.choice([0, 1, 4, 100]))
    return case


# ------------------------------------------------------------------------------------------------- sizes of a case
def _lengths(case, lo, hi, salt):
    """As many lengths between lo and hi as the case has streams, the longest and, where there are two, the shortest among them."""
    rng = random.Random(case["spread"] * 7 + salt)
    got = [_log(rng, lo, hi) for _ in range(case["streams"])]
    at = rng.randrange(case["streams"])
    got[at] = hi
    if case["streams"] > 1:
        got[at - 1] = lo
    return got


def _queries(case):
    return _lengths(case, case["new"], case["new_most"], 1)


def _keys(case):
    if case["kind"] == "cross":
        return _lengths(case, case["states"], case["states_most"], 2)
    return [max(n, m) for n, m in zip(_lengths(case, case["kv"], case["kv_most"], 2), _queries(case))]


def _visible(case, n, keys):
    """(pairs of query and key, keys that any query sees) of a stream with n new tokens."""
    if case["kind"] == "cross":
        return n * keys, keys
    pos = torch.arange(keys - n, keys, dtype=torch.float64)
    last = pos + 1 if case["causal"] else torch.full_like(pos, keys)
    if not case["window"]:
        return int(last.sum()), keys
    first = (pos - case["window"] + 1).clamp(min=0)
    sink = torch.minimum(torch.full_like(pos, case["sink"]), first)
    return int((last - first + sink).sum()), int(keys - first[0] + min(case["sink"], int(first[0])))


def work(case):
    D, Hq, Hk = case["dim"], case["heads"], case["kv_heads"]
    if case["kind"] == "norm":
        T, moved = case["tokens"], Hq + (2 if case["page"] else 1) * Hk
        return {"bytes": T * (2 * moved * D * 2 + case["rotary"] * 4 + (16 if case["page"] else 8)), "flops": T * (Hq + Hk) * (4 * D + 3 * case["rotary"])}
    rows, seen = list(zip(_queries(case), _keys(case))), [0, 0]
    for n, keys in rows:
        a, b = _visible(case, n, keys)
        seen = [seen[0] + a, seen[1] + b]
    return {"bytes": 2 * 2 * sum(n for n, _ in rows) * Hq * D + 2 * 2 * seen[1] * Hk * D, "flops": 4 * D * Hq * seen[0]}


# ------------------------------------------------------------------------------------------------- inputs
def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEVICE)


def _starts(lengths):
    return torch.tensor([0] + lengths, dtype=torch.int32).cumsum(0, dtype=torch.int32).to(DEVICE)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(int(seed))
    typ, D, Hq, Hk = TYPES[case["type"]], case["dim"], case["heads"], case["kv_heads"]
    if case["kind"] == "norm":
        T, R = case["tokens"], case["rotary"]
        # what a projection of q, k and v leaves: one row a token, channels of different size
        rows = (_randn(gen, T, (Hq + 2 * Hk) * D) * (0.2 + _randn(gen, (Hq + 2 * Hk) * D).abs())).to(typ)
        q, k, v = (x.unflatten(1, (-1, D)) for x in rows.split([Hq * D, Hk * D, Hk * D], dim=1))
        limit = 32768
        angles = torch.arange(limit, dtype=torch.float64, device=DEVICE)[:, None] * 10000.0 ** (
            -torch.arange(0, R, 2, dtype=torch.float64, device=DEVICE) / R)
        state = dict(case=case, q=q, k=k, v=v, q_weight=(1 + 0.1 * _randn(gen, D)).to(typ), k_weight=(1 + 0.1 * _randn(gen, D)).to(typ), eps=1e-6,
                     cos=angles.cos().float(), sin=angles.sin().float(), positions=torch.randint(0, limit, (T,), generator=gen, device=DEVICE))
        if case["page"]:
            pages = -(-T // case["page"]) + 3
            state["cache"] = {name: _randn(gen, pages, case["page"], Hk, D).to(typ) for name in ("k_pages", "v_pages")}
            state["slots"] = torch.randperm(pages * case["page"], generator=gen, device=DEVICE)[:T]
        return state
    new, keys = _queries(case), _keys(case)
    T = sum(new)
    # behind a norm of every head: some channels larger than others, products of q and k of about two
    channels = 0.5 + _randn(gen, D).abs()
    state = dict(case=case, q=(2 * _randn(gen, T, Hq, D) * channels).to(typ), q_starts=_starts(new), new=new, keys=keys,
                 max_new=max(new), max_keys=max(keys))
    if case["kind"] == "cross":
        state.update(k=(_randn(gen, sum(keys), Hk, D) / channels).to(typ), v=_randn(gen, sum(keys), Hk, D).to(typ), k_starts=_starts(keys))
        if case["masked"]:
            state["key_mask"] = torch.rand(sum(keys), generator=gen, device=DEVICE) < 0.8
        return state
    page = case["page"]
    held = [-(-n // page) for n in keys]
    pages = sum(held) + 2
    order = torch.randperm(pages, generator=gen, device=DEVICE).int()
    width = max(held) + 1
    at = torch.tensor([0] + held[:-1], device=DEVICE).cumsum(0)[:, None] + torch.arange(width, device=DEVICE)
    table = order[at.clamp(max=pages - 1)]
    state["page_table"] = torch.where(torch.arange(width, device=DEVICE) < torch.tensor(held, device=DEVICE)[:, None], table, 0).contiguous()
    state["cache"] = {"k_pages": (_randn(gen, pages, page, Hk, D) / channels).to(typ), "v_pages": _randn(gen, pages, page, Hk, D).to(typ)}
    state["kv_lens"] = torch.tensor(keys, dtype=torch.int32, device=DEVICE)
    return state


# ------------------------------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if own:
        return _run_own(state)
    return _plain_norm(state) if case["kind"] == "norm" else _plain_attention(state)


def _run_own(s):
    c = s["case"]
    if c["kind"] == "norm":
        from longlive_amd.utils.paged_kv import head_norm_rope_paged
        from longlive_amd.utils.rope import head_norm_rope
        interleaved = c["pairs"] == "interleaved"
        if "cache" in s:
            q = head_norm_rope_paged(s["q"], s["k"], s["v"], s["cache"], s["slots"], s["q_weight"], s["k_weight"], s["eps"], s["cos"], s["sin"],
                                     s["positions"], interleaved=interleaved)
            return q, s["cache"]["k_pages"], s["cache"]["v_pages"]
        return head_norm_rope(s["q"], s["k"], s["q_weight"], s["k_weight"], s["eps"], s["cos"], s["sin"], s["positions"], interleaved=interleaved)
    if c["kind"] == "paged":
        from longlive_amd.utils.paged_kv import paged_attention
        return paged_attention(s["q"], s["cache"], s["page_table"], s["kv_lens"], s["q_starts"], causal=c["causal"], window=c["window"] or None,
                               sink_tokens=c["sink"], max_q_len=s["max_new"], max_kv_len=s["max_keys"])
    from longlive_amd.utils.cross_attention import ragged_cross_attention
    return ragged_cross_attention(s["q"], s["k"], s["v"], s["q_starts"], s["k_starts"], key_mask=s.get("key_mask"), max_q_len=s["max_new"],
                                  max_k_len=s["max_keys"])


def _plain_rotate(x, weight, s):
    """Every head of x [T, H, D]: norm, weight, rotation of the first columns; in 32 bits."""
    x = x.float()
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + s["eps"]) * weight.float()
    R = s["case"]["rotary"]
    cos, sin = s["cos"][s["positions"]][:, None], s["sin"][s["positions"]][:, None]
    if s["case"]["pairs"] == "halves":
        a, b = x[..., :R // 2], x[..., R // 2:R]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., R:]], dim=-1)
    a, b = x[..., 0:R:2], x[..., 1:R:2]
    return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2), x[..., R:]], dim=-1)


def _plain_norm(s):
    q, k = (_plain_rotate(s[n], s[n + "_weight"], s).to(s[n].dtype) for n in ("q", "k"))
    if "cache" not in s:
        return q, k
    for pages, new in ((s["cache"]["k_pages"], k), (s["cache"]["v_pages"], s["v"])):
        pages.view(-1, *pages.shape[2:])[s["slots"]] = new
    return q, s["cache"]["k_pages"], s["cache"]["v_pages"]


def _plain_attention(s):
    c = s["case"]
    typ, dev, T, B, most, G = s["q"].dtype, s["q"].device, s["q"].shape[0], c["streams"], s["max_new"], c["heads"] // c["kv_heads"]
    first, n_new = s["q_starts"][:-1].long(), s["q_starts"].diff().long()
    # the padded batch: queries [B, kv heads, group * most, D], keys and values [B, kv heads, keys, D]
    at = first[:, None] + torch.arange(most, device=dev)
    q = s["q"].float()[at.clamp(max=T - 1)].unflatten(2, (c["kv_heads"], G)).permute(0, 2, 3, 1, 4).flatten(2, 3)
    key = torch.arange(s["max_keys"], device=dev)
    if c["kind"] == "paged":
        page = c["page"]
        entry = s["page_table"].long()[:, key // page]
        k, v = (s["cache"][n][entry, key % page].float() for n in ("k_pages", "v_pages"))
        n_keys = s["kv_lens"].long()
        pos = (n_keys - n_new)[:, None] + torch.arange(most, device=dev)
        seen = (key < n_keys[:, None])[:, None].expand(B, most, -1)
        if c["causal"]:
            seen = seen & (key <= pos[..., None])
        if c["window"]:
            seen = seen & ((key > pos[..., None] - c["window"]) | (key < c["sink"]))
    else:
        n_keys, start = s["k_starts"].diff().long(), s["k_starts"][:-1].long()
        row = (start[:, None] + key).clamp(max=s["k"].shape[0] - 1)
        k, v = s["k"][row].float(), s["v"][row].float()
        seen = key < n_keys[:, None]
        if c["masked"]:
            seen = seen & s["key_mask"][row]
        seen = seen[:, None].expand(B, most, -1)
    k, v = k.permute(0, 2, 3, 1).contiguous(), v.transpose(1, 2).contiguous()
    score = torch.matmul(q, k).mul_(c["dim"] ** -0.5).unflatten(2, (G, most))
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    score.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = score.sum(-1, keepdim=True)
    out = torch.matmul(score.flatten(2, 3), v).unflatten(2, (G, most)) / torch.where(total == 0, 1.0, total)
    out = out.permute(0, 3, 1, 2, 4).flatten(2, 3)  # [B, most, heads, D]
    stream = torch.repeat_interleave(torch.arange(B, device=dev), n_new, output_size=T)
    return out[stream, torch.arange(T, device=dev) - first[stream]].to(typ)


# ------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return _exact_norm(case, s) if case["kind"] == "norm" else _exact_attention(case, s)


def _exact_norm(case, s):
    R, halves = case["rotary"], case["pairs"] == "halves"
    first = torch.arange(R // 2, device=DEVICE) * (1 if halves else 2)
    second = first + (R // 2 if halves else 1)
    cos, sin = (s[n].double()[s["positions"]].unsqueeze(1) for n in ("cos", "sin"))
    done = []
    for name in ("q", "k"):
        x = s[name].double()
        x = s[name + "_weight"].double() * x / (x.pow(2).sum(-1, keepdim=True) / case["dim"] + s["eps"]).sqrt()
        a, b = x[..., first], x[..., second]
        x[..., first], x[..., second] = cos * a - sin * b, sin * a + cos * b
        done.append(x)
    if not case["page"]:
        return tuple(done)
    k_pages, v_pages = (s["cache"][n].double() for n in ("k_pages", "v_pages"))
    page, row = s["slots"] // case["page"], s["slots"] % case["page"]
    k_pages[page, row] = done[1]
    v_pages[page, row] = s["v"].double()
    return done[0], k_pages, v_pages


def _exact_attention(case, s):
    D, Hk, G = case["dim"], case["kv_heads"], case["heads"] // case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE)
    q_at = k_at = 0
    for b, (n, keys) in enumerate(zip(s["new"], s["keys"])):
        j, i = torch.arange(keys, device=DEVICE), torch.arange(n, device=DEVICE)[:, None]
        hidden = torch.zeros(n, keys, dtype=torch.bool, device=DEVICE)
        if case["kind"] == "paged":
            table = s["page_table"][b, :-(-keys // case["page"])].long()
            k, v = (s["cache"][name][table].flatten(0, 1)[:keys] for name in ("k_pages", "v_pages"))
            pos = keys - n + i
            if case["causal"]:
                hidden |= j > pos
            if case["window"]:
                hidden |= (j <= pos - case["window"]) & (j >= case["sink"])
        else:
            k, v = s["k"][k_at:k_at + keys], s["v"][k_at:k_at + keys]
            if case["masked"]:
                hidden |= ~s["key_mask"][k_at:k_at + keys]
        for h in range(Hk):
            kh, vh = k[:, h].double(), v[:, h].double()
            for g in range(G):
                t = (s["q"][q_at:q_at + n, h * G + g].double() @ kh.T / math.sqrt(D)).masked_fill(hidden, -math.inf)
                # a row that sees nothing has no weights, and zeros for its result
                w = torch.softmax(t, dim=-1).masked_fill(hidden, 0.0).nan_to_num(0.0)
                out[q_at:q_at + n, h * G + g] = w @ vh
        q_at, k_at = q_at + n, k_at + keys
    return out
