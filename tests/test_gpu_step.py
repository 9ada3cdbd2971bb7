"""Operators around a step of several streams on the GPU: its layout on the device, rotation by positions, attention over a shared beginning, and a
run of them together; against plain forms, whose allowed errors count roundings."""
import pytest
import torch

import step_reference as step_ref
import streams_reference as ref
from longlive_amd.utils.paged_kv import (initialize_paged_kv_cache, lay_out_step, paged_attention, rotate_by_position_paged,
                                         shared_prefix_attention)
from longlive_amd.utils.rope import head_norm_rope, rotary_frequencies, rotate_by_position, video_frequencies

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def randn(seed, *shape, dtype=BF16, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def int32(values, device=None):
    return torch.tensor(values, dtype=torch.int32, device=device)


def starts(lengths, first=0):
    return torch.tensor([first] + list(lengths), dtype=torch.int32).cumsum(0, dtype=torch.int32)


def close(got, want, error, what=""):
    got = got.detach().cpu().double()
    off = (got - want).abs()
    assert torch.isfinite(got).all(), what
    worst = (off / error.clamp(min=1e-300)).max().item() if off.numel() else 0.0
    assert (off <= error).all(), f"{what}: {worst:.2f} of the allowed error, at {(off > error).nonzero()[:3].tolist()}"


# ------------------------------------------------------------------------------------------------ layout
def check_layout(gpu, new, before, width, page, spare=3, extra=0, prefix_lens=None, group_starts=None, cursor=None, in_place=False, seed=1):
    g = torch.Generator().manual_seed(seed)
    held = [min(-(-max(m, 0) // page), width) for m in before]
    wanted = sum(max(min(-(-(max(m, 0) + max(n, 0)) // page), width) - h, 0) for n, m, h in zip(new, before, held))
    order = torch.randperm(sum(held) + max(wanted + spare, 0) + (cursor or 0), generator=g).tolist()
    table = [[order.pop() for _ in range(h)] + [-1] * (width - h) for h in held]
    free = order
    tokens = max(sum(max(n, 0) for n in new) + extra, 0)
    want = step_ref.step_layout(new, before, table, free, page, tokens, prefix_lens, group_starts, cursor or 0)
    on = torch.full((len(new), width + 3), 77, dtype=torch.int32, device=gpu)     # rows within wider ones
    on[:, :width] = int32(table, gpu).view(len(new), width)
    lens = int32(before, gpu)
    at = None if cursor is None else int32([cursor], gpu)
    got = lay_out_step(int32(new, gpu), lens, on[:, :width], int32(free, gpu), page, tokens, prefix_lens=None if prefix_lens is None else int32(prefix_lens, gpu),
                       group_starts=None if group_starts is None else int32(group_starts, gpu), cursor=at, kv_lens_out=lens if in_place else None)
    assert [got.q_starts.tolist(), got.kv_lens.tolist(), got.positions.tolist(), got.slots.tolist(), got.pages_wanted.tolist()] == [*want[:4], [want[4]]]
    assert on[:, :width].tolist() == want[5] and (on[:, width:] == 77).all()
    assert (got.kv_lens is lens) == in_place and lens.tolist() == (want[1] if in_place else before)
    if cursor is not None:
        assert at.tolist() == [want[6]]
    return got


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("cursor", [None, 2])
@pytest.mark.parametrize("new,before,width,page", [
    ([1], [0], 1, 1), ([1], [15], 2, 16), ([1], [16], 2, 16), ([3, 0, 5, 1], [0, 7, 14, 33], 4, 16), ([0, 0], [5, 0], 2, 8), ([40, 1, 7], [3, 24, 0], 60, 1),
    ([100, 2000, 1], [5, 0, 880], 4, 880), ([4000, 1, 900, 300], [7, 100, 9, 0], 300, 16), ([5000], [1000], 800, 8)])
def test_layout(gpu, new, before, width, page, cursor, in_place):
    check_layout(gpu, new, before, width, page, cursor=cursor, in_place=in_place)


@pytest.mark.parametrize("streams", [63, 64, 65, 255, 256, 257, 1023, 1024, 1025, 5000])
@pytest.mark.parametrize("most", [2, 9])
def test_layout_of_many_streams(gpu, streams, most):
    g = torch.Generator().manual_seed(streams)
    new = torch.randint(0, most, (streams,), generator=g).tolist()
    before = torch.randint(0, 70, (streams,), generator=g).tolist()
    cuts = sorted(torch.randint(0, streams + 1, (9,), generator=g).tolist())
    check_layout(gpu, new, before, 9, 8, prefix_lens=[5, 0, 1000, 7, -3, 2 ** 31 - 1, 12, 1], group_starts=cuts, cursor=1, in_place=streams % 2 == 0)


def test_layout_lists_and_tables_that_end(gpu):
    check_layout(gpu, [30, 30, 30], [5, 0, 8], 8, 8, spare=-5)                # fewer free pages than are wanted
    check_layout(gpu, [30, 30, 3000], [5, 0, 8], 8, 8, spare=-1, cursor=4)
    check_layout(gpu, [30, 30], [100, 60], 8, 8)                              # tables that are too narrow
    check_layout(gpu, [3, 3, 3], [1, 2, 3], 1, 8, spare=-100)                 # no free pages at all
    check_layout(gpu, [5, 6, 7], [1, 2, 3], 4, 4, extra=9)                    # rows behind the last
    check_layout(gpu, [5, 6, 7, 8], [1, 2, 3, 2 ** 31 - 4], 4, 4, extra=-12)  # rows that are too few
    check_layout(gpu, [5, 6, 7], [1, 2, 3], 4, 4, extra=-18)                  # none
    check_layout(gpu, [2 ** 31 - 1, 2 ** 31 - 1, 4], [0, 3, 4], 4, 4, extra=100 - 2 * (2 ** 31 - 1) - 4, spare=3 - 12)
    check_layout(gpu, [-4, 3, -(2 ** 31)], [-7, -1, 3], 4, 4)                 # negative lengths are none
    check_layout(gpu, [9, 1], [2 ** 31 - 4, 2 ** 31 - 1], 2, 16)              # lengths end at 2^31 - 1
    check_layout(gpu, [1, 1], [3, 5], 4, 4, prefix_lens=[100])                # one group of all streams
    check_layout(gpu, [1, 1], [3, 5], 4, 4, prefix_lens=[100, 50], group_starts=[1, 1, 2])
    check_layout(gpu, [1, 1], [3, 5], 4, 4, cursor=0, spare=-1)


def test_layout_without_streams_or_tokens(gpu):
    none = torch.zeros(0, dtype=torch.int32, device=gpu)
    got = lay_out_step(none, none, none.view(0, 4), none, 16, 5)
    assert got.q_starts.tolist() == [0] and got.slots.tolist() == [-1] * 5 and got.positions.tolist() == [0] * 5 and got.pages_wanted.tolist() == [0]
    got = lay_out_step(int32([2], gpu), int32([3], gpu), none.view(1, 0), none, 16, 2)   # no table
    assert got.slots.tolist() == [-1, -1] and got.positions.tolist() == [3, 4] and got.pages_wanted.tolist() == [0]
    got = lay_out_step(int32([2], gpu), int32([3], gpu), int32([[0]], gpu), none, 16, 0)
    assert got.q_starts.tolist() == [0, 0] and got.kv_lens.tolist() == [3]


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("tokens", [4, 3000])
def test_layouts_that_would_overwrite_what_they_read_are_refused(gpu, tokens, native, monkeypatch):
    from longlive_amd import _native
    if not native:   # by way of ctypes
        monkeypatch.setattr(_native, "host", lambda: type("None", (), {"step_layout": staticmethod(lambda *a: None)}))
    memory = torch.arange(100, dtype=torch.int32, device=gpu)
    new, held, table, free, cursor = memory[:4], memory[4:8], memory[10:34].view(4, 6)[:, :4], memory[40:60], memory[60:61]
    ok = dict(new_lens=new, kv_lens=held, page_table=table, free_pages=free, page_size=16, num_tokens=tokens, cursor=cursor)
    for bad in (dict(kv_lens_out=new), dict(kv_lens_out=memory[5:9]), dict(kv_lens_out=memory[1:5]), dict(kv_lens_out=memory[57:61]), dict(kv_lens_out=memory[8:12]), dict(cursor=memory[2:3]),
                dict(cursor=memory[6:7]), dict(cursor=memory[45:46]), dict(cursor=memory[16:17]), dict(page_table=memory[6:30].view(4, 6)[:, :4]), dict(free_pages=memory[20:40])):
        with pytest.raises(ValueError, match="overlap"):
            lay_out_step(**{**ok, **bad})
    torch.cuda.synchronize()
    assert memory.tolist() == list(range(100))
    # side by side, the cursor between two rows of the table
    got = lay_out_step(**{**ok, "cursor": memory[14:15], "kv_lens_out": held})
    n = [0, 1, 2, 3] if tokens == 3000 else [0, 1, 2, 1]
    assert got.kv_lens is held and memory[:8].tolist() == [0, 1, 2, 3] + [m + i for m, i in zip([4, 5, 6, 7], n)] and memory[40:60].tolist() == list(range(40, 60))


@pytest.mark.parametrize("tokens", [7, 3000])
def test_steps_that_a_graph_replays_go_on_from_one_another(gpu, tokens):
    page, new, lens = 4, [1, 0, 3, 1, 1], [0, 9, 4, 3, 2]
    if tokens > 7:
        new[2] = 2500
    steps, width = 4, (max(new) * 4 + 20) // page
    held = [-(-m // page) for m in lens]
    table, at = [], 0
    for h in held:
        table.append(list(range(at, at + h)) + [-1] * (width - h))
        at += h
    free = list(range(at, at + sum(new) * steps))
    on, kv, cursor, new_lens, pages = int32(table, gpu), int32(lens, gpu), int32([0], gpu), int32(new, gpu), int32(free, gpu)

    def step():
        return lay_out_step(new_lens, kv, on, pages, page, tokens, cursor=cursor, kv_lens_out=kv)

    kept = [t.clone() for t in (on, kv, cursor)]
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for t, before in zip((on, kv, cursor), kept):
        t.copy_(before)
    taken = 0
    for _ in range(steps):
        graph.replay()
        torch.cuda.synchronize()
        want = step_ref.step_layout(new, lens, table, free, page, tokens, cursor=taken)
        assert [got.q_starts.tolist(), got.kv_lens.tolist(), got.positions.tolist(), got.slots.tolist()] == list(want[:4])
        assert on.tolist() == want[5] and cursor.tolist() == [want[6]]
        lens, table, taken = want[1], want[5], want[6]


# ------------------------------------------------------------------------------------------------ rotation by positions
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("T,Hq,Hk,D,R,dtype", [
    (1, 1, 1, 128, 128, BF16), (5, 4, 2, 64, 64, F16), (37, 7, 1, 64, 32, BF16), (300, 24, 24, 128, 128, BF16), (33, 3, 3, 128, 16, F16),
    (9, 5, 5, 8, 8, BF16), (11, 6, 2, 96, 64, BF16), (64, 2, 2, 256, 256, BF16), (7, 3, 1, 200, 136, F16), (2049, 40, 8, 128, 64, F16)])
def test_rotation_by_positions(gpu, T, Hq, Hk, D, R, dtype, interleaved):
    q, k = randn(1, T, Hq, D, dtype=dtype), randn(2, T, Hk, D, dtype=dtype, scale=3.0)
    f = rotary_frequencies(R, scaling="base", factor=4.0) if R > 2 else rotary_frequencies(R)
    positions = torch.randint(-(1 << 22), 1 << 31, (T,), generator=torch.Generator().manual_seed(5))
    positions[0] = 0
    got = rotate_by_position(q.to(gpu), k.to(gpu), positions.to(gpu), f.to(gpu), interleaved=interleaved, amplitude=1.25)
    for x, y in zip((q, k), got):
        assert y.dtype == dtype and y.shape == x.shape
        close(y, *step_ref.rotate(x, None, 0.0, f, positions, interleaved, 1.25))
    assert torch.equal(got[0][..., R:].cpu(), q[..., R:])


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_rotation_behind_norms(gpu, dtype):
    q, k = randn(1, 77, 6, 128, dtype=dtype), randn(2, 77, 2, 128, dtype=dtype)
    wq, wk, f = randn(3, 128, dtype=dtype), randn(4, 128, dtype=torch.float32), rotary_frequencies(64)
    got = rotate_by_position(q.to(gpu), k.to(gpu), None, f.to(gpu), q_weight=wq.to(gpu), k_weight=wk.to(gpu), eps=1e-5)
    for x, w, y in ((q, wq, got[0]), (k, wk, got[1])):
        close(y, *step_ref.rotate(x, w, 1e-5, f, None, True))


@pytest.mark.parametrize("grid", [(22, 40), (1, 1), (3, 7)])
@pytest.mark.parametrize("interleaved", [True, False])
def test_rotation_by_places_in_a_video(gpu, grid, interleaved):
    f, sections = video_frequencies(128)
    T = 200
    q, k = randn(1, T, 3, 128), randn(2, T, 1, 128)
    positions = torch.randint(-5000, 1 << 20, (T,), generator=torch.Generator().manual_seed(2))
    positions[:4] = torch.tensor([0, -1, (1 << 32) + 12345, -(1 << 33) - 7])
    got = rotate_by_position(q.to(gpu), k.to(gpu), positions.to(gpu), f.to(gpu), grid=grid, sections=sections, interleaved=interleaved)
    for x, y in zip((q, k), got):
        close(y, *step_ref.rotate(x, None, 0.0, f, positions, interleaved, 1.0, grid, sections))


def test_rotation_of_a_video_chunk_is_the_tables(gpu):
    from longlive_amd.utils.rope import build_rope_angles, rope_cos_sin
    q, k = randn(1, 3 * 880, 4, 128).to(gpu), randn(2, 3 * 880, 4, 128).to(gpu)
    cos, sin = rope_cos_sin(build_rope_angles(), 3, 22, 40, start_frame=9, device=gpu)
    want = head_norm_rope(q, k, None, None, 1e-6, cos, sin)
    f, sections = video_frequencies(128, device=gpu)
    got = rotate_by_position(q, k, torch.arange(9 * 880, 12 * 880, device=gpu), f, grid=(22, 40), sections=sections)
    for x, a, b in zip((q, k), got, want):
        # each within half a bf16 step of the exact value, give or take 2^-21 of the pair's size
        size = x.float().unflatten(-1, (-1, 2)).abs().sum(-1, keepdim=True).expand(-1, -1, -1, 2).flatten(-2)
        assert ((a.float() - b.float()).abs() <= 2.0 ** -7 * torch.maximum(a.float().abs(), b.float().abs()) + 2.0 ** -21 * size).all()


@pytest.mark.parametrize("T,Hq,Hk,D,page,dtype", [(1, 8, 2, 128, 16, BF16), (50, 4, 4, 64, 3, F16), (129, 6, 3, 128, 1, BF16)])
def test_rotation_into_pages(gpu, T, Hq, Hk, D, page, dtype):
    rows = randn(1, T, (Hq + 2 * Hk) * D, dtype=dtype)
    split = lambda t: (x.unflatten(1, (-1, D)) for x in t.split([Hq * D, Hk * D, Hk * D], dim=1))  # noqa: E731  views of one projection
    (q, k, v), (qd, kd, vd) = split(rows), split(rows.to(gpu))
    f, pages = rotary_frequencies(D), -(-T // page) + 2
    cache = {n: randn(7, pages, page, Hk, D, dtype=dtype).to(gpu) for n in ("k_pages", "v_pages")}
    before = {n: t.cpu().clone() for n, t in cache.items()}
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(1))[:T]
    slots[T // 2] = -1 if T > 1 else slots[0]
    positions = torch.arange(T) * 1000
    out = qd.clone()
    assert rotate_by_position_paged(out, kd, vd, cache, slots.to(gpu), positions.to(gpu), f.to(gpu), interleaved=False, out=out) is out   # in place of q
    close(out, *step_ref.rotate(q, None, 0.0, f, positions, False))
    want, error = step_ref.rotate(k, None, 0.0, f, positions, False)
    ok = slots >= 0
    for name, new, err in (("k_pages", want, error), ("v_pages", v.double(), torch.zeros_like(error))):
        now = cache[name].cpu().flatten(0, 1)
        close(now[slots[ok]], new[ok], err[ok], name)
        left = torch.ones(pages * page, dtype=torch.bool)
        left[slots[ok]] = False
        assert torch.equal(now[left], before[name].flatten(0, 1)[left]), name


def test_rotation_of_nothing_and_by_nothing(gpu):
    q, f = randn(1, 3, 4, 64).to(gpu), rotary_frequencies(64, device=gpu)
    got = rotate_by_position(q[:0], q[:0], None, f)
    assert got[0].shape == got[1].shape == (0, 4, 64)
    got = rotate_by_position(q, q, None, f[:0])      # no pairs
    assert torch.equal(got[0], q) and torch.equal(got[1], q)
    cache = initialize_paged_kv_cache(1, 0, 16, 4, 64, gpu)[0]
    got = rotate_by_position_paged(q, q, q, cache, torch.full((3,), -1, device=gpu), None, f)
    close(got, *step_ref.rotate(q.cpu(), None, 0.0, f.cpu(), None, True))


# ------------------------------------------------------------------------------------------------ shared beginnings
def batch(seed, new, keys, shared, Hq, Hk, D, page, dtype, fill=None, scale=1.5):
    """(q, cache, prefix_table, prefix_lens, page_table, kv_lens, q_starts) on the CPU: pages in any order, rows that hold no key filled with `fill`."""
    g = torch.Generator().manual_seed(seed)
    lens = list(keys) + list(shared)
    held = [-(-n // page) for n in lens]
    pages = sum(held) + 2
    order = torch.randperm(pages, generator=g).int()
    cache = {n: randn(seed + i, pages, page, Hk, D, dtype=dtype) for i, n in enumerate(("k_pages", "v_pages"), 1)}
    used = torch.zeros(pages, page, dtype=torch.bool)
    at, tables = 0, []
    for part, more in ((held[:len(keys)], 1), (held[len(keys):], 0)):
        table = torch.full((len(part), max(part + [1]) + more), 1 << 30, dtype=torch.int32)
        for b, n in enumerate(part):
            table[b, :n] = order[at:at + n]
            at += n
        tables.append(table)
    for table, part in zip(tables, (keys, shared)):
        for b, n in enumerate(part):
            for i in range(-(-n // page)):
                used[table[b, i], :min(page, n - i * page)] = True
    if fill is not None:
        for t in cache.values():
            t[~used] = fill
    return randn(seed + 5, sum(new), Hq, D, dtype=dtype, scale=scale), cache, tables[1], int32(shared), tables[0], int32(keys), starts(new)


def attend(gpu, b, group_starts=None, causal=True, **kw):
    q, cache, *rest = b
    return shared_prefix_attention(q.to(gpu), {n: t.to(gpu) for n, t in cache.items()}, *(t.to(gpu) for t in rest),
                                   group_starts=None if group_starts is None else int32(group_starts, gpu), causal=causal, **kw)


def check_shared(gpu, b, group_starts=None, causal=True, what="", told=True, **kw):
    new, keys, shared = b[6].diff().tolist(), b[5].tolist(), b[3].tolist()
    if told:
        kw = dict(dict(max_q_len=max(new), max_kv_len=max(keys), max_prefix_len=max(shared + [0])), **kw)
    got = attend(gpu, b, group_starts, causal, **kw)
    want, error, _ = step_ref.shared_prefix(*b, None if group_starts is None else int32(group_starts), causal, kw.get("softmax_scale") or b[0].shape[-1] ** -0.5)
    close(got, want, error, what)
    return got


TYPES = [(64, F16), (128, BF16), (128, F16), (64, BF16)]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D,dtype", TYPES)
@pytest.mark.parametrize("new,keys,shared,groups,Hq,Hk,page", [
    ([1], [1], [1], None, 1, 1, 1),
    ([1, 1, 1], [40, 300, 1], [129], None, 8, 2, 16),
    ([1, 5, 0, 70], [257, 5, 33, 200], [500, 63], [0, 2, 4], 4, 4, 24),
    ([130, 1, 64], [130, 64, 1000], [64, 65], [0, 1, 3], 5, 1, 7),
    ([33, 2], [65, 2], [700], None, 14, 2, 64),
    ([300], [700], [1000], None, 3, 3, 880)])
def test_shared_beginnings(gpu, new, keys, shared, groups, Hq, Hk, page, D, dtype, causal):
    check_shared(gpu, batch(11, new, keys, shared, Hq, Hk, D, page, dtype, fill=float("nan")), groups, causal)


@pytest.mark.parametrize("D,dtype", TYPES)
@pytest.mark.parametrize("shared", [1, 63, 64, 127, 128, 191, 1000, 4099])
@pytest.mark.parametrize("streams,Hq,Hk", [(2, 4, 4), (9, 16, 2), (70, 3, 3), (40, 8, 1)])
def test_single_tokens_that_share_a_beginning(gpu, streams, Hq, Hk, shared, D, dtype):
    keys = [1 + 7 * b % 90 for b in range(streams)]
    check_shared(gpu, batch(21, [1] * streams, keys, [shared], Hq, Hk, D, 16, dtype, fill=float("nan")))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D,dtype", [(64, F16), (128, BF16)])
@pytest.mark.parametrize("new", [[4] * 30, [2, 3, 1, 0, 9, 1, 1, 40], [1] * 20 + [150] + [1] * 20, [60, 70, 64, 33]])
def test_a_few_tokens_each_over_a_long_beginning(gpu, new, D, dtype, causal):
    keys = [n + 11 * b % 300 for b, n in enumerate(new)]
    check_shared(gpu, batch(31, new, keys, [3001], 8, 2, D, 32, dtype, fill=float("nan")), None, causal)


@pytest.mark.parametrize("D,dtype", [(64, F16), (128, BF16)])
def test_long_own_keys_behind_a_beginning(gpu, D, dtype):
    check_shared(gpu, batch(41, [1, 2, 1], [4000, 2, 2600], [3000], 8, 2, D, 16, dtype))
    check_shared(gpu, batch(42, [200, 129], [2000, 129], [2500], 2, 1, D, 24, dtype, fill=float("nan")))


def test_groups_of_all_kinds(gpu):
    # empty groups, streams outside every group, streams without tokens, groups without a beginning, more streams than a wave has lanes
    g = torch.Generator().manual_seed(3)
    new = torch.randint(0, 4, (150,), generator=g).tolist()
    new[70] = 140
    keys = [n + int(k) for n, k in zip(new, torch.randint(0, 200, (150,), generator=g))]
    cuts = [2, 2, 50, 50, 69, 72, 140, 145]
    shared = [300, 700, 1, 0, 900, 1500, 20]
    b = batch(51, new, keys, shared, 4, 2, 64, 16, BF16, fill=float("nan"))
    check_shared(gpu, b, cuts)
    check_shared(gpu, b, cuts, causal=False)
    check_shared(gpu, b, cuts, told=False)


def test_more_groups_than_a_wave_has_lanes(gpu):
    new = [1 + b % 3 for b in range(200)]
    keys = [n + b % 50 for b, n in enumerate(new)]
    check_shared(gpu, batch(52, new, keys, [130 + b % 200 for b in range(100)], 6, 2, 128, 8, F16, fill=float("nan")), list(range(0, 202, 2)))


def test_rows_that_see_the_beginning_only_and_rows_that_see_nothing(gpu):
    # more new tokens than own keys: the first of them sit before the first own key; none at all; tables of holes
    b = batch(61, [5, 3, 4, 2], [2, 0, 20, 6], [200, 0], 4, 2, 64, 8, BF16, fill=float("nan"))
    b[4][3] = -1
    got = check_shared(gpu, b, [0, 3, 4])
    assert (got[:8] != 0).any() and (got[12:] == 0).all()
    b[2][0] = -1
    got = check_shared(gpu, b, [0, 3, 4])
    assert (got[:3] == 0).all() and (got[3:5] != 0).any() and (got[5:8] == 0).all()


@pytest.mark.parametrize("new", [[3, 1, 1], [90, 70, 1], [1, 1, 1]])
def test_holes_in_both_tables(gpu, new):
    b = batch(62, new, [300, 120, 40], [500], 8, 4, 128, 16, BF16)
    for table, entry in ((b[2], (0, 0)), (b[2], (0, 7)), (b[2], (0, 8)), (b[2], (0, 9)), (b[2], (0, 10)), (b[2], (0, 11)), (b[4], (1, 0)), (b[4], (0, 3))):
        b[1]["k_pages"][table[entry]] = b[1]["v_pages"][table[entry]] = float("nan")
        table[entry] = -1 if entry[1] % 2 else b[1]["k_pages"].shape[0]
    check_shared(gpu, b)
    check_shared(gpu, b, causal=False)


def test_later_tokens_that_are_not_finite(gpu):
    # V of a token that its stream's earlier tokens do not see; and of a shared key, which all of the group see and no one else
    for new in ([3, 2, 1], [70, 40, 30]):
        b = batch(63, new, [n + 100 for n in new], [300, 200], 2, 1, 64, 8, BF16)
        last = b[5][0].item() - 1
        want, error, _ = step_ref.shared_prefix(*b, int32([0, 2, 3]), True, 64 ** -0.5)   # rows that do not see it: what it is makes no difference
        b[1]["v_pages"][b[4][0, last // 8], last % 8, 0, 5] = float("inf")
        got = attend(gpu, b, [0, 2, 3])
        assert torch.isinf(got[new[0] - 1, :, 5]).all()
        keep = torch.ones_like(want, dtype=torch.bool)
        keep[new[0] - 1, :, 5] = False
        close(torch.where(keep, got.cpu().double(), 0.0), torch.where(keep, want, 0.0), torch.where(keep, error, 1.0))
        b[1]["v_pages"][b[2][0, 3], 2, 0, 7] = float("nan")
        got = attend(gpu, b, [0, 2, 3]).cpu()
        inside = new[0] + new[1]
        assert got[:inside, :, 7].isnan().all() and torch.isfinite(got[inside:]).all() and torch.isfinite(got[:inside, :, 8:]).all()


@pytest.mark.parametrize("hints", [(1, 1, 1), (7, 100, 64), (10 ** 9, 10 ** 12, 10 ** 12), (None, None, None), (0, 0, 0)])
@pytest.mark.parametrize("new,keys", [([300, 1, 40], [1200, 900, 40]), ([1, 1, 2], [1000, 7, 500])])
def test_lengths_that_the_host_does_not_know(gpu, hints, new, keys):
    b = batch(81, new, keys, [2100], 8, 2, 128, 16, BF16)
    check_shared(gpu, b, told=False, max_q_len=hints[0], max_kv_len=hints[1], max_prefix_len=hints[2])


def test_lengths_beyond_the_tables_end_with_them(gpu):
    b = list(batch(82, [4, 1], [64, 64], [160], 4, 2, 64, 16, BF16))
    b[4] = b[4][:, :4].contiguous()
    want = attend(gpu, b, causal=False)
    b[3], b[5] = b[3] + 5000, b[5] + 1000
    assert torch.equal(attend(gpu, b, causal=False), want)


@pytest.mark.parametrize("new", [[3, 2], [1, 1]])
def test_rows_outside_every_stream(gpu, new):
    b = list(batch(91, [20], [33], [300], 4, 2, 64, 16, BF16))
    b[4], b[5], b[6] = b[4].repeat(2, 1), int32([33, 20]), starts(new, first=4)
    rows = torch.zeros(20, dtype=torch.bool)
    rows[4:4 + sum(new)] = True
    got = check_shared(gpu, b)
    assert (got[~rows.to(gpu)] == 0).all()
    out = torch.full_like(got, 7.0)
    assert attend(gpu, b, max_q_len=max(new), max_kv_len=33, max_prefix_len=300, out=out) is out
    assert torch.equal(out[rows.to(gpu)], got[rows.to(gpu)]) and (out[~rows.to(gpu)] == 7.0).all()


def test_nothing_shared_and_nothing_owned(gpu):
    new, keys = [1, 40, 3], [100, 300, 70]
    q, cache, prefix_table, prefix_lens, table, lens, q_starts = batch(101, new, keys, [400], 8, 2, 128, 16, BF16)
    dev = {n: t.to(gpu) for n, t in cache.items()}
    b = (q, cache, prefix_table, prefix_lens, table, lens, q_starts)
    check_shared(gpu, (*b[:3], prefix_lens * 0, *b[4:]))
    check_shared(gpu, b, [3, 3])                                                # a group without streams
    check_shared(gpu, (*b[:2], prefix_table[:0], prefix_lens[:0], *b[4:]), [0])   # no groups
    check_shared(gpu, (*b[:5], lens * 0, q_starts))
    check_shared(gpu, (*b[:4], table[:, :0], lens * 0, q_starts))               # no own table
    check_shared(gpu, (*b[:2], prefix_table[:, :0], prefix_lens * 0, *b[4:]))   # no table of what is shared
    assert attend(gpu, (q[:0], *b[1:6], q_starts * 0)).shape == (0, 8, 128)
    none = {n: t[:0] for n, t in cache.items()}
    assert (attend(gpu, (q, none, *b[2:])) == 0).all()
    i32 = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=gpu)  # noqa: E731
    assert (shared_prefix_attention(q.to(gpu), dev, prefix_table.to(gpu), prefix_lens.to(gpu), i32(0, 5), i32(0), i32(1)) == 0).all()   # no streams


def test_views_of_one_table_are_the_paged_attention(gpu):
    # a beginning of whole pages at the front of every row of a table
    q, cache, prefix_table, prefix_lens, own, lens, q_starts = batch(105, [1, 2, 1], [90, 33, 7], [160], 4, 2, 128, 16, BF16)
    table = torch.cat([prefix_table.expand(3, -1), own], dim=1).to(gpu)
    dev = {n: t.to(gpu) for n, t in cache.items()}
    got = shared_prefix_attention(q.to(gpu), dev, table[:1, :10], prefix_lens.to(gpu), table[:, 10:], lens.to(gpu), q_starts.to(gpu))
    want, error, _ = step_ref.shared_prefix(q, cache, prefix_table, prefix_lens, own, lens, q_starts, None, True, 128 ** -0.5)
    close(got, want, error)
    close(paged_attention(q.to(gpu), dev, table, (lens + 160).to(gpu), q_starts.to(gpu)), want, error)


@pytest.mark.parametrize("new", [[3, 50], [1, 1]])
def test_shared_beginnings_with_strides(gpu, new):
    q, cache, *tables, q_starts = batch(111, new, [100, 129], [300], 4, 2, 64, 16, BF16)
    want = check_shared(gpu, (q, cache, *tables, q_starts))
    T = sum(new)
    wide = torch.zeros(T, 11, 64, dtype=BF16, device=gpu)
    wide[:, 2:6] = q.to(gpu)
    both = torch.stack([cache["k_pages"], cache["v_pages"]], dim=1).transpose(2, 3).contiguous().to(gpu)   # [pages, 2, heads, rows, D]
    paged = {"k_pages": both[:, 0].transpose(1, 2), "v_pages": both[:, 1].transpose(1, 2)}
    out = torch.full((4, T, 64), 7.0, dtype=BF16, device=gpu).transpose(0, 1)
    on = [t.to(gpu) for t in tables]
    args = (paged, torch.cat([on[0], on[0]], dim=1)[:, :on[0].shape[1]], on[1], torch.cat([on[2], on[2]], dim=1)[:, :on[2].shape[1]], on[3], q_starts.to(gpu))
    told = dict(max_q_len=max(new), max_kv_len=129, max_prefix_len=300)
    shared_prefix_attention(wide[:, 2:6], *args, out=out, **told)
    assert torch.equal(out, want)
    odd = torch.zeros(T * 256 + 1, dtype=BF16, device=gpu)[1:].view(T, 4, 64).copy_(q)   # rows at an odd address are copied first
    assert torch.equal(shared_prefix_attention(odd, *args, **told), want)
    mine = q.to(gpu)
    assert shared_prefix_attention(mine, *args, out=mine, **told) is mine and torch.equal(mine, want)   # in place of the queries


def test_scales_and_large_scores(gpu):
    for scale in (0.01, 3.0):
        check_shared(gpu, batch(121, [1] * 8, [30] * 8, [700], 4, 2, 128, 16, BF16), softmax_scale=scale)
        check_shared(gpu, batch(122, [1] * 8, [30] * 8, [700], 4, 2, 64, 16, F16), softmax_scale=scale)


def test_a_cache_beyond_32_bits_of_offsets(gpu):
    # pages far apart: 2^31 elements and more between the first and the last
    q, cache, *rest = batch(131, [1, 1, 60], [40, 90, 60], [300], 4, 2, 64, 16, F16)
    far = torch.empty(cache["k_pages"].shape[0], 1 << 26, dtype=F16, device=gpu)
    assert far.numel() > 1 << 31
    size = 16 * 2 * 64
    dev = {}
    for i, n in enumerate(("k_pages", "v_pages")):
        dev[n] = far[:, i * size:(i + 1) * size].unflatten(1, (16, 2, 64))
        dev[n].copy_(cache[n])
    got = shared_prefix_attention(q.to(gpu), dev, *(t.to(gpu) for t in rest))
    want, error, _ = step_ref.shared_prefix(q, cache, *rest, None, True, 64 ** -0.5)
    close(got, want, error)


def test_on_streams_of_their_own_and_twice_at_once(gpu):
    b = batch(141, [1] * 12, [90] * 12, [5000], 16, 2, 128, 16, BF16)
    q, cache, *rest = b
    args = (q.to(gpu), {n: t.to(gpu) for n, t in cache.items()}, *(t.to(gpu) for t in rest))
    told = dict(max_q_len=1, max_kv_len=90, max_prefix_len=5000)
    want = shared_prefix_attention(*args, **told)
    torch.cuda.synchronize()
    sides, got = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(3):
        for s in sides:
            with torch.cuda.stream(s):
                got.append(shared_prefix_attention(*args, **told))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


# ------------------------------------------------------------------------------------------------ together
def test_steps_of_streams_that_share_a_beginning(gpu):
    """Two groups of streams decode behind their beginnings: layout, rotation into pages and attention as one recorded step, replayed, against plain
    forms that follow it."""
    Hq, Hk, D, page, shared, new = 8, 2, 64, 8, [90, 200], [1, 2, 1, 0, 3, 1]
    cuts, B, T, steps = [0, 2, 6], len(new), sum(new), 5
    pages_shared = [-(-n // page) for n in shared]
    pages, width = sum(pages_shared) + 40, 5
    cache = {n: randn(i, pages, page, Hk, D).to(gpu) for i, n in enumerate(("k_pages", "v_pages"), 1)}
    prefix_table = torch.full((2, max(pages_shared)), -1, dtype=torch.int32)
    prefix_table[0, :pages_shared[0]] = torch.arange(pages_shared[0])
    prefix_table[1, :pages_shared[1]] = torch.arange(pages_shared[1]) + pages_shared[0]
    free = torch.randperm(40, generator=torch.Generator().manual_seed(9)).int() + sum(pages_shared)
    f = rotary_frequencies(D, scaling="positions", factor=2.0)
    rows = torch.zeros(T, Hq + 2 * Hk, D, dtype=BF16, device=gpu)
    table, kv, cursor = torch.full((B, width), -1, dtype=torch.int32, device=gpu), torch.zeros(B, dtype=torch.int32, device=gpu), int32([0], gpu)
    on = dict(new=int32(new, gpu), free=free.to(gpu), prefix_lens=int32(shared, gpu), starts=int32(cuts, gpu), prefix_table=prefix_table.to(gpu), f=f.to(gpu))

    def step():
        at = lay_out_step(on["new"], kv, table, on["free"], page, T, prefix_lens=on["prefix_lens"], group_starts=on["starts"], cursor=cursor, kv_lens_out=kv)
        q, k, v = rows.split([Hq, Hk, Hk], dim=1)
        q = rotate_by_position_paged(q, k, v, cache, at.slots, at.positions, on["f"], interleaved=False)
        return q, shared_prefix_attention(q, cache, on["prefix_table"], on["prefix_lens"], table, at.kv_lens, at.q_starts, group_starts=on["starts"], max_q_len=3,
                                          max_kv_len=width * page, max_prefix_len=200)

    state = (table, kv, cursor, *cache.values())
    kept = [t.clone() for t in state]
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q_now, out = step()
    for t, before in zip(state, kept):
        t.copy_(before)
    lens, tables, taken = [0] * B, table.tolist(), 0
    for i in range(steps):
        new_rows = randn(100 + i, T, Hq + 2 * Hk, D)
        rows.copy_(new_rows)
        graph.replay()
        torch.cuda.synchronize()
        q_starts, lens, positions, slots, _, tables, taken = step_ref.step_layout(new, lens, tables, free.tolist(), page, T, shared, cuts, taken)
        assert kv.tolist() == lens and table.tolist() == tables and cursor.tolist() == [taken]
        q, k, v = new_rows.split([Hq, Hk, Hk], dim=1)
        close(q_now, *step_ref.rotate(q, None, 0.0, f, torch.tensor(positions), False))
        now = {n: t.cpu() for n, t in cache.items()}
        close(now["k_pages"].flatten(0, 1)[slots], *step_ref.rotate(k, None, 0.0, f, torch.tensor(positions), False))
        assert torch.equal(now["v_pages"].flatten(0, 1)[slots], v)
        want, error, _ = step_ref.shared_prefix(q_now.cpu(), now, prefix_table, int32(shared), int32(tables), int32(lens), int32(q_starts), int32(cuts), True, D ** -0.5)
        close(out, want, error, f"step {i}")


def test_recorded_attention_follows_its_lengths(gpu):
    B, T, Hq, Hk, D, page = 20, 60, 8, 2, 128, 16
    cache = {n: randn(i, 90, page, Hk, D).to(gpu) for i, n in enumerate(("k_pages", "v_pages"), 1)}
    q = randn(3, T, Hq, D).to(gpu)
    order = torch.randperm(90, generator=torch.Generator().manual_seed(1)).int()
    table, prefix_table = order[:60].view(20, 3).to(gpu), order[60:].view(2, 15).to(gpu)
    kv, q_starts, shared, cuts = int32([1] * B, gpu), int32([0] * (B + 1), gpu), int32([0, 0], gpu), int32([0, 0, 0], gpu)
    call = lambda: shared_prefix_attention(q, cache, prefix_table, shared, table, kv, q_starts, cuts, max_q_len=40, max_kv_len=48, max_prefix_len=240)  # noqa: E731
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded = call()
    cases = [([3] * 20, [48] * 20, [240, 100], [0, 10, 20]), ([1] * 20, [7] * 20, [0, 0], [0, 0, 20]), ([40, 1] + [0] * 10 + [1] * 8, [45] * 20, [200, 240], [0, 2, 20]),
             ([0] * 20, [0] * 20, [5, 5], [20, 20, 20])]
    for new, keys, lens, at in cases + cases[::-1]:
        q_starts.copy_(starts(new))
        for t, values in ((kv, keys), (shared, lens), (cuts, at)):
            t.copy_(int32(values))
        graph.replay()
        torch.cuda.synchronize()
        replayed = recorded.clone()
        eager = call()
        torch.cuda.synchronize()
        assert torch.isfinite(replayed).all() and torch.equal(replayed, eager), (new, keys, lens, at)
        want, error, _ = step_ref.shared_prefix(q.cpu(), {n: t.cpu() for n, t in cache.items()}, prefix_table.cpu(), int32(lens), table.cpu(), int32(keys), starts(new),
                                                int32(at), True, D ** -0.5)
        close(replayed, want, error)
