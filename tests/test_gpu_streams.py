"""Several streams in one batch on the GPU: norms per head with rotation and page write, attention over the paged cache, cross
attention to ragged encoder states; against plain 64-bit forms whose allowed errors count roundings."""
import pytest
import torch

import streams_reference as ref
from longlive_amd.utils.cross_attention import ragged_cross_attention
from longlive_amd.utils.paged_kv import head_norm_rope_paged, initialize_paged_kv_cache, paged_attention, paged_slots
from longlive_amd.utils.rope import head_norm_rope

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def randn(seed, *shape, dtype=BF16, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def starts(lengths, first=0):
    return torch.tensor([first] + lengths, dtype=torch.int32).cumsum(0, dtype=torch.int32)


def close(got, want, error, what=""):
    got = got.detach().cpu().double()
    off = (got - want).abs()
    assert torch.isfinite(got).all(), what
    worst = (off / error.clamp(min=1e-300)).max().item() if off.numel() else 0.0
    assert (off <= error).all(), f"{what}: {worst:.2f} of the allowed error, at {(off > error).nonzero()[:3].tolist()}"


# ------------------------------------------------------------------------------------------------ norms and rotation
def angles(rows, R, seed=3):
    a = torch.rand(rows, R // 2, generator=torch.Generator().manual_seed(seed)) * 6.0
    return a.cos(), a.sin()


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("T,Hq,Hk,D,R,dtype", [
    (1, 1, 1, 128, 128, BF16), (5, 4, 2, 64, 64, F16), (37, 7, 1, 64, 32, BF16), (300, 24, 24, 128, 128, BF16), (33, 3, 3, 128, 16, F16),
    (9, 5, 5, 8, 8, BF16), (11, 6, 2, 96, 64, BF16), (64, 2, 2, 256, 256, BF16), (7, 3, 1, 200, 136, F16), (2049, 40, 8, 128, 64, BF16)])
def test_norm_per_head_and_rotation(gpu, T, Hq, Hk, D, R, dtype, interleaved):
    q, k = randn(1, T, Hq, D, dtype=dtype), randn(2, T, Hk, D, dtype=dtype, scale=3.0)
    wq, wk = randn(3, D, dtype=dtype), randn(4, D, dtype=torch.float32)
    cos, sin = angles(T + 3, R)
    positions = torch.randint(0, T + 3, (T,), generator=torch.Generator().manual_seed(5))
    got = head_norm_rope(*(t.to(gpu) for t in (q, k, wq, wk)), 1e-6, cos.to(gpu), sin.to(gpu), positions.to(gpu), interleaved=interleaved)
    for x, w, y in ((q, wq, got[0]), (k, wk, got[1])):
        assert y.dtype == dtype and y.shape == x.shape
        close(y, *ref.head_norm_rope(x, w, 1e-6, cos, sin, positions, interleaved))


@pytest.mark.parametrize("weights,rotation", [(False, True), (True, False), (False, False)])
def test_norm_and_rotation_each_alone(gpu, weights, rotation):
    q, k, w = randn(1, 19, 6, 128), randn(2, 19, 2, 128), randn(3, 128)
    cos, sin = angles(19, 128)
    w = w if weights else None
    cos, sin = (cos, sin) if rotation else (None, None)
    dev = lambda t: None if t is None else t.to(gpu)  # noqa: E731
    got = head_norm_rope(q.to(gpu), k.to(gpu), dev(w), dev(w), 1e-5, dev(cos), dev(sin))
    for x, y in zip((q, k), got):
        close(y, *ref.head_norm_rope(x, w, 1e-5, cos, sin, None, True))


def test_rows_beyond_the_table_are_normed_and_not_rotated(gpu):
    q, w = randn(1, 6, 2, 64), randn(2, 64)
    cos, sin = angles(4, 64)
    positions = torch.tensor([0, 3, 4, -1, 1 << 40, 2])
    got, _ = head_norm_rope(q.to(gpu), q.to(gpu), w.to(gpu), w.to(gpu), 1e-6, cos.to(gpu), sin.to(gpu), positions.to(gpu))
    close(got, *ref.head_norm_rope(q, w, 1e-6, cos, sin, positions, True))


def test_rows_of_zeros_and_of_infinities(gpu):
    q = randn(1, 4, 2, 64)
    q[0] = 0.0
    q[1, 0, 5] = float("inf")
    w = randn(2, 64)
    got, _ = head_norm_rope(q.to(gpu), q.to(gpu), w.to(gpu), w.to(gpu), 1e-6, None, None)
    got = got.cpu().float()
    assert (got[0] == 0).all() and got[1, 0, 5].isnan() and (got[1, 0, :5] == 0).all()
    close(got[2:], *(t[2:] for t in ref.head_norm_rope(q, w, 1e-6, None, None, None, True)))


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("T,Hq,Hk,D,page,dtype", [(1, 8, 2, 128, 16, BF16), (50, 4, 4, 64, 3, F16), (129, 6, 3, 128, 1, BF16)])
def test_write_into_pages(gpu, T, Hq, Hk, D, page, dtype, interleaved):
    rows = randn(1, T, (Hq + 2 * Hk) * D, dtype=dtype)
    q, k, v = (x.unflatten(1, (-1, D)) for x in rows.split([Hq * D, Hk * D, Hk * D], dim=1))   # views of one projection
    wq, wk = randn(2, D, dtype=dtype), randn(3, D, dtype=dtype)
    cos, sin = angles(T, D)
    pages = -(-T // page) + 2
    cache = {n: randn(7, pages, page, Hk, D, dtype=dtype).to(gpu) for n in ("k_pages", "v_pages")}
    before = {n: t.cpu().clone() for n, t in cache.items()}
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(1))[:T]
    slots[T // 2] = -1 if T > 1 else slots[0]
    if T > 2:
        slots[0] = pages * page      # behind the cache
    on = rows.to(gpu)
    qd, kd, vd = (x.unflatten(1, (-1, D)) for x in on.split([Hq * D, Hk * D, Hk * D], dim=1))
    got = head_norm_rope_paged(qd, kd, vd, cache, slots.to(gpu), wq.to(gpu), wk.to(gpu), 1e-6, cos.to(gpu), sin.to(gpu), interleaved=interleaved)
    close(got, *ref.head_norm_rope(q, wq, 1e-6, cos, sin, None, interleaved))
    want, error = ref.head_norm_rope(k, wk, 1e-6, cos, sin, None, interleaved)
    ok = (slots >= 0) & (slots < pages * page)
    for name, new, err in (("k_pages", want, error), ("v_pages", v.double(), torch.zeros_like(error))):
        now = cache[name].cpu().flatten(0, 1)
        close(now[slots[ok]], new[ok], err[ok], name)
        left = torch.ones(pages * page, dtype=torch.bool)
        left[slots[ok]] = False
        assert torch.equal(now[left], before[name].flatten(0, 1)[left]), name


def test_queries_alone_where_the_cache_has_no_pages(gpu):
    q, k = randn(1, 3, 4, 64).to(gpu), randn(2, 3, 2, 64).to(gpu)
    cache = initialize_paged_kv_cache(1, 0, 16, 2, 64, gpu)[0]
    got = head_norm_rope_paged(q, k, k, cache, torch.full((3,), -1, device=gpu), None, None, 1e-6, None, None)
    assert torch.equal(got, q)


# ------------------------------------------------------------------------------------------------ paged attention
def batch(seed, new, keys, Hq, Hk, D, page, dtype, spare=2, fill=None, scale=1.5):
    """(q, cache, page_table, kv_lens, q_starts) on the CPU: pages in any order, rows that hold no key filled with `fill`."""
    g = torch.Generator().manual_seed(seed)
    held = [-(-n // page) for n in keys]
    pages = sum(held) + spare
    order = torch.randperm(pages, generator=g).int()
    table = torch.full((len(keys), max(held + [1]) + 1), 1 << 30, dtype=torch.int32)
    cache = {n: randn(seed + i, pages, page, Hk, D, dtype=dtype) for i, n in enumerate(("k_pages", "v_pages"), 1)}
    used = torch.zeros(pages, page, dtype=torch.bool)
    at = 0
    for b, n in enumerate(held):
        table[b, :n] = order[at:at + n]
        for i in range(n):
            used[order[at + i], :min(page, keys[b] - i * page)] = True
        at += n
    if fill is not None:
        for t in cache.values():
            t[~used] = fill
    q = randn(seed + 5, sum(new), Hq, D, dtype=dtype, scale=scale)
    return q, cache, table, torch.tensor(keys, dtype=torch.int32), starts(new)


def check_paged(gpu, b, what="", causal=True, window=None, sink=0, **kw):
    q, cache, table, lens, q_starts = b
    dev = {n: t.to(gpu) for n, t in cache.items()}
    got = paged_attention(q.to(gpu), dev, table.to(gpu), lens.to(gpu), q_starts.to(gpu), causal=causal, window=window, sink_tokens=sink, **kw)
    keys_of, seen_of = ref.paged_keys(cache, table, lens)
    want, error, _ = ref.ragged_attention(q, q_starts, kw.get("softmax_scale") or q.shape[-1] ** -0.5, keys_of, seen_of(causal, window, sink))
    close(got, want, error, what)
    return got


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D,dtype", [(64, F16), (128, BF16), (128, F16), (64, BF16)])
@pytest.mark.parametrize("new,keys,Hq,Hk,page", [
    ([1], [1], 1, 1, 1),
    ([1, 1, 1], [40, 300, 1], 8, 2, 16),
    ([1, 5, 0, 70], [257, 5, 33, 200], 4, 4, 24),
    ([130, 1, 64], [130, 64, 1000], 5, 1, 7),
    ([33, 2], [65, 2], 14, 2, 64),
    ([300], [700], 3, 3, 880)])
def test_paged_attention(gpu, new, keys, Hq, Hk, page, D, dtype, causal):
    check_paged(gpu, batch(11, new, keys, Hq, Hk, D, page, dtype, fill=float("nan")), causal=causal)


@pytest.mark.parametrize("D,dtype", [(64, F16), (128, BF16)])
@pytest.mark.parametrize("window,sink", [(1, 0), (17, 0), (64, 4), (100, 130), (1 << 40, 3), (3, 64)])
@pytest.mark.parametrize("causal", [True, False])
def test_windows_and_kept_first_keys(gpu, window, sink, causal, D, dtype):
    check_paged(gpu, batch(21, [150, 1, 3], [400, 333, 3], 4, 2, D, 16, dtype, fill=float("nan")), causal=causal, window=window, sink=sink)


@pytest.mark.parametrize("D,dtype", [(64, F16), (128, BF16)])
@pytest.mark.parametrize("Hq,Hk", [(8, 8), (32, 4), (48, 1)])
def test_single_tokens_over_long_caches(gpu, Hq, Hk, D, dtype):
    keys = [1, 4099, 700, 2047, 9000]
    check_paged(gpu, batch(31, [1] * 5, keys, Hq, Hk, D, 16, dtype), max_q_len=1, max_kv_len=9000)


@pytest.mark.parametrize("new", [[2, 3, 1], [9, 9, 9], [16, 1, 30], [40, 1, 1]])
def test_a_few_tokens_each_over_long_caches(gpu, new):
    check_paged(gpu, batch(41, new, [5000, 777, 2500], 16, 4, 128, 32, BF16), max_q_len=max(new), max_kv_len=5000)


@pytest.mark.parametrize("D,dtype", [(64, F16), (128, BF16)])
@pytest.mark.parametrize("causal,window,sink", [(True, None, 0), (False, None, 0), (True, 3000, 130), (False, 2500, 70)])
@pytest.mark.parametrize("new,keys,Hq,Hk,page", [([150, 40, 1], [5000, 3000, 4500], 2, 1, 16), ([200], [6000], 3, 1, 24), ([1, 2], [9000, 6400], 4, 2, 880),
                                                 ([300, 2, 33, 129], [1700, 3333, 33, 2500], 5, 1, 8)])
def test_tiles_whose_keys_are_cut(gpu, new, keys, Hq, Hk, page, causal, window, sink, D, dtype):
    b = batch(45, new, keys, Hq, Hk, D, page, dtype, fill=float("nan"))
    check_paged(gpu, b, causal=causal, window=window, sink=sink, max_q_len=max(new), max_kv_len=max(keys))


@pytest.mark.parametrize("most_keys", [200, 2600])
def test_more_streams_than_a_wave_has_lanes(gpu, most_keys):
    g = torch.Generator().manual_seed(3)
    new = (torch.randint(0, 5, (200,), generator=g) ** 2).tolist()
    new[7], new[64], new[130], new[199] = 150, 0, 77, 3
    keys = [max(n, int(k)) for n, k in zip(new, torch.randint(0, most_keys // 8, (200,), generator=g))]
    keys[7], keys[63], keys[130], keys[199] = most_keys, most_keys - 1, 140, most_keys // 2
    check_paged(gpu, batch(46, new, keys, 4, 2, 64, 16, BF16, fill=float("nan")), max_q_len=max(new), max_kv_len=max(keys))


def test_streams_that_find_no_records_left_stay_whole(gpu):
    # 64 kv heads leave a stream fewer records than its 16 tiles would take; the smaller one before it is cut
    new, keys, H, D = [20, 2048], [4000, 5300], 64, 64
    q, cache, table, lens, q_starts = batch(47, new, keys, H, H, D, 16, F16)
    dev = {n: t.to(gpu) for n, t in cache.items()}
    got = paged_attention(q.to(gpu), dev, table.to(gpu), lens.to(gpu), q_starts.to(gpu), max_q_len=2048, max_kv_len=5300)
    keys_of, seen_of = ref.paged_keys({n: t[:, :, [0, 63]] for n, t in cache.items()}, table, lens)
    rows = torch.cat([torch.arange(20), torch.tensor([20, 21, 900, 2066, 2067])])
    for h, head in enumerate((0, 63)):
        for b, first in ((0, 0), (1, 20)):
            k, v = (t[:, h] for t in keys_of(b))
            at = rows[(rows >= first) & (rows < first + new[b])]
            want, error = ref.attend(q[at, head], k, v, seen_of()(b, new[b], len(k))[at - first], D ** -0.5)
            close(got[at.to(gpu), head], want, error, f"stream {b} head {head}")


def test_one_long_stream_among_short_ones_finds_no_records_left(gpu):
    # room for 496 records of a head; 16 tiles in 8 parts want 512, the stream before them is cut in two
    new, keys, H, D = [20, 2048] + [1] * 70, [2000, 13000] + [16] * 70, 64, 64   # more than 64 streams: parts by the host
    q, cache, table, lens, q_starts = batch(48, new, keys, H, H, D, 16, F16)
    dev = {n: t.to(gpu) for n, t in cache.items()}
    got = paged_attention(q.to(gpu), dev, table.to(gpu), lens.to(gpu), q_starts.to(gpu), max_q_len=2048, max_kv_len=13000)
    keys_of, seen_of = ref.paged_keys({n: t[:, :, [0, 63]] for n, t in cache.items()}, table, lens)
    firsts = q_starts.tolist()
    for h, head in enumerate((0, 63)):
        for b, at in ((0, torch.arange(20)), (1, torch.tensor([0, 1, 900, 2046, 2047])), (2, torch.tensor([0])), (71, torch.tensor([0]))):
            k, v = (t[:, h] for t in keys_of(b))
            want, error = ref.attend(q[firsts[b] + at, head], k, v, seen_of()(b, new[b], len(k))[at], D ** -0.5)
            close(got[(firsts[b] + at).to(gpu), head], want, error, f"stream {b} head {head}")


def test_rows_that_see_nothing_are_zeros(gpu):
    # more new tokens than keys: the first of them sit before the stream's beginning; no keys at all; a table of holes
    b = batch(51, [5, 3, 4], [2, 0, 20], 4, 2, 64, 8, BF16, fill=float("nan"))
    b[2][2] = -1
    got = check_paged(gpu, b)
    assert (got[:3] == 0).all() and (got[3:5] != 0).any() and (got[5:] == 0).all()


@pytest.mark.parametrize("new", [[3, 1], [90, 70], [1, 1]])
def test_holes_in_the_page_table(gpu, new):
    b = batch(61, new, [500, 320], 8, 4, 128, 16, BF16)
    for entry in ((0, 0), (0, 7), (0, 8), (0, 9), (0, 10), (0, 11), (1, 19)):
        b[1]["k_pages"][b[2][entry]] = b[1]["v_pages"][b[2][entry]] = float("nan")
        b[2][entry] = -1 if entry[1] % 2 else b[1]["k_pages"].shape[0]
    check_paged(gpu, b)
    check_paged(gpu, b, causal=False, window=100, sink=130)


def test_streams_that_share_pages(gpu):
    q, cache, table, lens, q_starts = batch(71, [1, 33], [200, 240], 4, 2, 128, 16, BF16)
    table[1, :10] = table[0, :10]
    check_paged(gpu, (q, cache, table, lens, q_starts))


def test_lengths_beyond_the_table_end_with_it(gpu):
    q, cache, table, lens, q_starts = batch(72, [4, 4], [64, 64], 4, 2, 64, 16, BF16)
    table = table[:, :4].contiguous()
    want = paged_attention(q.to(gpu), {n: t.to(gpu) for n, t in cache.items()}, table.to(gpu), lens.to(gpu), q_starts.to(gpu), causal=False)
    got = paged_attention(q.to(gpu), {n: t.to(gpu) for n, t in cache.items()}, table.to(gpu), (lens + 1000).to(gpu), q_starts.to(gpu), causal=False)
    assert torch.equal(got, want)


@pytest.mark.parametrize("hints", [(1, 1), (7, 100), (10 ** 9, 10 ** 12), (None, None), (0, 0)])
@pytest.mark.parametrize("new,keys", [([300, 1, 40], [1200, 900, 40]), ([1, 1, 2], [3000, 7, 1500])])
def test_lengths_that_the_host_does_not_know(gpu, hints, new, keys):
    check_paged(gpu, batch(81, new, keys, 8, 2, 128, 16, BF16), max_q_len=hints[0], max_kv_len=hints[1])


@pytest.mark.parametrize("new", [[3, 2], [1, 1]])
def test_rows_outside_every_stream(gpu, new):
    q, cache, table, lens, _ = batch(91, [20], [33], 4, 2, 64, 16, BF16)
    table, lens = table.repeat(2, 1), torch.tensor([33, 20], dtype=torch.int32)
    q_starts = starts(new, first=4)
    rows = torch.zeros(20, dtype=torch.bool)
    rows[4:4 + sum(new)] = True
    args = (q.to(gpu), {n: t.to(gpu) for n, t in cache.items()}, table.to(gpu), lens.to(gpu), q_starts.to(gpu))
    keys_of, seen_of = ref.paged_keys(cache, table, lens)
    want, error, _ = ref.ragged_attention(q, q_starts, 64 ** -0.5, keys_of, seen_of())
    got = paged_attention(*args)
    close(got, want, error)
    assert (got[~rows.to(gpu)] == 0).all()
    out = torch.full_like(got, 7.0)
    assert paged_attention(*args, out=out) is out
    assert torch.equal(out[rows.to(gpu)], got[rows.to(gpu)]) and (out[~rows.to(gpu)] == 7.0).all()


def test_no_streams_and_no_rows(gpu):
    cache = initialize_paged_kv_cache(1, 4, 16, 2, 64, gpu)[0]
    i32 = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=gpu)  # noqa: E731
    q = randn(1, 3, 4, 64).to(gpu)
    assert (paged_attention(q, cache, i32(0, 5), i32(0), i32(1)) == 0).all()
    assert paged_attention(q[:0], cache, i32(2, 5), i32(2), i32(3)).shape == (0, 4, 64)
    assert (paged_attention(q, cache, i32(1, 0), i32(1), starts([3]).to(gpu)) == 0).all()
    none = initialize_paged_kv_cache(1, 0, 16, 2, 64, gpu)[0]
    assert (paged_attention(q, none, i32(1, 5), i32(1) + 9, starts([3]).to(gpu)) == 0).all()


def test_queries_outputs_and_pages_with_strides(gpu):
    q, cache, table, lens, q_starts = batch(101, [3, 50], [100, 129], 4, 2, 64, 16, BF16)
    want = check_paged(gpu, (q, cache, table, lens, q_starts))
    # q and out in the middle of wider rows, pages of K and V interleaved, heads before rows, a table within a wider one
    wide = torch.zeros(53, 11, 64, dtype=BF16, device=gpu)
    wide[:, 2:6] = q.to(gpu)
    both = torch.stack([cache["k_pages"], cache["v_pages"]], dim=1).transpose(2, 3).contiguous().to(gpu)   # [pages, 2, heads, rows, D]
    paged = {"k_pages": both[:, 0].transpose(1, 2), "v_pages": both[:, 1].transpose(1, 2)}
    out = torch.full((4, 53, 64), 7.0, dtype=BF16, device=gpu).transpose(0, 1)
    tables = torch.cat([table, table], dim=1).to(gpu)[:, :table.shape[1]]
    paged_attention(wide[:, 2:6], paged, tables, lens.to(gpu), q_starts.to(gpu), out=out)
    assert torch.equal(out, want)
    # rows at an odd address are copied first
    odd = torch.zeros(53 * 256 + 1, dtype=BF16, device=gpu)[1:].view(53, 4, 64).copy_(q)
    assert torch.equal(paged_attention(odd, paged, tables, lens.to(gpu), q_starts.to(gpu)), want)


@pytest.mark.parametrize("new,keys", [([1, 1], [9000, 40]), ([150, 1, 9], [400, 3000, 70]), ([260], [9000])])
def test_results_in_place_of_the_queries(gpu, new, keys):
    q, cache, table, lens, q_starts = (t if isinstance(t, dict) else t.to(gpu) for t in batch(102, new, keys, 8, 2, 128, 16, BF16))
    cache = {n: t.to(gpu) for n, t in cache.items()}
    want = paged_attention(q, cache, table, lens, q_starts)
    assert paged_attention(q, cache, table, lens, q_starts, out=q) is q
    inside = slice(int(q_starts[0]), int(q_starts[-1]))
    assert torch.equal(q[inside], want[inside])


def test_inputs_that_repeat_their_rows(gpu):
    q, k, v = (randn(s, *shape).to(gpu) for s, shape in ((5, (1, 2, 64)), (6, (1, 2, 64)), (7, (300, 1, 64))))
    q_starts, k_starts = starts([3, 90]).to(gpu), starts([200, 100]).to(gpu)
    a, b, c = q.expand(93, 2, 64), k.expand(300, 2, 64), v.expand(300, 2, 64)
    want = ragged_cross_attention(a.contiguous(), b.contiguous(), c.contiguous(), q_starts, k_starts)
    assert torch.equal(ragged_cross_attention(a, b, c, q_starts, k_starts), want)
    for x, y in zip(head_norm_rope(a, c[:93], None, None, 1e-6, None, None), head_norm_rope(a.contiguous(), c[:93].contiguous(), None, None, 1e-6, None, None)):
        assert torch.equal(x, y)


def test_dimensions_of_one_with_any_stride(gpu):
    """Torch leaves anything in the stride of a dimension of size one: one row, one head, one page, pages of one row."""
    def odd(t, *dims):
        return t.as_strided(t.shape, [7 if d in dims else s for d, s in enumerate(t.stride())])

    q, cache, table, lens, q_starts = (t if isinstance(t, dict) else t.to(gpu) for t in batch(105, [1], [1], 1, 1, 64, 1, BF16, spare=0))
    cache = {n: t.to(gpu) for n, t in cache.items()}
    want = paged_attention(q, cache, table, lens, q_starts)
    pages = {n: odd(t, 0, 1, 2) for n, t in cache.items()}
    assert torch.equal(paged_attention(odd(q, 0, 1), pages, odd(table, 0), lens, q_starts), want)
    assert torch.equal(ragged_cross_attention(odd(q, 0, 1), odd(cache["k_pages"][0], 0, 1), odd(cache["v_pages"][0], 0, 1), q_starts, q_starts), want)
    k, w = randn(3, 1, 1, 64).to(gpu), randn(4, 64).to(gpu)
    first, _ = head_norm_rope(q, k, w, w, 1e-6, None, None)
    assert torch.equal(head_norm_rope(odd(q, 0, 1), odd(k, 0, 1), w, w, 1e-6, None, None)[0], first)
    cache = {n: torch.zeros(5, 1, 1, 64, dtype=BF16, device=gpu) for n in cache}
    head_norm_rope_paged(q, k, k, {n: odd(t, 1, 2) for n, t in cache.items()}, torch.tensor([3], device=gpu), None, None, 1e-6, None, None)
    assert torch.equal(cache["k_pages"][3, 0], k[0]) and torch.equal(cache["v_pages"][3, 0], k[0]) and not cache["k_pages"][:3].any()


@pytest.mark.parametrize("native", [True, False])
def test_both_host_paths_give_the_same(gpu, native, monkeypatch):
    from longlive_amd import _native

    q, cache, table, lens, q_starts = (t if isinstance(t, dict) else t.to(gpu) for t in batch(106, [3, 1], [100, 700], 4, 2, 64, 16, F16))
    cache = {n: t.to(gpu) for n, t in cache.items()}
    cos, sin = (t.to(gpu) for t in angles(4, 64))
    slots = paged_slots(table, lens, q_starts, 4, 16)
    k = randn(3, 4, 2, 64, dtype=F16).to(gpu)

    def everything():
        pages = {n: t.clone() for n, t in cache.items()}
        roped = head_norm_rope_paged(q, k, k, pages, slots, None, None, 1e-6, cos, sin, interleaved=False)
        rows = pages["k_pages"].flatten(0, 1)
        return (roped, *pages.values(), *head_norm_rope(q, k, None, None, 1e-6, cos, sin), paged_attention(roped, pages, table, lens, q_starts, window=50),
                ragged_cross_attention(roped, rows, rows, q_starts, q_starts, k_lens=lens, key_mask=torch.arange(len(rows), device=gpu) % 3 > 0))

    want = everything()
    if not native:
        monkeypatch.setattr(_native, "_host", _native._NoHostPath())
    for a, b in zip(everything(), want):
        assert torch.equal(a, b)
    taken = _native.host().ragged_attention(q, q_starts, 0.125, 0, 0, None, cache["k_pages"], cache["v_pages"], table, lens, True, 0, 0, None, None, None)
    assert (taken is not None) == native
    taken = _native.host().head_norm_rope(q, k, None, None, None, 1e-6, cos, sin, None, True, None, None, None, None)
    assert (taken is not None) == native


def test_pages_beyond_4_gib(gpu):
    pages, page, Hk, D = 70000, 64, 4, 128     # 4.3 GiB of K and as much of V
    cache = initialize_paged_kv_cache(1, pages, page, Hk, D, gpu)[0]
    q, small, table, lens, q_starts = batch(111, [2, 70], [300, 200], 8, Hk, D, page, BF16, spare=0)
    far = pages - 1 - torch.arange(small["k_pages"].shape[0])
    k, v = (randn(i, sum([2, 70]), Hk, D).to(gpu) for i in (1, 2))
    for n in small:
        cache[n][far.to(gpu)] = small[n].to(gpu)
    far_table = torch.where(table < len(far), far.int()[table.clamp(max=len(far) - 1).long()], table)
    slots = paged_slots(far_table.to(gpu), lens.to(gpu), q_starts.to(gpu), 72, page)
    head_norm_rope_paged(q.to(gpu), k, v, cache, slots, None, None, 1e-6, None, None)
    near = paged_slots(table, lens, q_starts, 72, page)
    small["k_pages"].flatten(0, 1)[near], small["v_pages"].flatten(0, 1)[near] = k.cpu(), v.cpu()
    got = paged_attention(q.to(gpu), cache, far_table.to(gpu), lens.to(gpu), q_starts.to(gpu))
    keys_of, seen_of = ref.paged_keys(small, table, lens)
    close(got, *ref.ragged_attention(q, q_starts, D ** -0.5, keys_of, seen_of())[:2])


@pytest.mark.parametrize("new", [[1, 1], [80, 5]])
def test_scores_of_any_size(gpu, new):
    # weights of a single key, of all keys alike, rows of very large and of no scores
    q, cache, table, lens, q_starts = batch(121, new, [300, 90], 4, 2, 128, 16, BF16, scale=30.0)
    q[0], q[1] = 0.0, q[1] * 1000
    check_paged(gpu, (q, cache, table, lens, q_starts))
    check_paged(gpu, (q, cache, table, lens, q_starts), softmax_scale=1e-6)
    check_paged(gpu, batch(121, new, [300, 90], 4, 2, 128, 16, BF16), softmax_scale=3.0)


def test_nan_and_infinities_reach_the_rows_that_see_them(gpu):
    q, cache, table, lens, q_starts = batch(131, [70, 1], [70, 200], 2, 1, 64, 16, F16)
    page, row = table[0, 3].item(), 2       # key 50 of the first stream
    cache["k_pages"][page, row, 0, 0] = float("nan")
    got = paged_attention(q.to(gpu), {n: t.to(gpu) for n, t in cache.items()}, table.to(gpu), lens.to(gpu), q_starts.to(gpu)).cpu()
    assert torch.isfinite(got[:50]).all() and got[50:70].isnan().all() and torch.isfinite(got[70:]).all()


@pytest.mark.parametrize("D,dtype", [(64, F16), (128, BF16)])
@pytest.mark.parametrize("window,sink", [(None, 0), (40, 3)])
@pytest.mark.parametrize("bad", ["k_pages", "v_pages"])
@pytest.mark.parametrize("new,keys", [([150, 1, 9], [400, 300, 70]), ([1, 20], [900, 2000])])
def test_what_is_not_finite_stays_with_the_rows_that_see_it(gpu, new, keys, bad, window, sink, D, dtype):
    """NaN and infinities at keys that are later than a row or lie behind its window: they have no part in that row."""
    b = batch(136, new, keys, 4, 2, D, 16, dtype)
    q, cache, table, lens, q_starts = b
    clean = {n: t.clone() for n, t in cache.items()}
    at = [{keys[i] - n + j for j in (n // 3, n - 1)} | ({keys[i] - n - 60, keys[i] - 41, 7} if window else set()) for i, n in enumerate(new)]
    values = [float("nan"), float("inf"), -float("inf")]
    for i, places in enumerate(at):
        for j, place in enumerate(sorted(p for p in places if p >= 0)):
            cache[bad][table[i, place // 16], place % 16, :, 3 * j] = values[j % 3]
    got = paged_attention(q.to(gpu), {n: t.to(gpu) for n, t in cache.items()}, table.to(gpu), lens.to(gpu), q_starts.to(gpu), window=window, sink_tokens=sink).cpu()
    keys_of, seen_of = ref.paged_keys(clean, table, lens)
    want, error, _ = ref.ragged_attention(q, q_starts, D ** -0.5, keys_of, seen_of(True, window, sink))
    seen_at = [seen_of(True, window, sink)(i, n, keys[i])[:, sorted(p for p in at[i] if p >= 0)].any(1) for i, n in enumerate(new)]
    touched = torch.cat(seen_at)
    close(got[~touched], want[~touched], error[~touched])
    assert touched.any()
    if bad == "v_pages":   # the rows that see it have it, in the columns concerned (a score of -inf would weigh nothing, so not with K)
        assert not torch.isfinite(got[touched]).flatten(1).all(1).any()
        close(got[touched][:, :, 20:], want[touched][:, :, 20:], error[touched][:, :, 20:])


# ------------------------------------------------------------------------------------------------ cross attention
def cross(seed, new, states, Hq, Hk, D, dtype):
    q = randn(seed, sum(new), Hq, D, dtype=dtype, scale=1.5)
    k, v = (randn(seed + i, sum(states), Hk, D, dtype=dtype) for i in (1, 2))
    return q, k, v, starts(new), starts(states)


def check_cross(gpu, q, k, v, q_starts, k_starts, k_lens=None, key_mask=None, **kw):
    dev = lambda t: None if t is None else t.to(gpu)  # noqa: E731
    got = ragged_cross_attention(dev(q), dev(k), dev(v), dev(q_starts), dev(k_starts), k_lens=dev(k_lens), key_mask=dev(key_mask), **kw)
    at = k_starts.tolist()
    end = at[1:] if k_lens is None else [s + n for s, n in zip(at, k_lens.tolist())]
    keep = torch.ones(k.shape[0], dtype=torch.bool) if key_mask is None else key_mask
    want, error, _ = ref.ragged_attention(q, q_starts, q.shape[-1] ** -0.5, lambda b: (k[at[b]:end[b]], v[at[b]:end[b]]),
                                          lambda b, n, m: keep[at[b]:end[b]].expand(n, m))
    close(got, want, error)
    return got


@pytest.mark.parametrize("D,dtype", [(64, F16), (128, BF16)])
@pytest.mark.parametrize("new,states,Hq,Hk", [
    ([1], [1], 1, 1), ([1, 1, 1], [30, 500, 1], 4, 4), ([200, 3], [77, 226], 6, 2), ([64, 0, 129], [512, 10, 63], 2, 2), ([5, 5], [0, 70], 7, 1),
    ([2, 1], [3000, 2], 8, 8)])
def test_cross_attention(gpu, new, states, Hq, Hk, D, dtype):
    check_cross(gpu, *cross(201, new, states, Hq, Hk, D, dtype), max_q_len=max(new), max_k_len=max(states))


def test_no_states_at_all(gpu):
    q, k, _, q_starts, _ = cross(205, [3, 4], [1, 0], 4, 2, 64, BF16)
    none = torch.zeros(3, dtype=torch.int32, device=gpu)
    assert (ragged_cross_attention(q.to(gpu), k[:0].to(gpu), k[:0].to(gpu), q_starts.to(gpu), none) == 0).all()


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("new,states", [([300, 130, 2, 70], [2000, 40, 1500, 700]), ([1, 3], [3000, 2500])])
def test_many_states(gpu, new, states, masked):
    q, k, v, q_starts, k_starts = cross(206, new, states, 6, 2, 128, BF16)
    mask = torch.rand(k.shape[0], generator=torch.Generator().manual_seed(1)) < 0.7 if masked else None
    check_cross(gpu, q, k, v, q_starts, k_starts, key_mask=mask, max_q_len=max(new), max_k_len=max(states))


@pytest.mark.parametrize("new", [[1, 1, 1, 1], [100, 3, 40, 7]])
def test_masked_states(gpu, new):
    q, k, v, q_starts, k_starts = cross(211, new, [130, 64, 200, 9], 4, 2, 64, BF16)
    mask = torch.rand(k.shape[0], generator=torch.Generator().manual_seed(1)) < 0.5
    mask[130:194] = False                     # a request all of whose states are masked
    mask[194:300] = False                     # ... and one that begins with masked ones (padding on the left)
    k[~mask], v[~mask] = float("nan"), float("inf")
    got = check_cross(gpu, q, k, v, q_starts, k_starts, key_mask=mask)
    assert (got[new[0]:new[0] + new[1]] == 0).all()


def test_padded_batch_of_states(gpu):
    q, k, v, q_starts, _ = cross(221, [9, 9, 9], [64, 64, 64], 4, 4, 128, BF16)
    lens = torch.tensor([64, 0, 17], dtype=torch.int32)
    k.view(3, 64, 4, 128)[2, 17:] = float("nan")
    v.view(3, 64, 4, 128)[2, 17:] = float("nan")
    check_cross(gpu, q, k, v, q_starts, torch.tensor([0, 64, 128], dtype=torch.int32), k_lens=lens)
    # lengths that reach beyond the rows end with them, negative ones are none
    got = ragged_cross_attention(q.to(gpu), k.to(gpu)[:140], v.to(gpu)[:140], q_starts.to(gpu), torch.tensor([0, 64, 128], dtype=torch.int32, device=gpu),
                                 k_lens=torch.tensor([-5, 64, 1 << 30], dtype=torch.int32, device=gpu))
    assert (got[:9] == 0).all()
    k, v = k[:140], v[:140]
    want, error, _ = ref.ragged_attention(q[9:], starts([9, 9]), 128 ** -0.5, lambda b: ((k[64:128], v[64:128]), (k[128:], v[128:]))[b],
                                          lambda b, n, m: torch.ones(n, m, dtype=torch.bool))
    close(got[9:], want, error)


# ------------------------------------------------------------------------------------------------ together
def test_a_run_of_steps(gpu):
    """Two prompts, a step of single tokens, a chunk beside a single token: rotation, page write and attention over the cache step by step
    give what attention over each stream's whole sequence gives."""
    Hq, Hk, D, page, dtype = 4, 2, 64, 8, BF16
    cache = initialize_paged_kv_cache(1, 40, page, Hk, D, gpu, dtype)[0]
    for t in cache.values():
        t.fill_(float("nan"))
    table = torch.randperm(40, generator=torch.Generator().manual_seed(2)).int().view(2, 20)
    wq, wk = randn(1, D, dtype=dtype), randn(2, D, dtype=dtype)
    cos, sin = angles(160, D)
    lens, past = [0, 0], [[], []]
    for step, new in enumerate([[37, 70], [1, 1], [1, 20], [1, 1]]):
        T = sum(new)
        q, k, v = (randn(10 * step + i, T, h, D, dtype=dtype) for i, h in ((3, Hq), (4, Hk), (5, Hk)))
        lens = [a + b for a, b in zip(lens, new)]
        kv_lens, q_starts = torch.tensor(lens, dtype=torch.int32), starts(new)
        positions = torch.cat([torch.arange(L - n, L) for L, n in zip(lens, new)])
        slots = paged_slots(table.to(gpu), kv_lens.to(gpu), q_starts.to(gpu), T, page)
        assert torch.equal(slots.cpu(), torch.cat([table[b].long()[p // page] * page + p % page for b, p in enumerate(positions.split(new))]))
        roped = head_norm_rope_paged(q.to(gpu), k.to(gpu), v.to(gpu), cache, slots, wq.to(gpu), wk.to(gpu), 1e-6, cos.to(gpu), sin.to(gpu), positions.to(gpu),
                                     interleaved=False)
        got = paged_attention(roped, cache, table.to(gpu), kv_lens.to(gpu), q_starts.to(gpu), max_q_len=max(new), max_kv_len=max(lens))
        # the streams' whole sequences, K as the kernel that wrote it rounds it
        _, rotated = head_norm_rope(q.to(gpu), k.to(gpu), wq.to(gpu), wk.to(gpu), 1e-6, cos.to(gpu), sin.to(gpu), positions.to(gpu), interleaved=False)
        for b, (kk, vv) in enumerate(zip(rotated.cpu().split(new), v.split(new))):
            past[b].append((kk, vv))
        whole = [tuple(torch.cat(t) for t in zip(*p)) for p in past]
        want, error, _ = ref.ragged_attention(roped.cpu(), q_starts, D ** -0.5, lambda b: whole[b],
                                              lambda b, n, m: torch.arange(m) <= (m - n + torch.arange(n))[:, None])
        close(got, want, error, f"step {step}")


@pytest.mark.parametrize("new_most,keys_most", [(1, 3000), (150, 600)])
def test_recorded_steps_follow_the_lengths(gpu, new_most, keys_most):
    """Rotation, page write and both attentions in one graph, replayed with other lengths, beside eager work."""
    Hq, Hk, D, page, B = 8, 2, 128, 16, 3
    T, width = B * new_most, -(-keys_most // page)
    cache = initialize_paged_kv_cache(1, B * width, page, Hk, D, gpu)[0]
    for i, t in enumerate(cache.values()):
        t.copy_(randn(i, *t.shape))
    table = torch.randperm(B * width, generator=torch.Generator().manual_seed(2)).int().view(B, width).to(gpu)
    q, k, v = (randn(i, T, h, D).to(gpu) for i, h in ((3, Hq), (4, Hk), (5, Hk)))
    text = randn(6, 90, Hk, D).to(gpu)
    w = randn(7, D).to(gpu)
    cos, sin = (t.to(gpu) for t in angles(keys_most, D))
    kv_lens, q_starts = torch.ones(B, dtype=torch.int32, device=gpu), torch.zeros(B + 1, dtype=torch.int32, device=gpu)
    k_starts, positions = torch.zeros(B + 1, dtype=torch.int32, device=gpu), torch.zeros(T, dtype=torch.int64, device=gpu)
    slots = torch.full((T,), -1, dtype=torch.int64, device=gpu)

    def step():
        roped = head_norm_rope_paged(q, k, v, cache, slots, w, w, 1e-6, cos, sin, positions)
        x = paged_attention(roped, cache, table, kv_lens, q_starts, max_q_len=new_most, max_kv_len=keys_most)
        return x, ragged_cross_attention(x, text, text, q_starts, k_starts, max_q_len=new_most, max_k_len=90)

    def set_to(new, keys, states):
        q_starts.copy_(starts(new))
        kv_lens.copy_(torch.tensor(keys, dtype=torch.int32))
        k_starts.copy_(starts(states))
        slots.copy_(paged_slots(table, kv_lens, q_starts, T, page))

    steps = [([1] * B, [keys_most, 17, 300], [90, 0, 0]), ([new_most, 0, 1], [keys_most - 3, 40, 2], [30, 30, 30]),
             ([0, new_most, new_most], [5, new_most, keys_most], [0, 64, 26])]
    set_to(*steps[0])
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded = step()
    for lengths in steps + steps[::-1]:
        set_to(*lengths)
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in recorded]
        eager = step()
        torch.cuda.synchronize()
        for a, b in zip(replayed, eager):
            assert torch.isfinite(a).all() and torch.equal(a, b), lengths


def test_on_a_stream_of_its_own_and_twice_at_once(gpu):
    b = batch(141, [1, 1, 1], [5000, 300, 4000], 16, 2, 128, 16, BF16)
    q, table, lens, q_starts = (b[i].to(gpu) for i in (0, 2, 3, 4))
    cache = {n: t.to(gpu) for n, t in b[1].items()}
    args = dict(max_q_len=1, max_kv_len=5000)
    want = paged_attention(q, cache, table, lens, q_starts, **args)
    torch.cuda.synchronize()
    sides = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(3):
        for s in sides:
            with torch.cuda.stream(s):
                got.append(paged_attention(q, cache, table, lens, q_starts, **args))
    torch.cuda.synchronize()
    for g in got:
        assert torch.equal(g, want)


def test_same_bits_every_time(gpu):
    for new, keys in (([1, 1], [9000, 800]), ([300, 2], [2000, 700])):
        q, cache, table, lens, q_starts = batch(151, new, keys, 8, 2, 128, 16, BF16)
        args = (q.to(gpu), {n: t.to(gpu) for n, t in cache.items()}, table.to(gpu), lens.to(gpu), q_starts.to(gpu))
        first = paged_attention(*args, max_q_len=max(new), max_kv_len=max(keys))
        for _ in range(3):
            assert torch.equal(first, paged_attention(*args, max_q_len=max(new), max_kv_len=max(keys)))
