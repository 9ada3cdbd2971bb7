"""Attention over shared beginnings on the GPU where groups attend them together: a launch that lists the items, one that works them off, one that
joins their results.  The sizes are such that the division is this one, which is checked; against the plain 64-bit form."""
import ctypes

import pytest
import torch

import step_reference as step_ref
from longlive_amd import _native
from longlive_amd.utils.paged_kv import lay_out_step, shared_prefix_attention
from test_gpu_step import BF16, F16, attend, batch, check_shared, close, int32, randn, starts

pytestmark = pytest.mark.gpu


def parts_asked_for(b, told=True):
    """Whether the call asks for the records of parts of joined groups: more memory than the same keys in one table take, or as much for other things."""
    q, cache, prefix_table, prefix_lens, table, lens, q_starts = b
    k = cache["k_pages"]
    own = _native.RaggedAttentionStruct(dtype=_native.DTYPE_CODES[q.dtype], head_dim=q.shape[2], num_heads=q.shape[1], num_kv_heads=k.shape[2], n_queries=q.shape[0],
                                        streams=len(lens), softmax_scale=1.0, n_pages=k.shape[0], page_size=k.shape[1], table_width=table.shape[1], causal=1,
                                        max_q_len=int(q_starts.diff().max()) if told else 0, max_kv_len=int(lens.max()) if told else 0)
    a = _native.SharedPrefixStruct(own=own, groups=len(prefix_lens), prefix_width=prefix_table.shape[1], max_prefix_len=int(prefix_lens.max()) if told else 0)
    n = [ctypes.c_size_t(), ctypes.c_size_t()]
    lib = _native.load()
    assert lib.ll_shared_prefix_attention_workspace(ctypes.byref(a), 256, ctypes.byref(n[0])) == 0
    own.table_width += prefix_table.shape[1]
    own.max_kv_len = int(lens.max() + prefix_lens.max()) if told else 0
    assert lib.ll_ragged_attention_workspace(ctypes.byref(own), 256, ctypes.byref(n[1])) == 0
    return n[0].value != n[1].value


def check(gpu, b, group_starts=None, causal=True, **kw):
    assert parts_asked_for(b)
    return check_shared(gpu, b, group_starts, causal, **kw)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D,dtype", [(64, F16), (128, BF16), (128, F16), (64, BF16)])
def test_more_streams_than_the_listing_has_threads(gpu, D, dtype, causal):
    # single tokens, some of no stream's own keys, tiles for one wave each; idle streams among them
    g = torch.Generator().manual_seed(4)
    new = (torch.rand(300, generator=g) < 0.9).long().tolist()
    keys = torch.randint(0, 200, (300,), generator=g).tolist()
    b = batch(201, new, keys, [900], 8, 8, D, 16, dtype, fill=float("nan"))
    check(gpu, b, None, causal)


def test_many_streams_without_new_tokens(gpu):
    new = [int(i % 37 == 5) + 2 * int(i % 211 == 9) for i in range(3000)]
    b = batch(219, new, [(n + 17 * i % 90) * (n > 0) for i, n in enumerate(new)], [2000, 1500], 8, 8, 128, 16, BF16)
    check(gpu, b, [0, 1800, 2990])


@pytest.mark.parametrize("Hq,Hk,D,dtype", [(6, 3, 128, BF16), (20, 4, 64, F16), (12, 12, 64, BF16), (24, 24, 128, BF16)])
@pytest.mark.parametrize("page", [16, 24, 880])
def test_single_tokens_drafts_and_prompts_together(gpu, Hq, Hk, D, dtype, page):
    new = [1] * 12 + [4, 7, 0, 31, 33, 64] + [1] * 12 + [300, 129, 1, 2]
    keys = [n + 37 * i % 500 for i, n in enumerate(new)]
    check(gpu, batch(202, new, keys, [5000], Hq, Hk, D, page, dtype, fill=float("nan")))


def test_groups_of_which_some_are_joined(gpu):
    # lengths from none to long, groups of one stream, of none, streams outside, groups whose streams fill tiles by themselves
    new = [1] * 40 + [1] * 3 + [256, 384] + [2] * 30 + [1] * 5
    keys = [n + 13 * i % 300 for i, n in enumerate(new)]
    keys[50], keys[3] = 0, 0
    b = batch(203, new, keys, [6000, 0, 2500, 63, 4000, 100], 8, 4, 64, 16, F16, fill=float("nan"))
    check(gpu, b, [1, 40, 41, 45, 45, 60, 78])
    check(gpu, b, [1, 40, 41, 45, 45, 60, 78], causal=False)


@pytest.mark.parametrize("D,Hk", [(64, 8), (128, 2)])
def test_long_beginnings_of_groups_that_are_not_joined(gpu, D, Hk):
    # single streams, of few and of many rows, over beginnings as long as those that others share: in parts, beginning and own keys in one
    new = [1] * 40 + [1, 3, 200, 64, 1]
    keys = [n + 50 * (i % 9) for i, n in enumerate(new)]
    keys[44] = 0
    b = batch(212, new, keys, [5000, 6001, 4000, 5500, 3500, 4500], Hk, Hk, D, 16, BF16, fill=float("nan"))
    for causal in (True, False):
        check(gpu, b, [0, 40, 41, 42, 43, 44, 45], causal)


def test_more_groups_than_are_joined_in_a_launch(gpu):
    new = [1] * 600
    keys = [1 + 7 * i % 40 for i in range(600)]
    shared = [300 + 5 * g % 400 for g in range(300)]
    b = batch(204, new, keys, shared, 4, 4, 64, 16, BF16)
    assert not parts_asked_for(b)      # each stream goes over its group's beginning
    check_shared(gpu, b, list(range(0, 602, 2)))
    b = batch(205, new, keys, shared[:256], 4, 4, 64, 16, BF16)
    check_shared(gpu, b, list(range(0, 512, 2)) + [600])
    long = [1900 + n % 100 for n in shared]                       # one head: 256 groups are joined, 257 are not
    b = batch(210, new, keys, long[:256], 1, 1, 64, 16, BF16)
    check(gpu, b, list(range(0, 512, 2)) + [600])
    b = batch(211, new, keys, long[:257], 1, 1, 64, 16, BF16)
    assert not parts_asked_for(b)
    check_shared(gpu, b, list(range(0, 514, 2)) + [600])


def test_rows_of_joined_groups_that_see_the_beginning_only(gpu):
    # more new tokens than own keys, own keys in holes, a beginning of holes
    new = [5] * 30 + [1] * 30
    keys = [3] * 30 + [1] * 30
    b = batch(206, new, keys, [3000, 4000], 8, 4, 128, 16, BF16, fill=float("nan"))
    b[4][40:50] = -1
    check(gpu, b, [0, 30, 60])
    b[2][1] = -1
    got = check(gpu, b, [0, 30, 60])
    assert (got[150 + 10:150 + 20] == 0).all()


def test_what_is_not_finite_stays_with_the_rows_that_see_it(gpu):
    for new in ([3] * 60, [1] * 300, [90] * 6 + [1] * 50):
        keys = [n + 20 for n in new]
        b = batch(207, new, keys, [3000], 8, 8, 64, 8, BF16)
        last = keys[0] - 1                                        # seen by the first stream's last token alone
        want, error, _ = step_ref.shared_prefix(*b, None, True, 64 ** -0.5)   # rows that do not see it: what it is makes no difference
        b[1]["v_pages"][b[4][0, last // 8], last % 8, 0, 5] = float("inf")
        assert parts_asked_for(b)
        got = attend(gpu, b, max_q_len=max(new), max_kv_len=max(keys), max_prefix_len=3000)
        assert torch.isinf(got[new[0] - 1, 0, 5])
        keep = torch.ones_like(want, dtype=torch.bool)
        keep[new[0] - 1, 0, 5] = False
        close(torch.where(keep, got.cpu().double(), 0.0), torch.where(keep, want, 0.0), torch.where(keep, error, 1.0))


@pytest.mark.parametrize("told", [True, False])
def test_rows_outside_every_stream_and_results_in_place_of_the_queries(gpu, told):
    new, keys = [1] * 50 + [20, 3], [40] * 50 + [25, 90]
    b = list(batch(208, new + [9], keys + [9], [4000], 8, 8, 128, 16, BF16))
    b[4], b[5], b[6] = b[4][:-1], b[5][:-1], starts(new, first=4)      # four rows before, five behind
    rows = torch.zeros(sum(new) + 9, dtype=torch.bool)
    rows[4:4 + sum(new)] = True
    assert parts_asked_for(b, told)
    hints = dict(max_q_len=20, max_kv_len=90, max_prefix_len=4000) if told else {}
    got = check_shared(gpu, b, told=False, **hints)
    assert (got[~rows.to(gpu)] == 0).all()
    on = [t.to(gpu) for t in (b[0], *b[2:])]
    cache = {n: t.to(gpu) for n, t in b[1].items()}
    mine = on[0].clone()
    assert shared_prefix_attention(mine, cache, *on[1:], out=mine, **hints) is mine
    assert torch.equal(mine[rows.to(gpu)], got[rows.to(gpu)]) and torch.equal(mine[~rows.to(gpu)], on[0][~rows.to(gpu)])


def test_same_bits_every_time_and_beside_another_stream(gpu):
    new = [1] * 60 + [40, 17, 90]
    b = batch(209, new, [n + 11 * i % 300 for i, n in enumerate(new)], [4000], 16, 4, 128, 16, BF16)
    assert parts_asked_for(b)
    q, cache, *rest = b
    args = (q.to(gpu), {n: t.to(gpu) for n, t in cache.items()}, *(t.to(gpu) for t in rest))
    told = dict(max_q_len=90, max_kv_len=390, max_prefix_len=4000)
    want = shared_prefix_attention(*args, **told)
    torch.cuda.synchronize()
    got, sides = [shared_prefix_attention(*args, **told) for _ in range(5)], [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        for s in sides:
            with torch.cuda.stream(s):
                got.append(shared_prefix_attention(*args, **told))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_recorded_listing_follows_the_lengths(gpu):
    B, T, Hq, Hk, D, page, reach = 64, 200, 8, 8, 128, 16, 4000
    cache = {n: randn(i, 460, page, Hk, D).to(gpu) for i, n in enumerate(("k_pages", "v_pages"), 1)}
    q = randn(3, T, Hq, D).to(gpu)
    order = torch.randperm(460, generator=torch.Generator().manual_seed(1)).int()
    table = torch.randint(0, 460, (B, 6), generator=torch.Generator().manual_seed(2)).int().to(gpu)
    prefix_table = torch.stack([order[:250], order[200:450]]).contiguous().to(gpu)
    kv, q_starts, shared, cuts = int32([1] * B, gpu), int32([0] * (B + 1), gpu), int32([0, 0], gpu), int32([0, 0, 0], gpu)
    call = lambda: shared_prefix_attention(q, cache, prefix_table, shared, table, kv, q_starts, cuts, max_q_len=3, max_kv_len=96, max_prefix_len=reach)  # noqa: E731
    assert parts_asked_for((q, cache, prefix_table, int32([reach, reach]), table, int32([96] * B), starts([3] * B)))
    call()
    graphs = []
    for _ in range(2):   # two recordings, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, call()))
    cases = [([3] * 64, [96] * 64, [4000, 2000], [0, 30, 64]), ([1] * 64, [7] * 64, [0, 0], [0, 0, 64]), ([1] * 64, [1 + i for i in range(64)], [4000, 64], [0, 60, 64]),
             ([0] * 64, [0] * 64, [5, 5], [64, 64, 64]), ([100, 1] + [0] * 20 + [1] * 42, [90] * 64, [1500, 4000], [0, 2, 64]), ([1] * 64, [0] * 64, [4000, 3999], [1, 32, 63])]
    for i, (new, keys, lens, at) in enumerate(cases + cases[::-1]):
        q_starts.copy_(starts(new))
        for t, values in ((kv, keys), (shared, lens), (cuts, at)):
            t.copy_(int32(values))
        graph, recorded = graphs[i % 2]
        graph.replay()
        torch.cuda.synchronize()
        replayed = recorded.clone()
        eager = call()
        torch.cuda.synchronize()
        assert torch.isfinite(replayed).all() and torch.equal(replayed, eager), (new, keys, lens, at)
        if i < len(cases):
            want, error, _ = step_ref.shared_prefix(q.cpu(), {n: t.cpu() for n, t in cache.items()}, prefix_table.cpu(), int32(lens), table.cpu(), int32(keys), starts(new),
                                                    int32(at), True, D ** -0.5)
            close(replayed, want, error, f"case {i}")


@pytest.mark.parametrize("hints", [(1, 1, 2100), (None, 1, 4500), (10 ** 9, 10 ** 12, 10 ** 12)])
def test_lengths_that_the_host_takes_to_be_others(gpu, hints):
    new = [1] * 50 + [70, 3, 40]
    b = batch(213, new, [n + 31 * i % 1100 for i, n in enumerate(new)], [4300, 4500, 700], 16, 8, 64, 16, F16)
    check_shared(gpu, b, [0, 30, 52, 53], told=False, max_q_len=hints[0], max_kv_len=hints[1], max_prefix_len=hints[2])


def test_lengths_beyond_the_tables(gpu):
    b = list(batch(214, [1] * 40 + [3] * 20, [64] * 60, [3008], 8, 8, 64, 16, BF16))
    b[4] = b[4][:, :4].contiguous()
    assert parts_asked_for(b)
    want = attend(gpu, b, causal=False, max_q_len=3)
    b[3], b[5] = b[3] + 5000, b[5] + 1000
    assert torch.equal(attend(gpu, b, causal=False, max_q_len=3), want)


@pytest.mark.parametrize("page", [24, 16])
def test_strides(gpu, page):
    new = [1] * 60 + [2, 50]
    q, cache, *tables, q_starts = b = batch(215, new, [n + 9 * i % 200 for i, n in enumerate(new)], [4000], 8, 4, 128, page, BF16)
    want = check(gpu, b)
    T = sum(new)
    wide = torch.zeros(T, 11, 128, dtype=BF16, device=gpu)
    wide[:, 2:10] = q.to(gpu)
    both = torch.stack([cache["k_pages"], cache["v_pages"]], dim=1).transpose(2, 3).contiguous().to(gpu)   # [pages, 2, heads, rows, D]
    paged = {"k_pages": both[:, 0].transpose(1, 2), "v_pages": both[:, 1].transpose(1, 2)}
    out = torch.full((8, T, 128), 7.0, dtype=BF16, device=gpu).transpose(0, 1)
    on = [t.to(gpu) for t in tables]
    args = (paged, torch.cat([on[0], on[0]], dim=1)[:, :on[0].shape[1]], on[1], torch.cat([on[2], on[2]], dim=1)[:, :on[2].shape[1]], on[3], q_starts.to(gpu))
    told = dict(max_q_len=max(new), max_kv_len=int(tables[3].max()), max_prefix_len=4000)
    shared_prefix_attention(wide[:, 2:10], *args, out=out, **told)
    assert torch.equal(out, want)


@pytest.mark.parametrize("D,dtype", [(64, BF16), (128, F16)])
def test_scales(gpu, D, dtype):
    for scale in (0.01, 3.0):
        check(gpu, batch(216, [1] * 70, [30 + i for i in range(70)], [3000], 8, 8, D, 16, dtype), softmax_scale=scale)


def test_shared_values_that_are_not_finite(gpu):
    # a row that sees an infinite or undefined value has it, and no other column or group has
    new = [1] * 40 + [35] + [1] * 40
    b = batch(217, new, [n + 5 for n in new], [3000, 2500], 8, 8, 64, 8, BF16)
    want, error, _ = step_ref.shared_prefix(*b, int32([0, 41, 81]), True, 64 ** -0.5)
    b[1]["v_pages"][b[2][0, 100], 3, 2, 9] = float("inf")
    b[1]["v_pages"][b[2][1, 200], 4, 5, 11] = float("nan")
    assert parts_asked_for(b)
    got = attend(gpu, b, [0, 41, 81], max_q_len=35, max_kv_len=40, max_prefix_len=3000).cpu()
    inside = 75
    assert (got[:inside, 2, 9] == float("inf")).all() and got[inside:, 5, 11].isnan().all()
    keep = torch.ones_like(want, dtype=torch.bool)
    keep[:inside, 2, 9] = False
    keep[inside:, 5, 11] = False
    close(torch.where(keep, got.double(), 0.0), torch.where(keep, want, 0.0), torch.where(keep, error, 1.0))


def test_a_cache_beyond_32_bits_of_offsets(gpu):
    q, cache, *rest = b = batch(218, [1] * 60 + [40], [40 + i for i in range(61)], [3000], 8, 8, 64, 64, F16)
    assert parts_asked_for(b)
    pages = cache["k_pages"].shape[0]
    apart = (1 << 31) // pages // 64 * 64 + 64 * 1024
    far = torch.empty(pages, apart, dtype=F16, device=gpu)   # 2^31 elements and more between the first page and the last
    size = 64 * 8 * 64
    dev = {}
    for i, n in enumerate(("k_pages", "v_pages")):
        dev[n] = far[:, i * size:(i + 1) * size].unflatten(1, (64, 8, 64))
        dev[n].copy_(cache[n])
    got = shared_prefix_attention(q.to(gpu), dev, *(t.to(gpu) for t in rest), max_q_len=40, max_kv_len=100, max_prefix_len=3000)
    want, error, _ = step_ref.shared_prefix(q, cache, *rest, None, True, 64 ** -0.5)
    close(got, want, error)


def test_layout_with_a_cursor_beyond_the_list_or_below_it(gpu):
    for cursor, pages in ((7, [-1, -1]), (3, [-1, -1]), (2, [12, -1]), (-5, [10, 11])):
        table, at = torch.full((2, 2), -1, dtype=torch.int32, device=gpu), int32([cursor], gpu)
        got = lay_out_step(int32([1, 1], gpu), int32([0, 4], gpu), table, int32([10, 11, 12], gpu), 4, 2, cursor=at)
        assert [table[0, 0].item(), table[1, 1].item()] == pages and got.pages_wanted.item() == 2
        assert at.item() == {7: 7, 3: 3, 2: 3, -5: 2}[cursor]
        assert got.slots.tolist() == [4 * p if p >= 0 else -1 for p in pages]
