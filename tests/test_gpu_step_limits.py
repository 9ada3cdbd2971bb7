"""Operators around a step of several streams on the GPU where their limits are: batches of more rows than a joining launch takes at once or than memory for
many parts is had, groups and lengths outside what there is, results in a recorded rotation, tensors that a layout returns."""
import ctypes

import pytest
import torch

import step_reference as step_ref
from longlive_amd import _native
from longlive_amd.utils.paged_kv import lay_out_step
from longlive_amd.utils.rope import rotary_frequencies, rotate_by_position
from test_gpu_step import BF16, F16, attend, batch, check_layout, check_shared, close, int32, randn

pytestmark = pytest.mark.gpu


def workspace(b, told):
    """(bytes that a call of shared_prefix_attention asks for, bytes of one part's results)."""
    q, cache, prefix_table, prefix_lens, table, lens, q_starts = b
    k = cache["k_pages"]
    own = _native.RaggedAttentionStruct(dtype=_native.DTYPE_CODES[q.dtype], head_dim=q.shape[2], num_heads=q.shape[1], num_kv_heads=k.shape[2], n_queries=q.shape[0],
                                        streams=len(lens), softmax_scale=1.0, n_pages=k.shape[0], page_size=k.shape[1], table_width=table.shape[1], causal=1,
                                        max_q_len=told["max_q_len"], max_kv_len=told["max_kv_len"])
    a = _native.SharedPrefixStruct(own=own, groups=len(prefix_lens), prefix_width=prefix_table.shape[1], max_prefix_len=told["max_prefix_len"])
    n = ctypes.c_size_t()
    assert _native.load().ll_shared_prefix_attention_workspace(ctypes.byref(a), 256, ctypes.byref(n)) == 0
    return n.value, q.shape[0] * q.shape[1] * (q.shape[2] + 2) * 4


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("Hq,Hk,D,dtype,shared,parts", [(8, 8, 64, F16, 700, 5), (20, 4, 128, BF16, 1500, 4), (64, 16, 64, BF16, 1000, 2)])
def test_joined_groups_of_more_rows_than_a_joining_launch_takes_at_once(gpu, Hq, Hk, D, dtype, shared, parts, causal):
    # 5400 rows, of which the joining launch has 4096 tokens to a turn; with 20 heads of 128 columns three parts of the beginning and one of own keys,
    # with 64 of 64 one and one
    new = [9] * 600
    keys = [9 + 7 * i % 23 for i in range(600)]
    b = batch(301, new, keys, [shared], Hq, Hk, D, 16, dtype, fill=float("nan"))
    told = dict(max_q_len=9, max_kv_len=max(keys), max_prefix_len=shared)
    asked, part = workspace(b, told)
    assert asked // part >= parts and (parts != 2 or asked // part == 2)
    got = attend(gpu, b, None, causal, **told)
    q, cache, *rest = b
    kv = [0, Hk - 1]                         # of all heads the first and the last kv head's
    heads = [h for h in range(Hq) if h // (Hq // Hk) in kv]
    want, error, _ = step_ref.shared_prefix(q[:, heads], {n: t[:, :, kv] for n, t in cache.items()}, *rest, None, causal, D ** -0.5)
    close(got[:, heads], want, error)
    assert torch.isfinite(got).all() and torch.equal(attend(gpu, b, None, causal, **told), got)


@pytest.mark.parametrize("new", [[1, 2, 1, 3], [1] * 70])
def test_groups_that_begin_ahead_of_the_first_stream_or_end_behind_the_last(gpu, new):
    keys = [n + 5 * i % 60 for i, n in enumerate(new)]
    B = len(new)
    b = batch(302, new, keys, [3000, 2000, 1000], 8, 8, 64, 16, BF16, fill=float("nan"))
    for cuts in ([-5, B // 2, B, B + 9], [-9, -5, B // 2, B + 7], [B // 2, B + 1, B + 2, 2 ** 31 - 1], [-(2 ** 31), 1, B // 2, 2 ** 31 - 1]):
        check_shared(gpu, b, cuts)
        check_layout(gpu, new, keys, 9, 16, prefix_lens=b[3].tolist(), group_starts=cuts)


@pytest.mark.parametrize("new", [[1, 2, 1, 3], [1] * 70])
def test_negative_lengths_are_none(gpu, new):
    keys = [n + 5 * i % 60 for i, n in enumerate(new)]
    half = len(new) // 2
    b = list(batch(303, new, keys, [3000, 2000], 8, 8, 64, 16, BF16, fill=float("nan")))
    told = dict(max_q_len=max(new), max_kv_len=max(keys), max_prefix_len=3000)
    for lens, shared in ((b[5].clone(), int32([-7, 2000])), (b[5].clone(), int32([3000, -(2 ** 31)])), (b[5].clone(), int32([-1, -1]))):
        lens[1] = -3
        lens[-1] = -(2 ** 31)
        got = attend(gpu, (*b[:3], shared, b[4], lens, b[6]), [0, half, len(new)], **told)
        want, error, _ = step_ref.shared_prefix(*b[:3], shared.clamp(min=0), b[4], lens.clamp(min=0), b[6], int32([0, half, len(new)]), True, 64 ** -0.5)
        close(got, want, error)


def test_a_recorded_rotation_follows_its_positions(gpu):
    T, f = 130, rotary_frequencies(128)
    q, k = randn(1, T, 8, 128), randn(2, T, 2, 128)
    on, positions, at = (q.to(gpu), k.to(gpu)), torch.zeros(T, dtype=torch.int64, device=gpu), f.to(gpu)
    call = lambda: rotate_by_position(*on, positions, at, interleaved=False)  # noqa: E731
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded = call()
    for seed in range(4):
        where = torch.randint(0, 1 << 20, (T,), generator=torch.Generator().manual_seed(seed))
        positions.copy_(where)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in recorded]
        for x, y, eager in zip((q, k), got, call()):
            close(y, *step_ref.rotate(x, None, 0.0, f, where, False))
            assert torch.equal(y, eager)


def test_what_a_layout_returns_is_written_to_without_harm(gpu):
    # results share allocations: writing to one of them leaves the others as they are
    got = lay_out_step(int32([2, 1], gpu), int32([3, 16], gpu), int32([[5, -1], [6, -1]], gpu), int32([8, 9], gpu), 16, 4)
    before = [t.clone() for t in got]
    for i, t in enumerate(got):
        assert t.is_contiguous() and t.data_ptr() % t.element_size() == 0
        t.fill_(-1)
        for j, (other, was) in enumerate(zip(got, before)):
            assert torch.equal(other, was if j > i else torch.full_like(was, -1))
    assert [t.tolist() for t in before] == [[0, 2, 3], [5, 17], [3, 4, 16, 0], [83, 84, 128, -1], [1]]
