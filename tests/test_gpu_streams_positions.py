"""Positions of the new tokens of several streams where lengths reach beyond what is there: token i of a stream's n sits at
``kv_lens[b] - n + i`` also where its page table ends before its keys do, and where its rows end before ``q_starts`` do."""
import pytest
import torch

import streams_reference as ref
from longlive_amd.utils.paged_kv import paged_attention, paged_slots
from test_gpu_streams import BF16, F16, batch, close, starts

pytestmark = pytest.mark.gpu


def seen_of(table, lens, page, pages, causal, window, sink):
    """What token i of stream b's n sees of the m keys that its table reaches: by positions that no table bounds."""
    def seen(b, n, m):
        j, p = torch.arange(m), (int(lens[b]) - n + torch.arange(n))[:, None]
        entry = table[b].long()[j // page]
        s = ((entry >= 0) & (entry < pages)).expand(n, m).clone()
        if causal:
            s &= j <= p
        if window:
            s &= (j > p - window) | (j < sink)
        return s
    return seen


def check(gpu, b, reach, causal, window, sink, **kw):
    """A batch through paged attention with the first `reach` columns of its page table."""
    q, cache, table, lens, q_starts = b
    table, page = table[:, :reach].contiguous(), cache["k_pages"].shape[1]
    got = paged_attention(q.to(gpu), {n: t.to(gpu) for n, t in cache.items()}, table.to(gpu), lens.to(gpu), q_starts.to(gpu), causal=causal, window=window,
                          sink_tokens=sink, **kw)
    keys_of, _ = ref.paged_keys(cache, table, lens)
    seen = seen_of(table, lens, page, cache["k_pages"].shape[0], causal, window, sink)
    want, error, _ = ref.ragged_attention(q, q_starts, q.shape[-1] ** -0.5, keys_of, seen)
    close(got, want, error)


@pytest.mark.parametrize("D,dtype", [(64, F16), (128, BF16)])
@pytest.mark.parametrize("causal,window,sink", [(True, None, 0), (True, 40, 0), (True, 40, 3), (False, 40, 3), (True, 64, 130), (True, 3, 64), (False, None, 0)])
@pytest.mark.parametrize("new,keys,reach", [([10], [100], 4), ([1, 1, 1], [65, 64, 300], 4), ([150, 30], [400, 333], 18), ([150, 3], [200, 100], 4), ([90], [100], 1)])
def test_a_table_that_ends_before_its_keys(gpu, new, keys, reach, causal, window, sink, D, dtype):
    check(gpu, batch(201, new, keys, 4, 2, D, 16, dtype), reach, causal, window, sink)


@pytest.mark.parametrize("D,dtype", [(64, F16), (128, BF16)])
@pytest.mark.parametrize("causal,window,sink", [(True, None, 0), (True, 3000, 130), (False, 2500, 70), (True, 1500, 0)])
@pytest.mark.parametrize("new,keys,reach", [([150, 1], [5000, 4000], 290), ([300], [5000], 305), ([1, 2], [9000, 6400], 400)])
def test_the_same_in_parts(gpu, new, keys, reach, causal, window, sink, D, dtype):
    check(gpu, batch(202, new, keys, 2, 1, D, 16, dtype), reach, causal, window, sink, max_q_len=max(new), max_kv_len=16 * reach)


def test_as_the_slots_of_the_new_tokens(gpu):
    """One token of ten lies in the table's last page, the others behind it: those without a slot see the keys before them all the same."""
    q, cache, table, lens, q_starts = batch(203, [10], [65 + 8], 4, 2, 64, 16, BF16)
    table = table[:, :4].contiguous()
    slots = paged_slots(table, lens, q_starts, 10, 16)
    assert (slots >= 0).tolist() == [True] + [False] * 9
    check(gpu, (q, cache, table, lens, q_starts), 4, True, None, 0)


@pytest.mark.parametrize("causal,window", [(True, None), (True, 30), (False, 30)])
@pytest.mark.parametrize("new,rows", [(12, 8), (200, 130)])
def test_rows_that_end_before_their_stream(gpu, new, rows, causal, window):
    """q holds the first rows of a stream whose q_starts go on: the rows that are there as if the others were too."""
    q, cache, table, lens, q_starts = batch(204, [new], [300], 4, 2, 64, 16, BF16)
    dev = {n: t.to(gpu) for n, t in cache.items()}
    rest = (dev, table.to(gpu), lens.to(gpu), q_starts.to(gpu), causal, window)
    got = paged_attention(q[:rows].to(gpu), *rest)
    keys_of, seen = ref.paged_keys(cache, table, lens)
    want, error, _ = ref.ragged_attention(q, q_starts, 64 ** -0.5, keys_of, seen(causal, window, 0))
    close(got, want[:rows], error[:rows])


@pytest.mark.parametrize("causal,window", [(True, None), (True, 30)])
def test_streams_that_begin_before_the_rows(gpu, causal, window):
    q, cache, table, lens, _ = batch(205, [12], [300], 4, 2, 64, 16, BF16)
    got = paged_attention(q[4:].to(gpu), {n: t.to(gpu) for n, t in cache.items()}, table.to(gpu), lens.to(gpu), starts([12], first=-4).to(gpu), causal, window)
    keys_of, seen = ref.paged_keys(cache, table, lens)
    want, error, _ = ref.ragged_attention(q, starts([12]), 64 ** -0.5, keys_of, seen(causal, window, 0))
    close(got, want[4:], error[4:])
