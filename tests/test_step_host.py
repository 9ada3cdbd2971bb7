"""CPU tests of the operators around a step of several streams: what they refuse before any launch, their plain forms by hand, frequencies."""
import ctypes
import math

import pytest
import torch

import step_reference as step_ref
from longlive_amd import _native
from longlive_amd.utils.paged_kv import initialize_paged_kv_cache, lay_out_step, paged_slots, rotate_by_position_paged, shared_prefix_attention
from longlive_amd.utils.rope import build_rope_angles, rope_params, rotary_frequencies, rotate_by_position, video_frequencies

BF16, INT = torch.bfloat16, torch.int32


def i32(*shape):
    return torch.zeros(shape, dtype=INT)


def test_plain_layout_by_hand():
    # pages of 4: the first stream goes on in its second page and takes one more, the second begins, the third finds the list at its end
    q_starts, lens, positions, slots, wanted, table, cursor = step_ref.step_layout([3, 2, 1], [6, 0, 4], [[9, 8, -1], [-1] * 3, [7, -1, -1]], [5, 3], 4, 8, [10, 100], [0, 2, 3])
    assert q_starts == [0, 3, 5, 6] and lens == [9, 2, 5] and wanted == 3 and cursor == 2
    assert positions == [16, 17, 18, 10, 11, 104, 0, 0] and slots == [34, 35, 20, 12, 13, -1, -1, -1]
    assert table == [[9, 8, 5], [3, -1, -1], [7, -1, -1]]
    # what the chain of torch operations makes of the result
    assert paged_slots(torch.tensor(table), torch.tensor(lens), torch.tensor(q_starts), 8, 4).tolist() == slots


def test_plain_shared_prefix_by_hand():
    q = torch.tensor([[[1.0]], [[0.0]]]).to(BF16)
    cache = {"k_pages": torch.tensor([0.0, 1.0, 2.0, 9.0]).to(BF16).view(4, 1, 1, 1), "v_pages": torch.tensor([1.0, 2.0, 4.0, 100.0]).to(BF16).view(4, 1, 1, 1)}
    # both streams share the first page; the first owns the second, the other one the third and what comes later
    want, error, rows = step_ref.shared_prefix(q, cache, torch.tensor([[0]], dtype=INT), torch.tensor([1], dtype=INT), torch.tensor([[1, -1], [2, 3]], dtype=INT),
                                               torch.tensor([1, 1], dtype=INT), torch.tensor([0, 1, 2], dtype=INT), None, True, 1.0)
    e = math.e
    assert want.flatten().tolist() == pytest.approx([(1 + 2 * e) / (1 + e), 2.5]) and (error > 0).all() and rows.all()


def test_frequencies():
    # powers and a reciprocal, each within a step of 64 bits
    assert torch.allclose(rotary_frequencies(64), rope_params(2, 64)[1], rtol=2.0 ** -50, atol=0.0)
    f, sections = video_frequencies(128)
    assert torch.equal(f, build_rope_angles(128, 2)[1]) and sections == (22, 21, 21)
    assert torch.equal(rotary_frequencies(8, scaling="positions", factor=4.0), rotary_frequencies(8) / 4.0)
    stretched = rotary_frequencies(64, scaling="base", factor=8.0)
    assert stretched[0] == 1.0 and stretched[-1].item() == pytest.approx(rotary_frequencies(64)[-1].item() / 8.0)
    f, parts = rotary_frequencies(128), rotary_frequencies(128, scaling="parts", factor=16.0, trained_positions=4096)
    turns = f * 4096 / (2 * math.pi)
    assert torch.equal(parts[turns >= 32], f[turns >= 32]) and torch.allclose(parts[turns <= 1], f[turns <= 1] / 16, rtol=1e-15)
    between = (turns > 1) & (turns < 32)
    assert between.any() and ((parts < f) & (parts > f / 16))[between].all() and (parts.diff() < 0).all()
    for bad in (dict(rotary_dim=7), dict(rotary_dim=0), dict(base=0.0), dict(factor=2.0), dict(scaling="others"), dict(scaling="base", factor=-1.0),
                dict(scaling="base", factor=2.0, rotary_dim=2), dict(scaling="parts", factor=2.0), dict(scaling="parts", factor=2.0, trained_positions=64, slow=3.0, fast=2.0)):
        with pytest.raises(ValueError):
            rotary_frequencies(**{**dict(rotary_dim=64), **bad})


def test_operators_run_on_the_gpu_only():
    x, f = torch.zeros(3, 2, 64, dtype=BF16), rotary_frequencies(64)
    cache = initialize_paged_kv_cache(1, 4, 16, 2, 64, "cpu")[0]
    with pytest.raises(ValueError, match="GPU"):
        lay_out_step(i32(2), i32(2), i32(2, 3), i32(5), 16, 4)
    with pytest.raises(ValueError, match="GPU"):
        rotate_by_position(x, x, None, f)
    with pytest.raises(ValueError, match="GPU"):
        rotate_by_position_paged(x, x, x, cache, torch.zeros(3, dtype=torch.int64), None, f)
    with pytest.raises(ValueError, match="GPU"):
        shared_prefix_attention(x, cache, i32(1, 2), i32(1), i32(1, 2), i32(1), i32(2))


@pytest.fixture
def no_gpu_needed(monkeypatch):
    """The checks of the Python layer with the check of the device taken out, and a library that must not be reached."""
    monkeypatch.setattr(_native, "_require_cuda", lambda *t: None)
    monkeypatch.setattr(_native, "load", lambda: pytest.fail("the call was not refused"))


def test_refusals_of_the_layout(no_gpu_needed):
    ok = dict(new_lens=i32(2), kv_lens=i32(2), page_table=i32(2, 3), free_pages=i32(5), page_size=16, num_tokens=4)
    for bad in (dict(new_lens=i32(3)), dict(new_lens=i32(2).long()), dict(new_lens=i32(4)[::2]), dict(kv_lens=i32(1)), dict(kv_lens=i32(2).float()), dict(page_table=i32(3, 3)),
                dict(page_table=i32(2, 3).long()), dict(page_table=i32(6)), dict(page_table=i32(3, 2).T), dict(page_table=i32(1, 3).expand(2, 3)),
                dict(page_table=torch.zeros(9, dtype=INT).as_strided((2, 3), (2, 1))), dict(free_pages=i32(5).long()), dict(free_pages=i32(5, 1)), dict(free_pages=i32(10)[::2]),
                dict(page_size=0), dict(page_size=1 << 31), dict(page_size=1.5), dict(num_tokens=-1), dict(num_tokens=1 << 31), dict(prefix_lens=i32(2)),
                dict(prefix_lens=i32(0)), dict(prefix_lens=i32(1).long()), dict(group_starts=i32(2)), dict(prefix_lens=i32(2), group_starts=i32(2)),
                dict(prefix_lens=i32(2), group_starts=i32(3).long()), dict(cursor=i32(2)), dict(cursor=torch.zeros(1, dtype=torch.int64)), dict(kv_lens_out=i32(3)),
                dict(kv_lens_out=i32(2).long())):
        with pytest.raises(ValueError):
            lay_out_step(**{**ok, **bad})


def test_refusals_of_rotation(no_gpu_needed):
    x, w, f = torch.zeros(3, 2, 64, dtype=BF16), torch.zeros(64, dtype=BF16), rotary_frequencies(64)
    slots = torch.zeros(3, dtype=torch.int64)
    cache = initialize_paged_kv_cache(1, 4, 16, 2, 64, "cpu")[0]
    ok = dict(q=x, k=x, positions=slots, frequencies=f)
    for bad in (dict(q=x.float()), dict(q=x[0]), dict(k=x.half()), dict(k=x[:2]), dict(k=x[..., :56]), dict(q_weight=w[:8]), dict(q_weight=w.half()), dict(k_weight=w.double()),
                dict(positions=slots.int()), dict(positions=slots[:2]), dict(frequencies=f.float()), dict(frequencies=f[:30]), dict(frequencies=f.view(4, 8)),
                dict(frequencies=rotary_frequencies(72)), dict(grid=(2, 3)), dict(sections=(12, 10, 10)), dict(grid=(2, 3), sections=(12, 10, 9)),
                dict(grid=(0, 3), sections=(12, 10, 10)), dict(grid=(2, 3, 4), sections=(12, 10, 10)), dict(grid=(1 << 16, 1 << 15), sections=(12, 10, 10)),
                dict(grid=(2, 3), sections=(42, -10, 0)), dict(grid=(2.5, 3), sections=(12, 10, 10)), dict(amplitude=float("nan")), dict(amplitude=float("inf")),
                dict(q=torch.zeros(3, 2, 264, dtype=BF16), k=torch.zeros(3, 2, 264, dtype=BF16))):
        with pytest.raises(ValueError):
            rotate_by_position(**{**ok, **bad})
    ok.update(v=x, cache=cache, slots=slots)
    half = {n: t.half() for n, t in cache.items()}
    for bad in (dict(v=x[:, :1]), dict(v=x.half()), dict(slots=slots[:2]), dict(slots=slots.int()), dict(cache=half), dict(out=x.half()), dict(out=x[:2]),
                dict(cache=initialize_paged_kv_cache(1, 4, 16, 3, 64, "cpu")[0])):
        with pytest.raises(ValueError):
            rotate_by_position_paged(**{**ok, **bad})


def test_amplitudes_beyond_32_bits_are_refused(no_gpu_needed):
    # infinite in the kernel, they would make zeros undefined
    x, f = torch.zeros(3, 2, 64, dtype=BF16), rotary_frequencies(64)
    for amplitude in (1e39, -1e39, 3.5e38):
        with pytest.raises(ValueError, match="amplitude"):
            rotate_by_position(x, x, None, f, amplitude=amplitude)


def test_library_refuses_amplitudes_that_are_not_finite():
    rows = _native.HeadRowsStruct(num_heads=0)
    for amplitude, want in ((1e39, -1), (float("nan"), -1), (3.4e38, 0)):
        angles = _native.PositionAnglesStruct(amplitude=amplitude)
        assert _native.load().ll_rotate_by_position(0, 1, 64, ctypes.byref(rows), ctypes.byref(rows), None, 0.0, ctypes.byref(angles), None, 1, None, 0, None) == want


def test_refusals_of_shared_prefix_attention(no_gpu_needed):
    q = torch.zeros(3, 4, 64, dtype=BF16)
    cache = initialize_paged_kv_cache(1, 4, 16, 2, 64, "cpu")[0]
    ok = dict(q=q, cache=cache, prefix_table=i32(2, 3), prefix_lens=i32(2), page_table=i32(2, 5), kv_lens=i32(2), q_starts=i32(3), group_starts=i32(3))
    three = initialize_paged_kv_cache(1, 4, 16, 3, 64, "cpu")[0]
    for bad in (dict(q=q.float()), dict(q=q.half()), dict(q=q[0]), dict(q=torch.zeros(3, 4, 96, dtype=BF16)), dict(cache=three), dict(page_table=i32(2, 5).long()),
                dict(page_table=i32(3, 5)), dict(page_table=i32(2, (1 << 26) + 1)), dict(prefix_table=i32(2, (1 << 26) + 1)), dict(prefix_table=i32(1, 3)),
                dict(prefix_table=i32(2, 3).long()), dict(prefix_table=i32(3, 2).T), dict(prefix_table=i32(6)), dict(prefix_lens=i32(3)), dict(prefix_lens=i32(2).long()),
                dict(prefix_lens=i32(4)[::2]), dict(group_starts=None), dict(group_starts=i32(2)), dict(group_starts=i32(3).long()), dict(kv_lens=i32(3)),
                dict(q_starts=i32(2)), dict(q_starts=i32(0)), dict(softmax_scale=0.0), dict(softmax_scale=float("nan")), dict(max_q_len=-1), dict(max_kv_len=-1),
                dict(max_prefix_len=-1), dict(max_prefix_len=0.5), dict(out=q.half()), dict(out=q[:2]), dict(out=torch.zeros(1, 4, 64, dtype=BF16).expand(3, 4, 64))):
        with pytest.raises(ValueError):
            shared_prefix_attention(**{**ok, **bad})


# ------------------------------------------------------------------------------------------------ the C ABI's own checks, none of which reach the device
def shared_args(**kw):
    own = {**dict(dtype=0, head_dim=128, num_heads=4, num_kv_heads=2, softmax_scale=0.1, n_queries=8, streams=4, page_size=16, table_width=4, n_pages=9), **kw.pop("own", {})}
    return _native.SharedPrefixStruct(own=_native.RaggedAttentionStruct(**own), **{**dict(groups=1, prefix_width=100), **kw})


def shared_bytes(args):
    n = ctypes.c_size_t()
    code = _native.load().ll_shared_prefix_attention_workspace(ctypes.byref(args), 256, ctypes.byref(n))
    return n.value if code == 0 else code


@pytest.mark.parametrize("bad", [dict(groups=-1), dict(prefix_width=-1), dict(prefix_width=(1 << 26) + 1), dict(max_prefix_len=-1), dict(own=dict(window=4)),
                                 dict(own=dict(sink_keys=4)), dict(own=dict(page_size=0)), dict(own=dict(table_width=(1 << 26) + 1)), dict(own=dict(head_dim=96)),
                                 dict(own=dict(dtype=2)), dict(own=dict(n_queries=-1)), dict(own=dict(num_heads=5)), dict(own=dict(softmax_scale=0.0))])
def test_library_refuses_shared_prefixes(bad):
    assert shared_bytes(shared_args(**bad)) == -1 and _native.load().ll_last_error()


def test_library_refuses_null_pointers():
    lib = _native.load()
    assert lib.ll_shared_prefix_attention(None, None) == -1 and lib.ll_step_layout(None, None) == -1
    assert lib.ll_shared_prefix_attention(ctypes.byref(shared_args()), None) == -1
    assert lib.ll_shared_prefix_attention(ctypes.byref(shared_args(own=dict(n_queries=0))), None) == 0   # nothing to do
    a = _native.StepLayoutStruct(streams=2, page_size=16, table_width=3, tokens=4)
    assert lib.ll_step_layout(ctypes.byref(a), None) == -1
    rows = _native.HeadRowsStruct(num_heads=0)
    angles = _native.PositionAnglesStruct(rotary_dim=64, amplitude=1.0)
    call = lambda angles, tokens=1: lib.ll_rotate_by_position(0, tokens, 64, ctypes.byref(rows), ctypes.byref(rows), None, 0.0, angles, None, 1, None, 0, None)  # noqa: E731
    assert call(None) == -1 and call(ctypes.byref(angles)) == -1
    angles.rotary_dim = 0
    assert call(ctypes.byref(angles)) == 0   # no heads
    for rows_columns in ((1, 0), (0, 1), (-1, -1), (1 << 16, 1 << 15)):
        angles.grid_rows, angles.grid_columns = rows_columns
        assert call(ctypes.byref(angles)) == -1
    angles.grid_rows = angles.grid_columns = 2
    for pairs in ((1, 0), (0, 1), (-1, 0)):
        angles.frame_pairs, angles.row_pairs = pairs
        assert call(ctypes.byref(angles)) == -1


@pytest.mark.parametrize("bad", [dict(streams=-1), dict(streams=1 << 31), dict(tokens=-1), dict(tokens=1 << 31), dict(page_size=0), dict(table_width=-1), dict(n_free=-1),
                                 dict(groups=-1), dict(n_free=1 << 31), dict(table_width=1 << 31)])
def test_library_refuses_layouts(bad):
    a, n = _native.StepLayoutStruct(**{**dict(streams=2, page_size=16, table_width=3, tokens=4), **bad}), ctypes.c_size_t()
    assert _native.load().ll_step_layout_workspace(ctypes.byref(a), ctypes.byref(n)) == -1


def test_library_refuses_layouts_whose_numbers_pass_31_bits_in_the_kernel():
    n = ctypes.c_size_t()
    for more, want in ((dict(streams=(1 << 31) - 2), -1), (dict(streams=1 << 28), -1), (dict(groups=(1 << 31) - 2), -1), (dict(groups=1 << 28), -1),
                       (dict(streams=(1 << 28) - 1, groups=(1 << 28) - 1), 0)):
        a = _native.StepLayoutStruct(**{**dict(streams=2, page_size=16, table_width=3, tokens=4), **more})
        assert _native.load().ll_step_layout_workspace(ctypes.byref(a), ctypes.byref(n)) == want, more


# addresses that no call reaches: without a device a layout that is not refused ends at its launch, which fails
def layout_args(**kw):
    return _native.StepLayoutStruct(**{**dict(streams=4, new_lens=0x1000, kv_lens=0x2000, page_table=0x3000, table_stride=10, table_width=8, page_size=16, free_pages=0x4000,
                                              n_free=5, cursor=0x4100, groups=2, group_starts=0x4200, prefix_lens=0x4300, tokens=6, q_starts=0x5000, kv_lens_out=0x6000,
                                              positions=0x7000, slots=0x8000, pages_wanted=0x9000), **kw})


TABLE_ENDS = 0x3000 + 4 * (3 * 10 + 8)


@pytest.mark.parametrize("tokens", [6, 5000])
@pytest.mark.parametrize("bad", [
    dict(kv_lens_out=0x1000), dict(kv_lens_out=0x1000 - 12), dict(kv_lens_out=0x2004), dict(kv_lens_out=0x1FFC), dict(kv_lens_out=0x4010), dict(kv_lens_out=0x4208),
    dict(kv_lens_out=0x4304), dict(cursor=0x1000), dict(cursor=0x200C), dict(cursor=0x4010), dict(cursor=0x4208), dict(cursor=0x4304), dict(cursor=0x6004),
    dict(page_table=0x1000), dict(kv_lens=0x3000), dict(kv_lens=0x3000 - 4), dict(new_lens=0x3004), dict(new_lens=0x3000 + 4 * 8), dict(free_pages=0x3000 + 4 * 17),
    dict(cursor=0x3000 + 4 * 10), dict(cursor=TABLE_ENDS - 4), dict(kv_lens_out=0x3000 + 4 * 9), dict(prefix_lens=TABLE_ENDS - 4), dict(group_starts=0x3000 - 8),
    dict(q_starts=0x1004), dict(q_starts=0x6000 - 16), dict(positions=0x2000), dict(slots=0x7000 + 8 * 5), dict(pages_wanted=0x4100), dict(pages_wanted=0x4300),
    dict(table_stride=7), dict(table_stride=0), dict(table_stride=-7), dict(table_stride=-10, cursor=0x3000 - 4 * 30)])
def test_library_refuses_layouts_that_overlap(bad, tokens):
    lib = _native.load()
    kept = dict(workspace=0x100000, workspace_bytes=1 << 12)
    if tokens > 6:
        kept.update(positions=0x200000, slots=0x300000)   # long ones
    moved = {"positions": 0x1FF8, "slots": 0x200000 + 8 * (tokens - 1)} if tokens > 6 else {}
    bad = {n: moved.get(n, at) for n, at in bad.items()}
    assert lib.ll_step_layout(ctypes.byref(layout_args(**{**dict(tokens=tokens), **kept, **bad})), None) == -1
    assert b"overlap" in lib.ll_last_error()


@pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses are nobody's: only where no launch can come of them")
@pytest.mark.parametrize("good", [
    dict(), dict(kv_lens_out=0x2000), dict(kv_lens_out=0x1010), dict(kv_lens_out=0x2000 - 16), dict(cursor=0x2010), dict(cursor=0x2000 - 4), dict(cursor=TABLE_ENDS),
    dict(cursor=0x3000 + 4 * 8), dict(cursor=0x3000 + 4 * 29), dict(cursor=0x3000 - 4), dict(prefix_lens=0x3000 + 4 * 18), dict(group_starts=TABLE_ENDS),
    dict(new_lens=0x2000), dict(prefix_lens=0x1000), dict(cursor=None), dict(groups=0, group_starts=0x2000, prefix_lens=None, kv_lens_out=0x2000),
    dict(table_width=0, cursor=0x3000), dict(streams=1, table_stride=0), dict(table_stride=-10, cursor=0x3000 + 4 * 8), dict(table_stride=-10, cursor=0x3000 - 4 * 31)])
def test_layouts_whose_parts_lie_side_by_side_pass_the_checks(good):
    args = layout_args(**{**dict(workspace=0x100000, workspace_bytes=1 << 12), **good})
    assert _native.load().ll_step_layout(ctypes.byref(args), None) == -2   # as far as the launch


def test_memory_that_calls_ask_for():
    lib, n = _native.load(), ctypes.c_size_t()
    for tokens, out, cursor, want in ((100, 8, 0, 0), (1 << 20, 8, 0, 0), (1 << 20, 16, 0, 44), (1 << 20, 8, 4, 44), (100, 16, 4, 0)):   # lengths at 16
        a = _native.StepLayoutStruct(streams=10, page_size=16, table_width=3, tokens=tokens, kv_lens=16, kv_lens_out=out, cursor=cursor or None)
        assert lib.ll_step_layout_workspace(ctypes.byref(a), ctypes.byref(n)) == 0 and n.value == want
    assert shared_bytes(shared_args(own=dict(n_queries=0))) == 0 and shared_bytes(shared_args(own=dict(streams=0))) == 0
    # results of parts for every row, whole records of fp32 columns, reference point and sum
    some = shared_bytes(shared_args(own=dict(n_queries=64, streams=64, num_heads=32, num_kv_heads=8, max_q_len=1, max_kv_len=64), prefix_width=1024))
    assert some // (64 * 32 * 130 * 4) > 1
    # several long chunks, each of which fills tiles by itself, go over the beginning one by one, as over keys of one table
    chunks = dict(n_queries=10560, streams=4, num_heads=24, num_kv_heads=24, max_q_len=2640, page_size=880)
    one = shared_args(own=dict(**chunks, table_width=15, max_kv_len=13200, causal=0)).own
    assert lib.ll_ragged_attention_workspace(ctypes.byref(one), 256, ctypes.byref(n)) == 0
    assert shared_bytes(shared_args(own=dict(**chunks, table_width=3, max_kv_len=2640), prefix_width=12, max_prefix_len=10560)) == n.value
    # streams without new tokens take no more than where they are listed
    few, many = (shared_bytes(shared_args(own=dict(n_queries=64, streams=n, num_heads=32, num_kv_heads=8, max_q_len=1, max_kv_len=64), prefix_width=1024))
                 for n in (64, 1 << 20))
    assert few < many <= few + 12 * (1 << 20)
