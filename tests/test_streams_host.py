"""CPU tests of the operators for several streams in one batch: what they refuse before any launch, where new tokens go, and the plain
64-bit forms that the GPU tests compare with."""
import ctypes
import math

import pytest
import torch

import streams_reference as ref
from longlive_amd import _native
from longlive_amd.utils.cross_attention import ragged_cross_attention
from longlive_amd.utils.paged_kv import head_norm_rope_paged, initialize_paged_kv_cache, paged_attention, paged_slots
from longlive_amd.utils.rope import head_norm_rope

BF16 = torch.bfloat16


def test_slots_of_new_tokens():
    table = torch.tensor([[3, 1, -1], [0, 2, 4], [5, 6, 7]], dtype=torch.int32)
    lens, q_starts = torch.tensor([5, 11, 30], dtype=torch.int32), torch.tensor([1, 3, 3, 6], dtype=torch.int32)
    # rows outside; keys 3 and 4 of the first stream; none of the second; keys 27..29 of the third, behind its table of 12
    assert paged_slots(table, lens, q_starts, 8, 4).tolist() == [-1, 15, 4, -1, -1, -1, -1, -1]
    lens[2] = 10
    assert paged_slots(table, lens, q_starts, 8, 4).tolist() == [-1, 15, 4, 27, 28, 29, -1, -1]
    lens[0], lens[2] = 10, 1       # a hole; places before the stream's beginning
    assert paged_slots(table, lens, q_starts, 8, 4).tolist() == [-1, -1, -1, -1, -1, 20, -1, -1]
    assert paged_slots(table[:0], lens[:0], q_starts[:1], 2, 4).tolist() == [-1, -1]
    assert paged_slots(table[:, :0], lens, q_starts, 2, 4).tolist() == [-1, -1]
    for bad in ((table[0], lens, q_starts, 8, 4), (table, lens[:2], q_starts, 8, 4), (table, lens, q_starts[:3], 8, 4), (table, lens, q_starts, 8, 0)):
        with pytest.raises(ValueError):
            paged_slots(*bad)


def test_plain_forms_on_a_case_by_hand():
    q, k, v = torch.tensor([[1.0, 0.0]]).to(BF16), torch.tensor([[0.0, 1.0], [2.0, 0.0], [9.0, 9.0]]).to(BF16), torch.tensor([[1.0], [3.0], [100.0]]).to(BF16)
    out, error = ref.attend(q, k, v, torch.tensor([[True, True, False]]), 0.5)
    assert out.item() == pytest.approx((1.0 + 3.0 * math.e) / (1.0 + math.e)) and 0 < error.item() < 0.05
    out, _ = ref.attend(q, k, v, torch.zeros(1, 3, dtype=torch.bool), 0.5)
    assert out.item() == 0.0
    x = torch.tensor([[[3.0, 4.0, 0.0, 0.0]]]).to(BF16)
    c, s = torch.tensor([[0.0, 1.0]]), torch.tensor([[1.0, 0.0]])
    y, _ = ref.head_norm_rope(x, None, 0.0, c, s, None, True)
    assert y.flatten().tolist() == [-4.0, 3.0, 0.0, 0.0]
    y, _ = ref.head_norm_rope(x, torch.full((4,), 2.0), 0.0, c, s, None, False)
    assert y.flatten().tolist() == pytest.approx([0.0, 3.2, 2.4, 0.0])


def test_operators_run_on_the_gpu_only():
    x, i = torch.zeros(3, 2, 64, dtype=BF16), torch.zeros(2, dtype=torch.int32)
    cache = initialize_paged_kv_cache(2, 4, 16, 2, 64, "cpu")
    assert len(cache) == 2 and cache[0]["k_pages"].shape == (4, 16, 2, 64)
    with pytest.raises(ValueError, match="GPU"):
        head_norm_rope(x, x, None, None, 1e-6, None, None)
    with pytest.raises(ValueError, match="GPU"):
        paged_attention(x, cache[0], i[:1, None], i[:1], i)
    with pytest.raises(ValueError, match="GPU"):
        ragged_cross_attention(x, x, x, i, i)


@pytest.mark.parametrize("kwargs", [dict(dtype=torch.float32), dict(head_dim=96), dict(page_size=0), dict(num_kv_heads=0), dict(num_pages=-1)])
def test_caches_that_cannot_be(kwargs):
    with pytest.raises(ValueError):
        initialize_paged_kv_cache(**{**dict(num_layers=1, num_pages=4, page_size=16, num_kv_heads=2, head_dim=64, device="cpu"), **kwargs})


@pytest.fixture
def no_gpu_needed(monkeypatch):
    """The checks of the Python layer with the check of the device taken out, and a library that must not be reached."""
    monkeypatch.setattr(_native, "_require_cuda", lambda *t: None)
    monkeypatch.setattr(_native, "load", lambda: pytest.fail("the call was not refused"))


def test_refusals_of_head_norm_rope(no_gpu_needed):
    x, w = torch.zeros(3, 2, 64, dtype=BF16), torch.zeros(64, dtype=BF16)
    cos = torch.zeros(5, 32)
    cache = initialize_paged_kv_cache(1, 4, 16, 2, 64, "cpu")[0]
    slots = torch.zeros(3, dtype=torch.int64)
    ok = dict(q=x, k=x, q_weight=w, k_weight=w, eps=1e-6, cos_f32=cos, sin_f32=cos, positions=slots)
    for bad in (dict(q=x.float()), dict(q=x[0]), dict(k=x.half()), dict(k=x[:2]), dict(k=x[..., :56]), dict(q_weight=w[:8]), dict(q_weight=w.half()),
                dict(k_weight=w.double()), dict(sin_f32=None), dict(cos_f32=cos.double()), dict(sin_f32=cos[:4]), dict(cos_f32=cos[:, :30], sin_f32=cos[:, :30]),
                dict(cos_f32=torch.zeros(5, 36), sin_f32=torch.zeros(5, 36)), dict(positions=slots.int()), dict(positions=slots[:2]),
                dict(q=x[..., :12], k=x[..., :12]), dict(q=torch.zeros(3, 2, 264, dtype=BF16), k=torch.zeros(3, 2, 264, dtype=BF16))):
        with pytest.raises(ValueError):
            head_norm_rope(**{**ok, **bad})
    ok.update(v=x, cache=cache, slots=slots)
    half = {n: t.half() for n, t in cache.items()}
    apart = {n: torch.zeros(4, 17, 2, 64, dtype=BF16)[:, :16] for n in cache}
    for bad in (dict(v=x[:, :1]), dict(v=x.half()), dict(slots=slots[:2]), dict(slots=slots.int()), dict(cache=half), dict(cache=apart), dict(out=x.half()),
                dict(out=x[:2]), dict(cache={"k_pages": cache["k_pages"], "v_pages": cache["v_pages"][:2]}),
                dict(cache=initialize_paged_kv_cache(1, 4, 16, 3, 64, "cpu")[0])):
        with pytest.raises(ValueError):
            head_norm_rope_paged(**{**ok, **bad})


def test_refusals_of_paged_attention(no_gpu_needed):
    q, i32 = torch.zeros(3, 4, 64, dtype=BF16), lambda *s: torch.zeros(s, dtype=torch.int32)
    cache = initialize_paged_kv_cache(1, 4, 16, 2, 64, "cpu")[0]
    ok = dict(q=q, cache=cache, page_table=i32(2, 5), kv_lens=i32(2), q_starts=i32(3))
    three = initialize_paged_kv_cache(1, 4, 16, 3, 64, "cpu")[0]
    rows = {n: torch.zeros(4, 16, 2, 65, dtype=BF16)[..., :64] for n in cache}
    for bad in (dict(q=q.float()), dict(q=q.half()), dict(q=q[0]), dict(q=torch.zeros(3, 4, 96, dtype=BF16)), dict(q=torch.zeros(3, 4, 128, dtype=BF16)),
                dict(cache=three), dict(cache=rows), dict(page_table=i32(2, 5).long()), dict(page_table=i32(3, 5)), dict(page_table=i32(10)),
                dict(page_table=i32(5, 2).T), dict(page_table=i32(2, 1 << 27)), dict(kv_lens=i32(3)), dict(kv_lens=i32(2).long()), dict(q_starts=i32(2)),
                dict(q_starts=i32(3).long()), dict(q_starts=i32(0)), dict(window=0), dict(window=-3), dict(sink_tokens=-1), dict(softmax_scale=0.0),
                dict(softmax_scale=-1.0), dict(softmax_scale=float("nan")), dict(softmax_scale=float("inf")), dict(max_q_len=-1), dict(max_kv_len=-1),
                dict(out=q.half()), dict(out=q[:2]), dict(out=torch.zeros(3, 64, 4, dtype=BF16).transpose(1, 2))):
        with pytest.raises(ValueError):
            paged_attention(**{**ok, **bad})


def test_refusals_of_cross_attention(no_gpu_needed):
    q, k, i32 = torch.zeros(3, 4, 64, dtype=BF16), torch.zeros(9, 2, 64, dtype=BF16), lambda *s: torch.zeros(s, dtype=torch.int32)
    ok = dict(q=q, k=k, v=k, q_starts=i32(3), k_starts=i32(3))
    for bad in (dict(k=k.half()), dict(v=k[:8]), dict(k=k[:, :, :32], v=k[:, :, :32]), dict(k=torch.zeros(9, 3, 64, dtype=BF16), v=torch.zeros(9, 3, 64, dtype=BF16)),
                dict(k_starts=i32(2)), dict(k_starts=i32(3).long()), dict(k_lens=i32(3)), dict(k_lens=i32(2), k_starts=i32(1)), dict(k_lens=i32(2).long()),
                dict(key_mask=torch.ones(9)), dict(key_mask=torch.ones(8, dtype=torch.bool)), dict(q_starts=i32(0))):
        with pytest.raises(ValueError):
            ragged_cross_attention(**{**ok, **bad})


def test_outputs_whose_elements_share_a_place_are_refused(no_gpu_needed):
    x, i32 = torch.zeros(3, 4, 64, dtype=BF16), lambda *s: torch.zeros(s, dtype=torch.int32)
    cache = initialize_paged_kv_cache(1, 4, 16, 4, 64, "cpu")[0]
    slots = torch.zeros(3, dtype=torch.int64)
    row = torch.zeros(64, dtype=BF16)
    for out in (row.expand(3, 4, 64), torch.zeros(3, 1, 64, dtype=BF16).expand(3, 4, 64), torch.zeros(500, dtype=BF16).as_strided((3, 4, 64), (64, 64, 1))):
        with pytest.raises(ValueError, match="place of its own"):
            paged_attention(x, cache, i32(2, 5), i32(2), i32(3), out=out)
        with pytest.raises(ValueError, match="place of its own"):
            ragged_cross_attention(x, x, x, i32(3), i32(3), out=out)
        with pytest.raises(ValueError, match="place of its own"):
            head_norm_rope_paged(x, x, x, cache, slots, None, None, 1e-6, None, None, out=out)
    for pages in (row.expand(4, 16, 4, 64), torch.zeros(64, 1, 64, dtype=BF16).expand(64, 4, 64).unflatten(0, (4, 16))):
        with pytest.raises(ValueError, match="place of its own"):
            head_norm_rope_paged(x, x, x, {**cache, "v_pages": pages}, slots, None, None, 1e-6, None, None)


def test_c_abi_refuses_bad_arguments_before_touching_the_gpu():
    lib, need = _native.load(), ctypes.c_size_t()
    ok = dict(dtype=0, head_dim=64, num_heads=4, num_kv_heads=2, n_queries=3, streams=2, softmax_scale=0.125, page_size=16, table_width=5, n_pages=4)
    for bad, says in ((dict(dtype=2), b"dtype"), (dict(head_dim=80), b"head_dim"), (dict(num_kv_heads=3), b"kv heads"), (dict(num_kv_heads=0), b"kv heads"),
                      (dict(n_queries=-1), b"queries"), (dict(n_queries=1 << 30), b"2^31"), (dict(streams=1 << 40), b"streams"), (dict(softmax_scale=0.0), b"softmax_scale"),
                      (dict(softmax_scale=float("inf")), b"softmax_scale"), (dict(table_width=1 << 40), b"2^31"), (dict(window=-1), b"window"),
                      (dict(page_size=0, causal=1), b"paged"), (dict(page_size=0, window=3), b"paged"), (dict(page_size=0, n_keys=-2), b"keys"),
                      (dict(max_q_len=-1), b"longest")):
        a = _native.RaggedAttentionStruct(**{**ok, **bad})
        assert lib.ll_ragged_attention_workspace(ctypes.byref(a), 256, ctypes.byref(need)) == -1 and says in lib.ll_last_error(), bad
        assert lib.ll_ragged_attention(ctypes.byref(a), None) == -1
    assert lib.ll_ragged_attention(None, None) == -1
    a = _native.RaggedAttentionStruct(**ok)
    assert lib.ll_ragged_attention_workspace(ctypes.byref(a), 256, ctypes.byref(need)) == 0
    assert lib.ll_ragged_attention(ctypes.byref(a), None) == -1 and b"null" in lib.ll_last_error()
    fields = dict(q=4096, out=8192, q_starts=64, kv_lens=64, page_table=64, k=4096, v=4096)
    for bad, says in ((dict(q=4098), b"16-byte"), (dict(v=4104), b"16-byte"), (dict(k_stride_row=4), b"multiples"), (dict(q_starts=0), b"null"), (dict(kv_lens=0), b"null"),
                      (dict(k=0), b"null")):
        a = _native.RaggedAttentionStruct(**{**ok, **fields, **bad})
        assert lib.ll_ragged_attention(ctypes.byref(a), None) == -1 and says in lib.ll_last_error(), bad
    a = _native.RaggedAttentionStruct(**{**ok, "n_queries": 0})
    assert lib.ll_ragged_attention(ctypes.byref(a), None) == 0

    row = lambda **kw: ctypes.byref(_native.HeadRowsStruct(**{**dict(x=4096, stride_token=128, stride_head=64, num_heads=2, out=8192, out_stride_token=128,  # noqa: E731
                                                                     out_stride_head=64), **kw}))
    def call(dtype=0, tokens=3, D=64, q=None, k=None, v=None, cos=4096, sin=4096, rows=5, R=64, slots=None, n_slots=0):
        return lib.ll_head_norm_rope(dtype, tokens, D, q or row(), k or row(), v, 1e-6, cos, sin, rows, R, None, 1, slots, n_slots, None)
    for bad, says in ((dict(dtype=2), b"dtype"), (dict(tokens=-1), b"tokens"), (dict(D=60), b"head_dim"), (dict(D=264), b"head_dim"), (dict(R=128), b"rotary_dim"),
                      (dict(R=12), b"rotary_dim"), (dict(cos=None), b"angles"), (dict(sin=4100), b"16-byte"), (dict(q=row(x=4098)), b"16-byte"),
                      (dict(q=row(stride_head=4)), b"multiples"), (dict(q=row(num_heads=-1)), b"heads"), (dict(k=row(out=None)), b"null"),
                      (dict(v=row()), b"slots"), (dict(v=row(weight=4096), slots=64), b"no norm"), (dict(v=row(num_heads=1), slots=64), b"as many heads"),
                      (dict(slots=64, n_slots=-1), b"slots")):
        assert call(**bad) == -1 and says in lib.ll_last_error(), bad
    assert call(tokens=0) == 0
    none = row(num_heads=0)
    assert call(q=none, k=none) == 0


def test_memory_that_launches_ask_for():
    lib = _native.load()

    def need(cus=256, **kw):
        a = _native.RaggedAttentionStruct(**{**dict(dtype=0, head_dim=128, num_heads=32, num_kv_heads=8, n_queries=32, streams=32, softmax_scale=0.1, page_size=16,
                                                    table_width=1024, n_pages=32768, max_q_len=1, max_kv_len=16384), **kw})
        n = ctypes.c_size_t()
        assert lib.ll_ragged_attention_workspace(ctypes.byref(a), cus, ctypes.byref(n)) == 0
        return n.value

    assert need(n_queries=0) == need(streams=0) == 0
    assert need(max_kv_len=300) == 0                       # one part
    assert 0 < need() <= 256 << 20                         # single tokens over long caches: parts
    assert need(n_queries=65536, streams=16, max_q_len=8192) <= 256 << 20
    assert need(streams=1, n_queries=2640, max_q_len=2640, num_heads=24, num_kv_heads=24, max_kv_len=13200, page_size=880, table_width=15) == 0
    assert need(streams=1, n_queries=1, num_heads=8) > 0   # one stream's token: its keys over the whole device
    assert need(max_kv_len=640) == need(max_kv_len=1024) == 0    # a second launch would cost more than it saves
    most = 0x7fffffff                                            # sizes at the ends of their ranges
    for kw in (dict(n_pages=most, page_size=most, table_width=1), dict(n_pages=most, page_size=most, table_width=1, n_queries=1 << 25, max_q_len=0, max_kv_len=0),
               dict(streams=0xfffffff // 8, n_queries=1 << 25, page_size=1, table_width=most, n_pages=most, max_q_len=0, max_kv_len=0),
               dict(page_size=0, n_keys=most, max_q_len=0, max_kv_len=0, n_queries=1 << 25)):
        assert 0 <= need(**kw) <= 256 << 20
    for cus in (1, 64, 304):
        assert need(cus=cus) <= 256 << 20
