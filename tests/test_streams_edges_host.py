"""CPU tests of the operators for several streams at the ends of what they take: divisions of launches, and calls that are refused or taken."""
import ctypes
import os

import pytest
import torch

from longlive_amd import _native
from longlive_amd.utils.cross_attention import ragged_cross_attention
from longlive_amd.utils.paged_kv import initialize_paged_kv_cache, paged_attention


@pytest.fixture(scope="module")
def hooks():
    lib = ctypes.CDLL(os.path.join(os.path.dirname(_native.LIB_PATH), "libll_nvfp4_testhooks.so"))
    lib.ll_test_head_norm_tokens.restype, lib.ll_test_head_norm_tokens.argtypes = ctypes.c_int64, [ctypes.c_uint32]
    lib.ll_test_head_norm_threads.restype, lib.ll_test_head_norm_threads.argtypes = ctypes.c_int64, [ctypes.c_int64, ctypes.c_uint32]
    return lib


@pytest.mark.parametrize("per_token", [1, 2, 3, 7, 100, 4097, 3 * 32768])   # 65536 heads of 256 columns each take as many as the last
def test_launches_of_head_norms_stay_within_the_grid(hooks, per_token):
    most = hooks.ll_test_head_norm_tokens(per_token)
    assert most >= 1
    for tokens in (1, most - 1, most):
        threads = hooks.ll_test_head_norm_threads(tokens, per_token)
        assert 64 * tokens * per_token <= threads < 64 * tokens * per_token + 256
        assert threads < 1 << 32   # what HIP takes


def need(**kw):
    """Bytes of workspace that a launch asks for on 256 compute units."""
    a = _native.RaggedAttentionStruct(**{**dict(dtype=0, head_dim=128, num_heads=4, num_kv_heads=4, softmax_scale=0.1), **kw})
    n = ctypes.c_size_t()
    assert _native.load().ll_ragged_attention_workspace(ctypes.byref(a), 256, ctypes.byref(n)) == 0
    return n.value


def test_a_window_without_causal_order_reaches_to_the_last_key():
    """2640 tokens over 13200 keys, window 64: a causal tile sees some 260 keys, one part; without causal order the first tile sees 2703."""
    chunk = dict(streams=1, n_queries=2640, max_q_len=2640, max_kv_len=13200, page_size=880, table_width=15, n_pages=15, window=64)
    assert need(**chunk, causal=1) == 0
    assert need(**chunk, causal=0) > 0
    assert need(**{**chunk, "n_queries": 20, "max_q_len": 20}, causal=0) == 0


def taken(new, keys, heads, kv_heads, D):
    """Records of a kv head that the wide tiles of each of several causal streams would take where the device forms the size of a part from
    their lengths (up to 64 streams that are not alike, in a cache with room to spare)."""
    group, share = heads // kv_heads, 0.9 * kv_heads / (256 * (3 if D == 64 else 2))
    tiles, steps = [-(-n * group // 128) for n in new], [-(-m // 64) for m in keys]
    part = max(int(sum(t * max(s - n // 128, 1) for t, s, n in zip(tiles, steps, new)) * share), 10)
    return [t * -(-s // part) * 4 if s > part else 0 for t, s in zip(tiles, steps)]


@pytest.mark.parametrize("new,keys,heads,kv_heads,D,found", [
    ([2000, 2000], [2000, 2000], 8, 2, 128, [True, False]), ([4000, 300], [4000, 300], 16, 4, 64, [False]), ([1500, 1900, 700], [1500, 1900, 700], 8, 2, 128, [True] * 3),
    ([600, 2000, 50, 900], [700, 2000, 3000, 2100], 16, 4, 128, [True, True, False])])
def test_which_streams_find_records(new, keys, heads, kv_heads, D, found):
    """Of the streams that are to be cut, in order, those that find records for all their parts: what the GPU test of streams that find none rests on."""
    records = need(head_dim=D, num_heads=heads, num_kv_heads=kv_heads, streams=len(new), n_queries=sum(new), max_q_len=max(new), max_kv_len=max(keys), page_size=16,
                   table_width=-(-max(keys) // 16), n_pages=4096, causal=1) // (kv_heads * 32 * (D + 2) * 4)
    want = taken(new, keys, heads, kv_heads, D)
    assert [sum(want[:i + 1]) <= records for i, w in enumerate(want) if w] == found


class OnGpu(torch.Tensor):
    """A tensor that says it is on the GPU, so that calls take the way that they take there."""
    is_cuda = True


@pytest.fixture
def no_gpu_needed(monkeypatch):
    """The checks of the Python layer with the check of the device taken out, a native host path that takes nothing, and a library that must
    not be reached."""
    monkeypatch.setattr(_native, "_require_cuda", lambda *t: None)
    monkeypatch.setattr(_native, "host", lambda: _native._NoHostPath())
    monkeypatch.setattr(_native, "load", lambda: pytest.fail("the call was not refused"))


@pytest.mark.parametrize("shape", [(), (64,), (3, 4, 0), (3, 0, 0), (3, 4, 64, 1)])
def test_queries_without_columns_or_dimensions_are_refused(no_gpu_needed, shape):
    q, i32 = torch.zeros(shape, dtype=torch.bfloat16).as_subclass(OnGpu), lambda *s: torch.zeros(s, dtype=torch.int32)
    cache = initialize_paged_kv_cache(1, 4, 16, 2, 64, "cpu")[0]
    k = torch.zeros(9, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        paged_attention(q, cache, i32(2, 5), i32(2), i32(3))
    with pytest.raises(ValueError):
        ragged_cross_attention(q, k, k, i32(3), i32(3))


def test_a_page_table_of_one_column_may_have_any_stride(no_gpu_needed, monkeypatch):
    class Reached(Exception):
        pass

    def load():
        raise Reached

    q, i32 = torch.zeros(3, 4, 64, dtype=torch.bfloat16), lambda *s: torch.zeros(s, dtype=torch.int32)
    cache = initialize_paged_kv_cache(1, 4, 16, 2, 64, "cpu")[0]
    for bad in (i32(5, 2).T, i32(2, 1).expand(2, 5)):
        with pytest.raises(ValueError, match="page_table"):
            paged_attention(q, cache, bad, i32(2), i32(3))
    monkeypatch.setattr(_native, "load", load)
    monkeypatch.setattr(torch.cuda, "device", lambda d: torch.no_grad())
    for good in (i32(2, 1), i32(2, 5, 3)[:, 2:3, 1], i32(2, 5)):
        with pytest.raises(Reached):
            paged_attention(q, cache, good, i32(2), i32(3))
