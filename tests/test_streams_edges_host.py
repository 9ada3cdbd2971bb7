"""CPU tests of the operators for several streams at the ends of what they take: divisions of launches, and calls that are refused or taken."""
import ctypes
import os

import pytest
import torch

from longlive_amd import _native


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
