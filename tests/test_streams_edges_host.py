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
