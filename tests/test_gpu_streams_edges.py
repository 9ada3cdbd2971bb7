"""The operators for several streams on the GPU at sizes and arguments at the ends of what they take."""
import pytest
import torch

from longlive_amd.utils.paged_kv import head_norm_rope_paged
from test_gpu_streams import BF16, angles

pytestmark = pytest.mark.gpu


def test_head_norms_of_more_tokens_than_a_launch_takes(gpu):
    """Three waves a token, of which a launch takes 2^25: two launches, the second with tokens, positions and slots of its own."""
    T, D, page = (1 << 24) + 1000, 8, 16
    g = torch.Generator(device=gpu).manual_seed(1)
    q, k, v = (torch.randn(T, 1, D, generator=g, device=gpu, dtype=BF16) for _ in range(3))
    w = torch.rand(D, generator=g, device=gpu).to(BF16)
    cos, sin = (t.to(gpu) for t in angles(1000, D))
    positions = torch.randint(0, 1000, (T,), generator=g, device=gpu)
    slots = torch.randperm(T + 24, generator=g, device=gpu)[:T]
    whole, pieces = ({n: torch.zeros((T + 24) // page, page, 1, D, dtype=BF16, device=gpu) for n in ("k_pages", "v_pages")} for _ in range(2))
    got = head_norm_rope_paged(q, k, v, whole, slots, w, w, 1e-6, cos, sin, positions)
    each = 1 << 20
    want = torch.cat([head_norm_rope_paged(*(t[i:i + each] for t in (q, k, v)), pieces, slots[i:i + each], w, w, 1e-6, cos, sin, positions[i:i + each])
                      for i in range(0, T, each)])
    assert torch.equal(got, want)
    for n in whole:
        assert torch.equal(whole[n], pieces[n])
    assert (whole["v_pages"].flatten(0, 1)[slots[-1000:]] == v[-1000:]).all()
