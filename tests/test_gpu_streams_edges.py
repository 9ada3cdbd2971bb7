"""The operators for several streams on the GPU at sizes and arguments at the ends of what they take."""
import pytest
import torch

import streams_reference as ref
from longlive_amd.utils.cross_attention import ragged_cross_attention
from longlive_amd.utils.paged_kv import head_norm_rope_paged, paged_attention
from test_gpu_streams import BF16, F16, angles, batch, close, starts

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


@pytest.mark.parametrize("new,keys,Hq,Hk,D,dtype", [([2000, 2000], [2000, 2000], 8, 2, 128, BF16), ([4000, 300], [4000, 300], 16, 4, 64, F16),
                                                    ([600, 2000, 50, 900], [700, 2000, 3000, 2100], 16, 4, 128, BF16)])
def test_prompts_of_which_some_find_no_records_left(gpu, new, keys, Hq, Hk, D, dtype):
    """Causal prompts in a cache of 4096 pages, cut by the device: the first streams are cut, the last ones stay whole for want of records (or the
    only one to be cut does)."""
    q, cache, table, lens, q_starts = batch(211, new, keys, Hq, Hk, D, 16, dtype)
    held = cache["k_pages"].shape[0]
    dev = {n: torch.cat([t, torch.full((4096 - held, *t.shape[1:]), float("nan"), dtype=dtype)]).to(gpu) for n, t in cache.items()}
    table = table[:, :-(-max(keys) // 16)].contiguous()
    got = paged_attention(q.to(gpu), dev, table.to(gpu), lens.to(gpu), q_starts.to(gpu), max_q_len=max(new), max_kv_len=max(keys)).cpu()
    keys_of, _ = ref.paged_keys(cache, table, lens)
    for b, (n, m) in enumerate(zip(new, keys)):
        k, v = keys_of(b)
        at = torch.cat([torch.arange(0, n, 97), torch.tensor([n - 1])])
        seen = torch.arange(m) <= (m - n + at)[:, None]
        for h in (0, Hq - 1):
            want, error = ref.attend(q[int(q_starts[b]) + at, h], k[:, h * Hk // Hq], v[:, h * Hk // Hq], seen, D ** -0.5)
            close(got[int(q_starts[b]) + at, h], want, error, f"stream {b} head {h}")


@pytest.mark.parametrize("native", [True, False])
def test_a_page_table_of_one_column_with_any_stride(gpu, native, monkeypatch):
    from longlive_amd import _native

    if not native:
        monkeypatch.setattr(_native, "_host", _native._NoHostPath())
    q, cache, table, lens, q_starts = batch(221, [3, 1], [14, 16], 4, 2, 64, 16, BF16)
    cache = {n: t.to(gpu) for n, t in cache.items()}
    rest = (lens.to(gpu), q_starts.to(gpu))
    want = paged_attention(q.to(gpu), cache, table[:, :1].contiguous().to(gpu), *rest)
    wide = torch.full((2, 5, 3), 1 << 30, dtype=torch.int32)
    wide[:, 2, 1] = table[:, 0]
    wide = wide.to(gpu)[:, 2:3, 1]
    assert wide.shape == (2, 1) and wide.stride() == (15, 3)
    assert torch.equal(paged_attention(q.to(gpu), cache, wide, *rest), want)
    for bad in (table[:, :1].to(gpu).expand(2, 2), table[:, :2].to(gpu).T):   # columns that are taken lie one behind the other
        with pytest.raises(ValueError, match="page_table"):
            paged_attention(q.to(gpu), cache, bad, *rest)


@pytest.mark.parametrize("n", [2, 80])
@pytest.mark.parametrize("dtype,size", [(F16, 2.0 ** 27), (BF16, 2.0 ** 27), (BF16, 2.0 ** 30)])
def test_scores_as_large_as_may_be(gpu, dtype, size, n):
    """Scores whose steps are many powers of two, of both signs: the largest alone has a weight."""
    m, D = 100, 64
    q, k = torch.zeros(n, D, dtype=dtype), torch.zeros(m, D, dtype=dtype)
    q[:, 0], k[:, 0] = size ** 0.5 * 0.999, torch.linspace(-1, 0.9, m) * size ** 0.5
    v = torch.randn(m, D, generator=torch.Generator().manual_seed(2)).to(dtype)
    for sign in (1, -1):
        got = ragged_cross_attention(sign * q[:, None].to(gpu), k[:, None].to(gpu), v[:, None].to(gpu), starts([n]).to(gpu), starts([m]).to(gpu), softmax_scale=1.0)
        assert torch.equal(got[:, 0].cpu(), v[m - 1 if sign > 0 else 0].expand(n, D))


@pytest.mark.parametrize("n", [2, 80])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_rows_whose_scores_are_all_minus_infinity_are_zeros(gpu, dtype, n):
    m, D = 300, 64
    q, k = torch.zeros(n, 1, D, dtype=dtype), torch.zeros(m, 1, D, dtype=dtype)
    q[:, 0, 0], k[:, 0, 0] = 1.0, -float("inf")
    v = torch.ones(m, 1, D, dtype=dtype)
    got = ragged_cross_attention(q.to(gpu), k.to(gpu), v.to(gpu), starts([n]).to(gpu), starts([m]).to(gpu))
    assert (got == 0).all()
    k[m - 1] = 0.0   # one key that counts
    got = ragged_cross_attention(q.to(gpu), k.to(gpu), v.to(gpu), starts([n]).to(gpu), starts([m]).to(gpu))
    assert (got == 1).all()
