"""float16 keys far below the largest of a row: many of them together count, so each must keep its weight."""
import pytest
import torch

import streams_reference as ref
from longlive_amd.utils.cross_attention import ragged_cross_attention
from longlive_amd.utils.paged_kv import paged_attention
from test_gpu_streams import F16, close, starts

pytestmark = pytest.mark.gpu

BELOW = 17.5   # nats: a weight of 2^-25.2


def attend(q, k, v, seen):
    """(result, allowed error) of :func:`streams_reference.attend` at a scale of 1, with what subnormal probabilities are off by.

    The largest probability of a row is kept at 2^13 or more, so a step of 2^-24 is off by at most 2^-25, 2^-38 of the largest weight, and
    the sum of all weights is no smaller than that one: m 2^-38 max |v| in the numerator, as much relative to the result in the sum."""
    out, _ = ref.attend(q, k, v, seen, 1.0)
    m, most = k.shape[0], v.double().abs().amax(0, keepdim=True)
    s = (q.double() @ k.double().T).masked_fill(~seen, float("-inf"))
    w = torch.softmax(s, dim=-1)
    size = w @ v.double().abs()
    reach = (q.double().abs() @ k.double().abs().T).masked_fill(~seen, 0.0).amax(-1, keepdim=True)
    score, sums, u = (q.shape[-1] + 4) * 2.0 ** -23 * reach + 2.0 ** -20, (m + 64) * 2.0 ** -23, ref.UNIT[F16]
    return out, u * out.abs() + size * (u + 2 * score + 2 * sums) + 2.0 ** -37 * m * most + 2.0 ** -25


def rows(n, m, D, at, seed=1):
    """Queries [n, D], keys [m, D] of which `at` alone has the score BELOW and the others 0, values of which `at`'s is 0 and the others about 1."""
    q, k = torch.zeros(n, D, dtype=F16), torch.zeros(m, D, dtype=F16)
    q[:, 0], k[at, 0] = 1.0, BELOW
    v = (1 + 0.25 * torch.randn(m, D, generator=torch.Generator().manual_seed(seed))).to(F16)
    v[at] = 0.0
    return q, k, v


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("last", [False, True])
@pytest.mark.parametrize("n,m", [(1, 40), (1, 30000), (3, 5000), (90, 700), (150, 6000)])
def test_one_key_above_many(gpu, n, m, last, D):
    q, k, v = rows(n, m, D, 0)
    if last:   # above what was summed up before it; seen by every row
        k, v = (torch.cat([t[1:], t[:1]]) for t in (k, v))
    got = ragged_cross_attention(q[:, None].to(gpu), k[:, None].to(gpu), v[:, None].to(gpu), starts([n]).to(gpu), starts([m]).to(gpu), softmax_scale=1.0)
    want, error = attend(q, k, v, torch.ones(n, m, dtype=torch.bool))
    assert (want > 2 * error).all()   # the many are not lost in the allowed error
    close(got[:, 0], want, error)


@pytest.mark.parametrize("hidden", [False, True])
@pytest.mark.parametrize("n,m", [(1, 4096), (5, 900), (100, 2000)])
def test_the_same_in_pages(gpu, n, m, hidden):
    """Causal; `hidden`: a value that is not finite and is seen by the last token alone has the others computed apart."""
    q, k, v = rows(n, m, 64, 3)
    seen = torch.arange(m) <= (m - n + torch.arange(n))[:, None]
    want, error = attend(q, k, v, seen)
    if hidden:
        v[m - 1] = float("inf")
    pages = {name: torch.zeros(-(-m // 16) * 16, 1, 64, dtype=F16) for name in ("k_pages", "v_pages")}
    pages["k_pages"][:m, 0], pages["v_pages"][:m, 0] = k, v
    table = torch.arange(-(-m // 16), dtype=torch.int32)[None]
    got = paged_attention(q[:, None].to(gpu), {name: t.unflatten(0, (-1, 16)).to(gpu) for name, t in pages.items()}, table.to(gpu),
                          torch.tensor([m], dtype=torch.int32, device=gpu), starts([n]).to(gpu), softmax_scale=1.0)
    cut = slice(0, n - 1 if hidden else n)
    close(got[cut, 0], want[cut], error[cut])
    assert not hidden or got[n - 1].isinf().all()


@pytest.mark.parametrize("n", [2, 80])
@pytest.mark.parametrize("size", [2.0 ** 20, 2.0 ** 22, 2.0 ** 24, 2.0 ** 26])
def test_large_scores(gpu, n, size):
    """Scores so large that their rounding is more than a power of two: the largest alone has a weight, and no probability overflows."""
    m, D = 100, 64
    q, k = torch.zeros(n, D, dtype=F16), torch.zeros(m, D, dtype=F16)
    q[:, 0], k[:, 0] = size ** 0.5, torch.linspace(-1, 1, m) * size ** 0.5
    v = torch.randn(m, D, generator=torch.Generator().manual_seed(2)).to(F16)
    got = ragged_cross_attention(q[:, None].to(gpu), k[:, None].to(gpu), v[:, None].to(gpu), starts([n]).to(gpu), starts([m]).to(gpu), softmax_scale=1.0)
    assert torch.equal(got[:, 0].cpu(), v[m - 1].expand(n, D))
