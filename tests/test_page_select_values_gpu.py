"""GPU: choice of pages where a query channel is -0 and where queries lie below the normal range of 32 bits, against the 64-bit
oracle.  Whole numbers: equal or not."""
import pytest
import torch

from oracle import cache_budget_oracle as R
from test_cache_budget_gpu import BF, HF, fa  # noqa: F401

pytestmark = pytest.mark.gpu


def check(m, q, bounds, pages, k):
    bt, sl = torch.arange(pages, dtype=torch.int32)[None], torch.tensor([pages * 64], dtype=torch.int32)
    got = m.kvcache_select_pages(q.cuda(), bounds.cuda(), bt.cuda(), sl.cuda(), 64, k)
    want = R.select_pages_ref(q, bounds, bt, sl, 64, k)
    for a, b in zip(got, want):
        assert torch.equal(a.cpu(), b)


@pytest.mark.parametrize("dtype,d", [(BF, 128), (HF, 64), (BF, 256)])
def test_a_channel_of_negative_zero_takes_the_largest_value(fa, dtype, d):   # noqa: F811
    m, _ = fa
    g = torch.Generator().manual_seed(51)
    q = torch.randn(1, 1, 4, d, generator=g)
    q[..., 3] = -0.0
    b = torch.randn(60, 2, 2, d, generator=g).sort(2).values
    b[5::7, :, 0, 3] = -float("inf")     # no part of the score: the channel takes the largest value, times -0
    check(m, q.to(dtype), b.to(dtype), 60, 9)


@pytest.mark.parametrize("d,qv,base,step", [
    (128, 2.0 ** -130, 2.0 ** 120, 2.0 ** 90), (256, -2.0 ** -131, -2.0 ** 122, -2.0 ** 92), (64, 2.0 ** -127, 2.0 ** 121, 2.0 ** 91),
    (128, 2.0 ** -131, 2.0 ** 100, 2.0 ** 70)])
def test_queries_below_the_normal_range(fa, d, qv, base, step):   # noqa: F811
    """The same values in another order of the channels for every page, whose 32-bit sums round differently, and one small term
    that decides.  64-bit sums are exact here: up to 2^8 values of 8 bits between 2^-18 and 2^2 times base."""
    m, _ = fa
    pages, g = 48, torch.Generator().manual_seed(52)
    q = torch.full((1, 1, 2, d), qv).to(BF)
    x = torch.exp2(torch.rand(d - 1, generator=g) * 20 - 18).to(BF).float()
    b = torch.zeros(pages, 2, 2, d)
    order = torch.randperm(pages, generator=g)
    for j in range(pages):
        b[j, :, :, :d - 1] = base * x[torch.randperm(d - 1, generator=g)]
    b[..., d - 1] = step * (1 + order % 120)[:, None, None]
    assert len(set(b.to(BF)[:, 0, 0, d - 1].tolist())) == pages
    check(m, q, b.to(BF), pages, 7)
