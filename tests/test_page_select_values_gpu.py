"""GPU: choice of pages where a query channel is -0, against the 64-bit
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
