"""GPU: decode with key weights at sixteen query rows over a long cache: every row of a query tile is real, the sequence is split into
many partitions and a CTA of the second launch takes several chunks of tokens."""
import pytest
import torch

from oracle import cache_budget_oracle as R
from _util import gen
from test_cache_budget_gpu import BF, F8, HF, check_out, fa, pools, score_error   # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("qt,kv,d,group,sq,page,window", [(BF, BF, 128, 4, 4, 64, -1), (HF, F8, 128, 16, 1, 256, -1), (BF, BF, 64, 2, 8, 16, 9000)])
def test_sixteen_rows_over_a_long_cache(fa, qt, kv, d, group, sq, page, window):   # noqa: F811
    m, cuda = fa
    g = gen(71)
    lens, h_k = [40003, 16385], 2
    kc, vc, bt, sl, kd, vd = pools(g, lens, h_k, page, kv, d)
    q = torch.randn(2, sq, group * h_k, d, generator=g).to(qt)
    w = torch.rand(2, h_k, bt.shape[1] * page, generator=g)
    out, lse, got = m.flash_attn_with_kvcache_weights(q.cuda(), kd, vd, sl.cuda(), bt.cuda(), w.cuda(), causal=True, window_size=(window, -1),
                                                      return_softmax_lse=True)
    ref, ref_lse, rw = R.decode_ref(q, kc, vc, bt, sl, d ** -0.5, True, window)
    check_out(out, ref, float(torch.nan_to_num(vc.float()).abs().amax()), "out")
    tol = score_error(q, kc, d ** -0.5) + 2.0 ** -20
    assert (lse.cpu().double() - ref_lse).abs().max() <= tol * ref_lse.abs().clamp(min=1).max()
    for i, n in enumerate(lens):
        for x in range(h_k):
            want = w[i, x, :n].double() + rw[i][x]
            assert ((got[i, x, :n].cpu().double() - want).abs() <= (2 * tol + 2.0 ** -20) * want).all()
        assert torch.equal(got[i, :, n:].cpu(), w[i, :, n:])
    assert cuda.device_status() == 0
