"""GPU: key weights of long causal prompts above d = 128, where the query tiles of a key tile are split into shares and some
shares hold no tile that sees the second 128 keys of their item."""
import ctypes

import pytest
import torch

from oracle import cache_budget_oracle as R
from _util import gen
from test_cache_budget_gpu import BF, HF, fa, pools, score_error  # noqa: F401

pytestmark = pytest.mark.gpu


def shares(cuda, h, h_k, d, page, blocks, max_q):
    p = cuda.TokenWeightsParams()
    p.b, p.max_seqlen_q, p.total_q, p.h, p.h_k, p.d, p.page_size = 1, max_q, max_q, h, h_k, d, page
    p.num_blocks = p.max_blocks_per_seq = blocks
    p.dtype = 1
    return cuda.lib().fa_b200_token_weights_workspace_bytes(ctypes.byref(p)) // (4 * h_k * blocks * page)


@pytest.mark.parametrize("dtype,d,h,h_k,page,n,queries", [
    (BF, 256, 4, 1, 64, 2048, 2048), (HF, 192, 4, 1, 128, 2048, 2048), (BF, 192, 2, 2, 64, 4096, 4096),
    (HF, 256, 2, 2, 16, 4096, 3000), (BF, 256, 8, 1, 64, 2304, 2048)])
def test_shares_that_do_not_see_the_second_keys(fa, dtype, d, h, h_k, page, n, queries):   # noqa: F811
    m, cuda = fa
    g = gen(31)
    kc, _, bt, sl, kd, _ = pools(g, [n], h_k, page, dtype, d, poison=False)
    group = h // h_k
    tt, c = 128 // group, shares(cuda, h, h_k, d, page, bt.shape[1], queries)
    tiles, first = -(-queries // tt), (n - 256 - (n - queries)) // tt    # query tiles that see the last item's keys
    assert c > 1 and any(first + x < tiles and (first + x + (tiles - 1 - first - x) // c * c) * tt + tt <= queries - 128 for x in range(c))
    q = torch.randn(queries, h, d, generator=g).to(dtype)
    lse = torch.empty(h, queries)
    for x in range(h_k):
        keys = R.rows(kc, bt[0], x, n)
        for y in range(x * group, (x + 1) * group):
            lse[y] = R.attention_ref(q[:, y:y + 1].double(), keys, keys[:, :1], d ** -0.5, True)[1][0].float()
    cap = bt.shape[1] * page
    w = torch.rand(1, h_k, cap, generator=g)
    cu = torch.tensor([0, queries], dtype=torch.int32)
    ref = R.token_weights_ref(q, kc, lse, cu, bt, sl, w, d ** -0.5)
    tol = score_error(q, kc, d ** -0.5) + 2.0 ** -19
    for _ in range(3):
        got = m.attn_token_weights(q.cuda(), kd, lse.cuda(), cu.cuda(), queries, sl.cuda(), bt.cuda(), w.cuda())
        assert ((got.cpu().double() - ref).abs() <= tol * ref.abs()).all()
    assert cuda.device_status() == 0
