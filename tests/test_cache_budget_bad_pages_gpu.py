"""GPU: page ids that are no pages, in the calls that attend to keys or weigh them.  Their keys are left out, as if the sequence
did not have them, and device_status reports them.  The plain implementation gets the sequence without those pages."""
import pytest
import torch

from oracle import cache_budget_oracle as R
from _util import gen
from test_cache_budget_gpu import BF, F8, HF, check_out, fa, pools, score_error  # noqa: F401

pytestmark = pytest.mark.gpu


def without(table, n, page, bad):
    """The table and length of a sequence without the pages at `bad` (whole ones), and which of its tokens remain."""
    keep = [j for j in range(-(-n // page)) if j not in bad]
    seen = torch.tensor([t // page not in bad for t in range(n)], dtype=torch.bool)
    out = torch.full_like(table, -1)
    out[:len(keep)] = table[keep]
    return out, int(seen.sum()), seen


@pytest.mark.parametrize("qt,kv,d,h,h_k,sq,page,n,partition", [
    (BF, BF, 128, 8, 2, 1, 64, 1000, None), (HF, HF, 64, 4, 4, 1, 16, 700, 256), (BF, F8, 128, 8, 2, 2, 32, 900, None),
    (F8, F8, 128, 8, 2, 1, 64, 1500, 512), (HF, HF, 256, 8, 2, 1, 192, 1500, None), (BF, F8, 128, 4, 2, 1, 16, 333, None)])
def test_sparse_attention_leaves_them_out(fa, monkeypatch, qt, kv, d, h, h_k, sq, page, n, partition):   # noqa: F811
    m, cuda = fa
    g = gen(41)
    if partition:
        monkeypatch.setenv("FA_B200_DECODE_PARTITION", str(partition))
    kc, vc, bt, _, kd, vd = pools(g, [n, n - 100], h_k, page, kv, d)
    q = torch.randn(2, sq, h, d, generator=g).to(qt)
    last = -(-(n - 100) // page) - 1
    table, lens = bt[:, None].expand(2, h_k, -1).clone(), torch.tensor([[n] * h_k, [n - 100] * h_k], dtype=torch.int32)
    bads = {(0, 0): {1: -7}, (0, 1): {0: 10 ** 6, 2: kc.shape[0]}, (1, 0): {}, (1, 1): {j: -1 for j in range(last + 1)}}
    ref_table, ref_lens = table.clone(), lens.clone()
    for (i, x), bad in bads.items():
        for j, v in bad.items():
            table[i, x, j] = v
        if len(bad) == last + 1:
            ref_lens[i, x] = 0
        else:
            ref_table[i, x], ref_lens[i, x], _ = without(bt[i], int(lens[i, x]), page, bad)
    for x in range(2, h_k):
        ref_table[:, x], ref_lens[:, x] = bt, lens[:, x]
    out, lse = m.sparse_attn_with_kvcache(q.cuda(), kd, vd, table.cuda(), lens.cuda(), causal=True, return_softmax_lse=True)
    assert cuda.device_status() == 14
    ref, ref_lse, _ = R.decode_ref(q.float(), kc.float(), vc.float(), ref_table, ref_lens, d ** -0.5)
    check_out(out, ref, torch.nan_to_num(vc.float()).abs().amax().item(), "out")
    tol = score_error(q, kc, d ** -0.5) + 2.0 ** -20 * 16
    fin = ref_lse.isfinite()
    assert torch.equal(lse.cpu().isfinite(), fin) and ((lse.cpu().double() - ref_lse)[fin].abs() <= tol).all()
    empty = out.cpu()[1, :, h // h_k:2 * h // h_k]
    assert (empty == 0).all() and (lse.cpu()[1, h // h_k:2 * h // h_k] == float("inf")).all()
    m.sparse_attn_with_kvcache(q.cuda(), kd, vd, bt[:, None].expand(2, h_k, -1).contiguous().cuda(), lens.cuda())
    assert cuda.device_status() == 0


@pytest.mark.parametrize("qt,kv,d,h,h_k,sq,page,n,partition", [
    (BF, BF, 128, 8, 2, 1, 64, 1000, None), (HF, HF, 128, 8, 1, 2, 16, 1500, 256), (BF, F8, 128, 8, 2, 1, 64, 900, None),
    (F8, F8, 128, 8, 2, 4, 32, 600, None), (BF, BF, 192, 4, 2, 3, 64, 700, None)])
def test_decode_with_weights_leaves_them_out(fa, monkeypatch, qt, kv, d, h, h_k, sq, page, n, partition):   # noqa: F811
    m, cuda = fa
    g = gen(42)
    if partition:
        monkeypatch.setenv("FA_B200_DECODE_PARTITION", str(partition))
    kc, vc, bt, sl, kd, vd = pools(g, [n, 3 * page], h_k, page, kv, d)
    q = torch.randn(2, sq, h, d, generator=g).to(qt)
    bad = bt.clone()
    bad[0, 1], bad[0, 4] = kc.shape[0], -1
    ref_table, seen = bt.clone(), []
    ref_lens = sl.clone()
    ref_table[0], ref_lens[0], seen = without(bt[0], n, page, {1, 4})
    w = torch.rand(2, h_k, bt.shape[1] * page, generator=g)
    out, lse, got = m.flash_attn_with_kvcache_weights(q.cuda(), kd, vd, sl.cuda(), bad.cuda(), w.cuda(), causal=True,
                                                      return_softmax_lse=True, decay=0.5)
    assert cuda.device_status() == 14
    ref, ref_lse, weights = R.decode_ref(q.float(), kc.float(), vc.float(), ref_table, ref_lens, d ** -0.5)
    check_out(out, ref, torch.nan_to_num(vc.float()).abs().amax().item(), "out")
    tol = score_error(q, kc, d ** -0.5) + 2.0 ** -20 * 16
    assert ((lse.cpu().double() - ref_lse).abs() <= tol).all()
    got = got.cpu().double()
    for x in range(h_k):
        want = 0.5 * w[0, x, :n].double()
        want[seen] += weights[0][x]
        assert ((got[0, x, :n] - want).abs() <= 2 * tol * want + 2.0 ** -24 * want).all()
        assert torch.equal(got[0, x, :n][~seen], 0.5 * w[0, x, :n][~seen].double())
        want = 0.5 * w[1, x, :3 * page].double() + weights[1][x]
        assert ((got[1, x, :3 * page] - want).abs() <= 2 * tol * want).all()
        assert torch.equal(got[0, x, n:], w[0, x, n:].double())


@pytest.mark.parametrize("dtype,d,h,h_k,page,n,queries", [
    (BF, 128, 8, 2, 64, 600, 600), (HF, 128, 4, 2, 16, 500, 20), (BF, 256, 4, 1, 64, 700, 300), (HF, 64, 8, 1, 256, 1500, 1500),
    (BF, 192, 8, 1, 128, 2304, 2048)])
def test_weights_of_a_prompt_leave_them_out(fa, dtype, d, h, h_k, page, n, queries):   # noqa: F811
    m, cuda = fa
    g = gen(43)
    kc, _, bt, sl, kd, _ = pools(g, [n], h_k, page, dtype, d)
    q = torch.randn(queries, h, d, generator=g).to(dtype)
    gone = {0, 2}
    bad = bt.clone()
    bad[0, 0], bad[0, 2] = -3, kc.shape[0]
    table, left, seen = without(bt[0], n, page, gone)
    lse = torch.empty(h, queries)
    position = torch.arange(n)
    w = torch.rand(1, h_k, bt.shape[1] * page, generator=g)
    want = 0.5 * w[..., :n].double()
    group = h // h_k
    for x in range(h_k):
        keys = R.rows(kc, bt[0], x, n)
        for y in range(x * group, (x + 1) * group):
            s = q[:, y].double() @ keys.T * d ** -0.5
            s[(position[None, :] > torch.arange(queries)[:, None] + n - queries) | ~seen[None, :]] = -float("inf")
            lse[y] = torch.logsumexp(s, -1).masked_fill(~(s > -float("inf")).any(-1), float("inf")).float()
            want[0, x] += torch.exp(s - lse[y].double()[:, None]).sum(0)
    cu = torch.tensor([0, queries], dtype=torch.int32)
    got = m.attn_token_weights(q.cuda(), kd, lse.cuda(), cu.cuda(), queries, sl.cuda(), bad.cuda(), w.cuda(), decay=0.5).cpu()
    assert cuda.device_status() == 14
    tol = score_error(q, kc, d ** -0.5) + 2.0 ** -19
    assert ((got[..., :n].double() - want).abs() <= tol * want).all()
    assert torch.equal(got[..., :n][..., ~seen], 0.5 * w[..., :n][..., ~seen])


def test_selection_reports_the_pages_that_it_lists(fa):   # noqa: F811
    """A sequence that keeps all its pages, and pages that are taken whatever their score."""
    m, cuda = fa
    g = gen(44)
    bounds = torch.randn(40, 2, 2, 128, generator=g).to(BF).cuda()
    q = torch.randn(2, 1, 4, 128, generator=g).to(BF).cuda()
    bt = torch.arange(40, dtype=torch.int32).reshape(2, 20)
    for lens, at in (([128, 100], (0, 1)), ([1280, 1280], (0, 0)), ([1280, 1280], (1, 19))):
        bad = bt.clone()
        bad[at] = 40
        sl = torch.tensor(lens, dtype=torch.int32).cuda()
        m.kvcache_select_pages(q, bounds, bt.cuda(), sl, 64, 5)
        assert cuda.device_status() == 0
        pages, _, index = m.kvcache_select_pages(q, bounds, bad.cuda(), sl, 64, 5)
        assert cuda.device_status() == 14
        assert ((index[at[0]] == at[1]) == (pages[at[0]] == 40)).all()


def test_weights_of_a_prompt_leave_out_a_page_that_one_query_tile_sees(fa):   # noqa: F811
    """Items of one step, which one of the two sets of summing warps takes while the other writes the sums: 40 sequences of 384 tokens,
    a query tile of 128 tokens, the last 64 tokens of every sequence in no page."""
    m, cuda = fa
    g = gen(45)
    b, n, h_k, d = 40, 384, 4, 128
    kc, _, bt, sl, kd, _ = pools(g, [n] * b, h_k, 64, BF, d)
    bad = bt.clone()
    bad[:, 5] = torch.tensor([-1, kc.shape[0]] * (b // 2), dtype=torch.int32)
    q = torch.randn(b * n, h_k, d, generator=g).to(BF)
    lse = torch.full((h_k, b * n), 7.0)
    cu = torch.arange(b + 1, dtype=torch.int32) * n
    w = torch.rand(b, h_k, bt.shape[1] * 64, generator=g)
    ref = R.token_weights_ref(q, kc, lse, cu, bt, sl, w, d ** -0.5)
    tol = score_error(q, kc, d ** -0.5) + 2.0 ** -19
    args = (q.cuda(), kd, lse.cuda(), cu.cuda(), n, sl.cuda(), bad.cuda())
    for _ in range(5):
        got = m.attn_token_weights(*args, w.cuda()).cpu()
        assert torch.equal(got[..., 320:n], w[..., 320:n])
        assert ((got[..., :320].double() - ref[..., :320]).abs() <= tol * ref[..., :320]).all()
        assert cuda.device_status() == 14
