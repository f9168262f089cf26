"""GPU: decode with a bounded KV cache (flash_attn/kvcache_budget.py) against a plain implementation in 64 bits.

Tolerances.  Whole numbers, bounds and moved rows are exact.  Attention outputs: P is rounded to 16 bits before P V and
the output once more, each off by at most half a step relative to a value that is bounded by max |v|, so
|out - ref| <= 2 * (eps / 2) * max |v| + what 32 bits leave (1e-5 of it); an e4m3 cache under 16-bit queries keeps f16 P.
Log-sum-exp and weights are 32-bit: a score q . k * scale of 128 products has an error of at most d * 2^-23 times the sum
of the products' absolute values, which moves a probability by that share of itself; `score_error` computes it from the
inputs, 2^-20 for the exponential, the scaling and the sum of the probabilities comes on top."""
import math

import pytest
import torch

from oracle import cache_budget_oracle as R
from _util import gen, make_paged

pytestmark = pytest.mark.gpu

BF, HF, F8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


@pytest.fixture(scope="module")
def fa():
    import flash_attn
    import flash_attn_2_cuda
    assert torch.cuda.is_available()
    flash_attn_2_cuda.device_status()
    return flash_attn, flash_attn_2_cuda


def pools(g, lens, h_k, page, dtype, d=128, poison=True, bhsd=False):
    """CPU pools for the oracle (NaN where no token lies), their device copies (bhsd: stored by head) and tables."""
    kc, vc, bt, sl = make_paged(g, lens, h_k, page, torch.float32, poison=poison, d=d)
    kc, vc = kc.to(dtype), vc.to(dtype)
    put = (lambda x: x.permute(0, 2, 1, 3).contiguous().cuda().permute(0, 2, 1, 3)) if bhsd else (lambda x: x.cuda())
    return kc, vc, bt, sl, put(kc), put(vc)


def score_error(q, kc, scale):
    """d * 2^-23 * max sum |q||k| * scale: bound on a score's error in 32 bits."""
    k = torch.nan_to_num(kc.float()).abs().amax()
    return q.shape[-1] * 2.0 ** -23 * float(q.float().abs().sum(-1).amax() * k) * scale


def check_out(out, ref, vmax, what):
    # an e4m3 cache under 16-bit queries and every 16-bit type: P in the type of out or finer
    eps = torch.finfo(out.dtype).eps
    tol = eps * vmax + 1e-5 * vmax
    err = (out.double().cpu() - ref).abs().max().item()
    assert err <= tol, f"{what}: {err:.3e} > {tol:.3e}"


# ------------------------------------------------------------------------------------------------ page bounds

@pytest.mark.parametrize("dtype,odt,d,h_k,page,bhsd", [
    (BF, BF, 128, 8, 64, False), (HF, HF, 128, 3, 16, True), (BF, BF, 64, 2, 32, True), (HF, HF, 192, 2, 64, False),
    (BF, BF, 256, 1, 128, True), (F8, BF, 128, 4, 64, False), (F8, HF, 128, 2, 256, True),
    (torch.float8_e5m2, BF, 128, 2, 64, False)])
def test_page_bounds(fa, dtype, odt, d, h_k, page, bhsd):
    m, cuda = fa
    g = gen(1)
    lens = [1, 5 * page, 0, 3 * page + 1, 7 * page - 1, page]
    kc, _, bt, sl, kd, _ = pools(g, lens, h_k, page, dtype, d, bhsd=bhsd)
    got = m.kvcache_page_bounds(kd, bt.cuda(), sl.cuda(), dtype=odt)
    ref = R.page_bounds_ref(kc, bt, sl, torch.zeros(kc.shape[0], h_k, 2, d, dtype=odt))
    assert torch.equal(got.cpu(), ref)
    # the pages of the last tokens only: the others stay as they were
    for new in (1, 2, page, page + 1, 10 ** 6):
        start = torch.full_like(ref, 7.0)
        got = m.kvcache_page_bounds(kd, bt.cuda(), sl.cuda(), new_tokens=new, page_bounds=start.cuda())
        assert torch.equal(got.cpu(), R.page_bounds_ref(kc, bt, sl, start, new)), new
    assert cuda.device_status() == 0


def test_page_bounds_values_at_the_edges(fa):
    m, _ = fa
    kc = torch.zeros(2, 16, 1, 64, dtype=HF)
    kc[0, 0, 0, 0] = float("nan")       # a NaN key makes the bound NaN
    kc[0, :, 0, 1] = float("-inf")
    kc[0, 3, 0, 2], kc[0, 4, 0, 2] = 6e-8, -6e-8   # smallest subnormals
    kc[0, :, 0, 3] = -65504.0
    got = m.kvcache_page_bounds(kc.cuda(), torch.tensor([[0]], dtype=torch.int32).cuda(), torch.tensor([16], dtype=torch.int32).cuda()).cpu()
    assert got[0, 0, :, 0].isnan().all() and (got[0, 0, :, 1] == float("-inf")).all()
    assert float(got[0, 0, 0, 2]) < 0 < float(got[0, 0, 1, 2]) and (got[0, 0, :, 3] == -65504.0).all()
    assert (got[1] == 0).all()


# ------------------------------------------------------------------------------------------------ choice of pages

def _bounds(g, blocks, h_k, d, dtype):
    x = torch.randn(blocks, h_k, 2, d, generator=g)
    x = torch.stack([x.amin(2) - 1, x.amax(2) + 1], 2)
    return x.to(dtype)


@pytest.mark.parametrize("dtype,d,h,h_k,sq,page,k,sink,recent", [
    (BF, 128, 32, 8, 1, 64, 16, 1, 1), (HF, 64, 8, 8, 1, 16, 4, 0, 0), (BF, 192, 15, 3, 3, 32, 9, 2, 3), (HF, 256, 16, 1, 1, 256, 5, 1, 0),
    (BF, 128, 8, 2, 4, 16, 31, 0, 7), (HF, 128, 5, 1, 2, 64, 200, 1, 1)])
def test_select_pages(fa, dtype, d, h, h_k, sq, page, k, sink, recent):
    m, cuda = fa
    g = gen(2)
    lens = [120 * page - 3, 0, 1, 40 * page + 1, page * k, page * k + 1, 77]
    n = [-(-x // page) for x in lens]
    bt = torch.full((len(lens), max(n) + 2), -1, dtype=torch.int32)
    perm, at = torch.randperm(sum(n) + 5, generator=g).int(), 0
    for i, x in enumerate(n):
        bt[i, :x] = perm[at:at + x]
        at += x
    bounds = _bounds(g, sum(n) + 5, h_k, d, dtype)
    q = torch.randn(len(lens), sq, h, d, generator=g).to(dtype)
    sl = torch.tensor(lens, dtype=torch.int32)
    got = m.kvcache_select_pages(q.cuda(), bounds.cuda(), bt.cuda(), sl.cuda(), page, k, sink, recent)
    for x, y in zip(got, R.select_pages_ref(q, bounds, bt, sl, page, k, sink, recent)):
        assert torch.equal(x.cpu(), y)
    assert cuda.device_status() == 0


@pytest.mark.parametrize("kind", ["equal", "zero_q", "nearly_equal", "inf", "nan", "huge"])
def test_select_pages_at_the_border(fa, kind):
    """Scores that are equal, or differ by less than 32 bits can tell, or are not finite."""
    m, _ = fa
    g = gen(3)
    P, k, d = 300, 40, 128
    q = torch.randn(1, 1, 4, d, generator=g).to(BF)
    bounds = _bounds(g, P, 1, d, BF)
    if kind == "equal":
        bounds[:] = bounds[torch.randint(0, 7, (P,), generator=g)]
    elif kind == "zero_q":
        q.zero_()
    elif kind == "nearly_equal":
        # one page's bounds, one channel moved by a step, under a q whose other channels are far larger
        bounds[:] = bounds[:1]
        q[..., 0] = 2.0 ** -18
        q[..., 1:] *= 4
        bounds[:, :, :, 0] = (1.0 + torch.randint(0, 100, (P, 1, 1), generator=g) * 2.0 ** -7).to(BF)
    elif kind == "inf":
        bounds[5:60:3, 0, 1, 3] = float("inf")
        bounds[70:90, 0, 0, 9] = float("-inf")
    elif kind == "nan":
        bounds[100:120, 0, :, 7] = float("nan")
    else:
        bounds = (bounds.float() * 1e37).to(BF)
        q = (q.float() * 1e3).to(BF)
    bt = torch.randperm(P, generator=g).int()[None]
    sl = torch.tensor([P * 64 - 5], dtype=torch.int32)
    got = m.kvcache_select_pages(q.cuda(), bounds.cuda(), bt.cuda(), sl.cuda(), 64, k)
    for x, y in zip(got, R.select_pages_ref(q, bounds, bt, sl, 64, k)):
        assert torch.equal(x.cpu(), y)


def test_select_pages_of_a_long_sequence(fa):
    m, _ = fa
    g = gen(4)
    P, k = 20001, 513
    q = torch.randn(2, 1, 8, 64, generator=g).to(HF)
    bounds = _bounds(g, P, 2, 64, HF)
    bt = torch.stack([torch.randperm(P, generator=g).int(), torch.randperm(P, generator=g).int()])
    sl = torch.tensor([P * 16, 9000 * 16 + 1], dtype=torch.int32)
    got = m.kvcache_select_pages(q.cuda(), bounds.cuda(), bt.cuda(), sl.cuda(), 16, k)
    for x, y in zip(got, R.select_pages_ref(q, bounds, bt, sl, 16, k)):
        assert torch.equal(x.cpu(), y)


# ------------------------------------------------------------------------------------------------ attention over listed pages

@pytest.mark.parametrize("qt,kv,d,h,h_k,sq,page,k,partition,bhsd", [
    (BF, BF, 128, 32, 8, 1, 64, 12, 0, False), (HF, HF, 128, 8, 8, 1, 16, 40, 0, True), (BF, BF, 64, 10, 2, 3, 32, 33, 512, False),
    (HF, HF, 192, 4, 2, 1, 64, 20, 512, True), (BF, BF, 256, 16, 1, 1, 128, 9, 0, False), (BF, F8, 128, 8, 2, 1, 64, 30, 1024, False),
    (HF, F8, 128, 8, 2, 4, 32, 50, 0, True), (BF, BF, 128, 8, 2, 4, 64, 24, 512, False)])
def test_sparse_attention(fa, monkeypatch, qt, kv, d, h, h_k, sq, page, k, partition, bhsd):
    """Page lists of each kv head, lengths of their own, split and not; NaN in every row that holds no listed token."""
    m, cuda = fa
    if partition:
        monkeypatch.setenv("FA_B200_DECODE_PARTITION", str(partition))
    g = gen(5)
    lens = [50 * page - 3, page * 2, 0, 31 * page + 1, 77]
    kc, vc, bt, sl, kd, vd = pools(g, lens, h_k, page, kv, d, bhsd=bhsd)
    q = torch.randn(len(lens), sq, h, d, generator=g).to(qt)
    table = torch.full((len(lens), h_k, k), -1, dtype=torch.int32)
    sel = torch.zeros(len(lens), h_k, dtype=torch.int32)
    for i, n in enumerate(lens):
        pages = -(-n // page)
        for x in range(h_k):
            if pages == 0 or (i == 4 and x == 0):
                continue                             # one head of a sequence without a page
            c = min(k, pages, 1 + (7 * x + 11 * i) % k)
            if sq > 1:
                c = min(max(c, 2), pages)
            own = torch.randperm(pages - 1, generator=g)[:c - 1].sort().values if pages > 1 else torch.empty(0)
            own = torch.cat([own, torch.tensor([pages - 1.0])]).long() if sq == 1 or pages < 2 else torch.tensor(
                sorted(set(own.tolist()) | {pages - 1, pages - 2}))[-k:].long()
            table[i, x, :len(own)] = bt[i, own]
            sel[i, x] = len(own) * page - (pages * page - n)
    kw = {}
    ks = vs = 1.0
    if kv == F8:
        ks, vs = 0.5, 1.25
        kw = {"k_descale": torch.full((1,), ks).cuda(), "v_descale": torch.full((1,), vs).cuda()}
    out, lse = m.sparse_attn_with_kvcache(q.cuda(), kd, vd, table.cuda(), sel.cuda(), causal=True, return_softmax_lse=True, **kw)
    ref, ref_lse, _ = R.decode_ref(q, kc, vc, table, sel, d ** -0.5, True, k_scale=ks, v_scale=vs)
    check_out(out, ref, vs * float(torch.nan_to_num(vc.float()).abs().amax()), "out")
    tol = score_error(q, kc, ks * d ** -0.5) + 2.0 ** -20
    fine = torch.isfinite(ref_lse)
    assert torch.equal(torch.isfinite(lse.cpu()), fine)
    assert (lse.cpu().double() - ref_lse)[fine].abs().max() <= tol * ref_lse[fine].abs().clamp(min=1).max()
    assert cuda.device_status() == 0


def test_sparse_attention_over_all_pages_is_the_dense_call(fa, monkeypatch):
    """Bit for bit, where neither is split (they split by rules of their own)."""
    m, _ = fa
    monkeypatch.setenv("FA_B200_DECODE_PARTITION", "2048")
    g = gen(6)
    lens = [1500, 64, 0, 777]
    kc, vc, bt, sl, kd, vd = pools(g, lens, 2, 64, BF)
    q = torch.randn(4, 1, 8, 128, generator=g).to(BF).cuda()
    s = torch.randn(8, generator=g).cuda()
    table = bt[:, None].expand(4, 2, -1).contiguous().cuda()
    a = m.sparse_attn_with_kvcache(q, kd, vd, table, sl[:, None].expand(4, 2).contiguous().cuda(), s_aux=s, return_softmax_lse=True)
    b = m.flash_attn_with_kvcache(q, kd, vd, cache_seqlens=sl.cuda(), block_table=bt.cuda(), s_aux=s, return_softmax_lse=True)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


# ------------------------------------------------------------------------------------------------ weights of a decode call

@pytest.mark.parametrize("qt,kv,d,h,h_k,sq,page,partition,window,sink,bhsd", [
    (BF, BF, 128, 32, 8, 1, 64, 0, -1, False, False), (HF, HF, 128, 40, 8, 1, 16, 512, -1, True, True),
    (BF, BF, 64, 10, 2, 3, 32, 512, 300, False, False), (HF, HF, 192, 4, 4, 1, 64, 0, 100, True, False),
    (BF, BF, 256, 16, 1, 1, 128, 1024, -1, False, True), (BF, F8, 128, 8, 2, 1, 64, 1024, -1, False, False),
    (F8, F8, 128, 8, 2, 1, 64, 0, -1, False, False), (HF, F8, 128, 8, 2, 4, 32, 0, -1, False, False)])
def test_decode_with_weights(fa, monkeypatch, qt, kv, d, h, h_k, sq, page, partition, window, sink, bhsd):
    m, cuda = fa
    if partition:
        monkeypatch.setenv("FA_B200_DECODE_PARTITION", str(partition))
    g = gen(7)
    lens = [2003, sq, 0, 1025, 64, 300]
    kc, vc, bt, sl, kd, vd = pools(g, lens, h_k, page, kv, d, bhsd=bhsd)
    q = torch.randn(len(lens), sq, h, d, generator=g).to(qt)
    cap = bt.shape[1] * page + 3
    w = torch.rand(len(lens), h_k, cap, generator=g)
    s_aux = torch.randn(h, generator=g) if sink else None
    kw = {}
    ks = vs = qs = 1.0
    if kv == F8:
        ks, vs = 0.5, 1.25
        kw = {"k_descale": torch.full((1,), ks).cuda(), "v_descale": torch.full((1,), vs).cuda()}
    ref, ref_lse, rw = R.decode_ref(q, kc, vc, bt, sl, d ** -0.5, True, window, s_aux, ks * qs, vs)
    tol = score_error(q, kc, ks * d ** -0.5) + 2.0 ** -20
    args = (q.cuda(), kd, vd, sl.cuda(), bt.cuda())
    for decay, own_out in ((1.0, True), (0.75, False)):
        wd, wo = w.cuda(), torch.full_like(w, -5.0).cuda() if own_out else None
        out, lse, got = m.flash_attn_with_kvcache_weights(
            *args, wd, causal=True, window_size=(window, 0 if window >= 0 else -1), s_aux=None if s_aux is None else s_aux.cuda(),
            return_softmax_lse=True, decay=decay, token_weights_out=wo, **kw)
        if qt == F8:       # P in e4m3 steps on this path: the existing decode's own bound, and bf16 out
            assert (out.double().cpu() - ref).abs().max() <= 7e-2
        else:
            check_out(out, ref, vs * float(torch.nan_to_num(vc.float()).abs().amax()), "out")
        fine = torch.isfinite(ref_lse)
        assert torch.equal(torch.isfinite(lse.cpu()), fine)
        assert (lse.cpu().double() - ref_lse)[fine].abs().max() <= tol * ref_lse[fine].abs().clamp(min=1).max()
        assert got is (wo if own_out else wd)
        if own_out:
            assert torch.equal(wd.cpu(), w)
        got = got.cpu()
        for i, n in enumerate(lens):
            behind = got[i, :, n:]
            assert torch.equal(behind, torch.full_like(behind, -5.0) if own_out else w[i, :, n:])
            for x in range(h_k):
                r = w[i, x, :n].double() * decay + rw[i][x]
                # each probability is off by at most 2 tol of itself (score and log-sum-exp), the sum by a rounding more
                assert ((got[i, x, :n].double() - r).abs() <= (2 * tol + 2.0 ** -20) * r.abs()).all(), (i, x)
    # the attention itself is the call without weights, bit for bit where neither is split
    if not sink and window < 0:
        monkeypatch.setenv("FA_B200_DECODE_PARTITION", "2048")
        out, _ = m.flash_attn_with_kvcache_weights(*args, w.cuda(), causal=True, **kw)
        plain = m.flash_attn_with_kvcache(q.cuda(), kd, vd, cache_seqlens=sl.cuda(), block_table=bt.cuda(), causal=True, **kw)
        assert torch.equal(plain, out)
    assert cuda.device_status() == 0


def test_decode_weights_from_nothing_and_short_capacity(fa):
    m, cuda = fa
    g = gen(8)
    kc, vc, bt, sl, kd, vd = pools(g, [200, 130], 2, 64, BF)
    q = torch.randn(2, 1, 4, 128, generator=g).to(BF)
    wo = torch.full((2, 2, 150), 3.0).cuda()      # fewer entries than keys: those that there are
    m.flash_attn_with_kvcache_weights(q.cuda(), kd, vd, sl.cuda(), bt.cuda(), None, token_weights_out=wo)
    _, _, rw = R.decode_ref(q, kc, vc, bt, sl, 128 ** -0.5)
    tol = 2 * score_error(q, kc, 128 ** -0.5) + 2.0 ** -19
    for i, n in enumerate((150, 130)):
        for x in range(2):
            assert ((wo[i, x, :n].cpu().double() - rw[i][x][:n]).abs() <= tol * rw[i][x][:n]).all()
    assert (wo[1, :, 130:] == 3.0).all()
    assert cuda.device_status() == 0


# ------------------------------------------------------------------------------------------------ weights of a prompt

@pytest.mark.parametrize("dtype,d,h,h_k,page,causal,lens,nq,bhsd", [
    (BF, 128, 8, 2, 64, True, [300, 1, 0, 129, 512], None, False),
    (HF, 128, 15, 3, 16, True, [257, 64, 200], [32, 7, 1], True),
    (BF, 64, 8, 8, 32, True, [700], None, False), (HF, 192, 8, 1, 128, True, [400, 130], [300, 0], False),
    (BF, 256, 4, 4, 64, False, [129, 260], [40, 260], True), (HF, 128, 16, 1, 64, False, [500], [33], False),
    (BF, 128, 7, 7, 256, True, [1100], None, False), (BF, 128, 40, 1, 64, True, [333], [100], False),
    (HF, 64, 128, 1, 64, True, [140, 70], [9, 70], False),                 # one token per query tile
    (BF, 128, 4, 2, 16, True, [1, 130, 0, 257] * 40, [1, 5, 0, 8] * 40, True)])   # a batch of short windows
def test_token_weights_of_a_prompt(fa, dtype, d, h, h_k, page, causal, lens, nq, bhsd):
    m, cuda = fa
    g = gen(9)
    kc, vc, bt, sl, kd, _ = pools(g, lens, h_k, page, dtype, d, bhsd=bhsd)
    nq = nq or lens
    cu = torch.tensor([0] + torch.tensor(nq).cumsum(0).tolist(), dtype=torch.int32)
    q = torch.randn(int(cu[-1]), h, d, generator=g).to(dtype)
    lse = torch.empty(h, q.shape[0])
    for i, n in enumerate(lens):
        a, e = int(cu[i]), int(cu[i + 1])
        for x in range(h_k if e > a else 0):
            hs = slice(x * h // h_k, (x + 1) * h // h_k)
            keys = R.rows(kc, bt[i], x, n)
            lse[hs, a:e] = R.attention_ref(q[a:e, hs].double(), keys, keys, d ** -0.5, causal)[1].float()
    cap = bt.shape[1] * page
    w = torch.rand(len(lens), h_k, cap, generator=g)
    for decay in (1.0, 0.5):
        wo = torch.full_like(w, -5.0).cuda()
        got = m.attn_token_weights(q.cuda(), kd, lse.cuda(), cu.cuda(), max(nq), sl.cuda(), bt.cuda(), w.cuda(), causal=causal,
                                   decay=decay, token_weights_out=wo).cpu()
        ref = R.token_weights_ref(q, kc, lse, cu, bt, sl, w, d ** -0.5, causal, decay)
        tol = score_error(q, kc, d ** -0.5) + 2.0 ** -19
        for i, n in enumerate(lens):
            assert ((got[i, :, :n].double() - ref[i, :, :n]).abs() <= tol * ref[i, :, :n].abs()).all(), i
            assert (got[i, :, n:] == -5.0).all()
    assert cuda.device_status() == 0


def test_token_weights_of_a_long_prompt(fa):
    """Enough query tiles that a key's sum is split between CTAs: equal to the sum of two halves of the queries, and the
    whole mass is the number of (query, head) rows."""
    m, cuda = fa
    g = gen(10)
    n, h, h_k = 4000, 8, 2
    kc, vc, bt, sl, kd, vd = pools(g, [n], h_k, 64, BF, poison=False)
    q = torch.randn(n, h, 128, generator=g).to(BF).cuda()
    cu = torch.tensor([0, n], dtype=torch.int32).cuda()
    _, lse = m.flash_attn_varlen_func(q, kd, vd, cu, None, n, n, seqused_k=sl.cuda(), causal=True, block_table=bt.cuda(),
                                      return_softmax_lse=True)
    zero = torch.zeros(1, h_k, bt.shape[1] * 64).cuda()
    w = m.attn_token_weights(q, kd, lse, cu, n, sl.cuda(), bt.cuda(), zero.clone())
    mass = w[..., :n].double().sum(-1).cpu()
    assert (mass / (n * h // h_k) - 1).abs().max() <= 1e-5
    last = torch.tensor([0, n - 1500], dtype=torch.int32).cuda()
    again = m.attn_token_weights(q[:1500], kd, lse[:, :1500], torch.tensor([0, 1500], dtype=torch.int32).cuda(), 1500,
                                 torch.tensor([1500], dtype=torch.int32).cuda(), bt.cuda(), zero.clone())
    again = m.attn_token_weights(q[1500:], kd, lse[:, 1500:], last, n - 1500, sl.cuda(), bt.cuda(), again)
    assert ((w - again).abs() <= 1e-5 * w.abs() + 1e-12).all()
    twice = m.attn_token_weights(q, kd, lse, cu, n, sl.cuda(), bt.cuda(), zero.clone())
    assert torch.equal(w, twice)
    assert cuda.device_status() == 0


# ------------------------------------------------------------------------------------------------ eviction

@pytest.mark.parametrize("dtype,d,h_k,page,budget,sink,recent,in_place,bhsd", [
    (BF, 128, 4, 64, 200, 4, 50, False, False), (HF, 64, 2, 16, 333, 0, 0, True, False), (BF, 256, 1, 128, 1, 1, 0, False, True),
    (HF, 192, 3, 32, 64, 0, 64, True, True), (F8, 128, 2, 64, 500, 16, 100, True, False), (BF, 128, 8, 64, 1024, 4, 256, True, False),
    (torch.float8_e5m2, 128, 2, 256, 257, 3, 7, False, False), (F8, 64, 2, 64, 300, 4, 40, False, False),
    (torch.float8_e5m2, 192, 1, 16, 300, 4, 40, True, False)])
def test_evict(fa, dtype, d, h_k, page, budget, sink, recent, in_place, bhsd):
    m, cuda = fa
    g = gen(11)
    lens = [2003, budget, 0, budget + 1, 1, 700]
    kc, vc, bt, sl, _, _ = pools(g, lens, h_k, page, dtype, d, poison=False)
    cap = bt.shape[1] * page
    w = torch.rand(len(lens), h_k, cap, generator=g)
    w[0, :, 100:900] = w[0, :, 100:101]                 # ties
    w[3, :, :] = 0.0                                    # nothing but ties
    w[5, 0, 33], w[5, 0, 34], w[5, 0, 35], w[5, 0, 36] = float("nan"), -1.0, float("inf"), -0.0
    nbt = None
    if not in_place:
        need = [-(-min(n, budget) // page) for n in lens]
        extra = torch.zeros(sum(need), *kc.shape[1:]).to(dtype)
        nbt = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
        perm, at = (torch.randperm(sum(need), generator=g) + kc.shape[0]).int(), 0
        for i, n in enumerate(need):
            nbt[i, :n] = perm[at:at + n]
            at += n
        cat = lambda x: torch.cat([x.view(torch.uint8) if x.element_size() == 1 else x,   # noqa: E731
                                   extra.view(torch.uint8) if x.element_size() == 1 else extra]).view(x.dtype)
        kc, vc = cat(kc), cat(vc)
    raw = lambda x: x.view(torch.uint8) if x.element_size() == 1 else x.view(torch.int16)   # noqa: E731
    put = (lambda x: x.permute(0, 2, 1, 3).contiguous().cuda().permute(0, 2, 1, 3)) if bhsd else (lambda x: x.cuda())
    kd, vd, wd = put(kc), put(vc), w.cuda()
    wo = None if in_place else torch.full_like(w, -5.0).cuda()
    kept, new = m.kvcache_evict(kd, vd, bt.cuda(), sl.cuda(), wd, budget, sink, recent,
                                new_block_table=None if nbt is None else nbt.cuda(), token_weights_out=wo)
    r = R.evict_ref(raw(kc), raw(vc), bt, sl, w, budget, sink, recent, nbt, None if in_place else torch.full_like(w, -5.0))
    assert torch.equal(kept.cpu(), r[0]) and torch.equal(new.cpu(), r[1])
    assert torch.equal((wd if in_place else wo).cpu().view(torch.int32), r[4].view(torch.int32))
    if in_place:      # rows behind the new length are what the old tokens left there
        page_of = {}
        for i, n in enumerate(new.tolist()):
            for t in range(n):
                page_of.setdefault(int(bt[i, t // page]), []).append(t % page)
        for pg, rws in page_of.items():
            assert torch.equal(raw(kd.cpu().contiguous())[pg][rws], r[2][pg][rws])
            assert torch.equal(raw(vd.cpu().contiguous())[pg][rws], r[3][pg][rws])
    else:
        assert torch.equal(raw(kd.cpu().contiguous()), r[2]) and torch.equal(raw(vd.cpu().contiguous()), r[3])
    assert cuda.device_status() == 0


# ------------------------------------------------------------------------------------------------ as they are used together

def test_a_serving_loop(fa):
    """Prompt, weights of its last queries, eviction, then steps that append a token, renew the bounds of its page, choose
    pages and attend to them, or attend to everything and accumulate weights; each against the plain implementation."""
    m, cuda = fa
    g = gen(12)
    b, h, h_k, d, page, window, budget, k = 3, 8, 2, 128, 16, 24, 128, 6
    lens = [400, 130, 250]
    room = [-(-x // page) + 2 for x in lens]
    kc, vc, bt, sl, kd, vd = pools(g, [x * page for x in room], h_k, page, BF, poison=False)
    sl = torch.tensor(lens, dtype=torch.int32)
    scale = d ** -0.5
    q = torch.randn(sum(lens), h, d, generator=g).to(BF)
    cu = torch.tensor([0, 400, 530, 780], dtype=torch.int32)
    _, lse = m.flash_attn_varlen_func(q.cuda(), kd, vd, cu.cuda(), None, 400, 400, seqused_k=sl.cuda(), causal=True,
                                      block_table=bt.cuda(), return_softmax_lse=True)
    last = torch.cat([torch.arange(int(cu[i + 1]) - window, int(cu[i + 1])) for i in range(b)])
    cuw = torch.arange(0, (b + 1) * window, window, dtype=torch.int32)
    w = torch.zeros(b, h_k, bt.shape[1] * page).cuda()
    m.attn_token_weights(q[last].cuda(), kd, lse[:, last.cuda()].contiguous(), cuw.cuda(), window, sl.cuda(), bt.cuda(), w)
    wr = R.token_weights_ref(q[last], kc, lse.cpu()[:, last], cuw, bt, sl, torch.zeros_like(w.cpu()), scale)
    assert ((w.cpu().double() - wr).abs() <= 1e-4 * wr.abs()).all()
    kept, new = m.kvcache_evict(kd, vd, bt.cuda(), sl.cuda(), w, budget, 4, 32)
    assert new.tolist() == [128, 128, 128] and (kept[:, :, :4].cpu() == torch.arange(4, dtype=torch.int32)).all()
    cur = new
    bounds = m.kvcache_page_bounds(kd, bt.cuda(), cur)
    for step in range(20):
        kn, vn = torch.randn(b, 1, h_k, d, generator=g).to(BF).cuda(), torch.randn(b, 1, h_k, d, generator=g).to(BF).cuda()
        qn = torch.randn(b, 1, h, d, generator=g).to(BF).cuda()
        _, cur = cuda.kv_append(qn, kd, vd, kn, vn, cur, bt.cuda())
        m.kvcache_page_bounds(kd, bt.cuda(), cur, new_tokens=1, page_bounds=bounds)
        pages, n, index = m.kvcache_select_pages(qn, bounds, bt.cuda(), cur, page, k)
        out = m.sparse_attn_with_kvcache(qn, kd, vd, pages, n)
        kh, vh, lh = kd.cpu(), vd.cpu(), cur.cpu()
        rb = R.page_bounds_ref(kh, bt, lh, torch.zeros_like(bounds.cpu()))
        rp, rn, ri = R.select_pages_ref(qn.cpu(), rb, bt, lh, page, k)
        assert torch.equal(pages.cpu(), rp) and torch.equal(n.cpu(), rn) and torch.equal(index.cpu(), ri)
        ro, _, _ = R.decode_ref(qn.cpu(), kh, vh, rp, rn, scale)
        check_out(out, ro, float(vh.float().abs().amax()), "sparse")
        before = w.cpu().double()
        out, _ = m.flash_attn_with_kvcache_weights(qn, kd, vd, cur, bt.cuda(), w)
        ro, _, rw = R.decode_ref(qn.cpu(), kh, vh, bt, lh, scale)
        check_out(out, ro, float(vh.float().abs().amax()), "dense")
        for i in range(b):
            for x in range(h_k):
                r = before[i, x, :int(lh[i])] + rw[i][x]
                assert ((w[i, x, :int(lh[i])].cpu().double() - r).abs() <= 1e-4 * r).all()
    kept, new = m.kvcache_evict(kd, vd, bt.cuda(), cur, w, 100, 4, 16)
    assert new.tolist() == [100] * 3
    assert cuda.device_status() == 0


def test_budget_calls_in_a_graph_and_on_two_streams(fa):
    """A captured step replays while eager calls run on another stream; both give what the calls give alone."""
    m, cuda = fa
    g = gen(13)
    lens = [3000, 777, 64, 0]
    kc, vc, bt, sl, kd, vd = pools(g, lens, 2, 64, BF, poison=False)
    bt, sl = bt.cuda(), sl.cuda()
    q = [torch.randn(4, 1, 8, 128, generator=g).to(BF).cuda() for _ in range(2)]
    w0 = torch.rand(4, 2, bt.shape[1] * 64, generator=g).cuda()
    qp = torch.randn(600, 8, 128, generator=g).to(BF).cuda()
    lse = torch.randn(8, 600, generator=g).add_(8).cuda()
    cu = torch.tensor([0, 400, 500, 550, 600], dtype=torch.int32).cuda()

    def step(x, wo):
        bounds = m.kvcache_page_bounds(kd, bt, sl)
        pages, n, index = m.kvcache_select_pages(x, bounds, bt, sl, 64, 9)
        a = m.sparse_attn_with_kvcache(x, kd, vd, pages, n)
        o, wo = m.flash_attn_with_kvcache_weights(x, kd, vd, sl, bt, w0, token_weights_out=wo)
        pw = m.attn_token_weights(qp, kd, lse, cu, 400, sl, bt, w0, token_weights_out=torch.zeros_like(w0))
        return [bounds, pages, n, index, a, o, wo, pw]

    alone = [[t.clone() for t in step(x, torch.zeros_like(w0))] for x in q]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    static_q, wo = q[0].clone(), torch.zeros_like(w0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(static_q, wo)
    for rounds in range(5):
        x = rounds % 2
        static_q.copy_(q[x])
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            other = step(q[1 - x], torch.zeros_like(w0))
        torch.cuda.synchronize()
        for a, r in zip(held, alone[x]):
            assert torch.equal(a, r)
        for a, r in zip(other, alone[1 - x]):
            assert torch.equal(a, r)
    assert cuda.device_status() == 0


def test_positions_past_the_table_are_cut_and_reported(fa):
    """Lengths beyond the block table's row and page ids that are no pages: reported by device_status, never read."""
    m, cuda = fa
    g = gen(14)
    kc, vc, bt, sl, kd, vd = pools(g, [256, 256], 2, 64, BF, poison=False)
    long = torch.tensor([256, 5000], dtype=torch.int32).cuda()
    ref = m.kvcache_page_bounds(kd, bt.cuda(), sl.cuda())
    assert cuda.device_status() == 0
    assert torch.equal(m.kvcache_page_bounds(kd, bt.cuda(), long), ref)
    assert cuda.device_status() == 14
    q = torch.randn(2, 1, 4, 128, generator=g).to(BF).cuda()
    a = m.kvcache_select_pages(q, ref, bt.cuda(), sl.cuda(), 64, 3)
    b = m.kvcache_select_pages(q, ref, bt.cuda(), long, 64, 3)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert cuda.device_status() == 14
    bad = bt.clone()
    bad[1, 2] = 10 ** 6
    bad[0, 1] = -7
    start = torch.full_like(ref, 3.0)
    got = m.kvcache_page_bounds(kd, bad.cuda(), sl.cuda(), page_bounds=start.clone())
    assert (got[bt[1, 2].item()] == 3).all() and torch.equal(got[bt[1, 1].item()], ref[bt[1, 1].item()])
    assert cuda.device_status() == 14
    m.kvcache_select_pages(q, ref, bad.cuda(), sl.cuda(), 64, 3)
    assert cuda.device_status() == 14
    w = torch.rand(2, 2, 256, generator=g).cuda()
    before = kd.clone()
    m.kvcache_evict(kd, vd, bad.cuda(), sl.cuda(), w, 100, new_block_table=torch.full((2, 2), -1, dtype=torch.int32).cuda(),
                    token_weights_out=torch.zeros_like(w))
    assert torch.equal(kd, before)
    assert cuda.device_status() == 14
