"""GPU: tensors whose strides the kernels cannot take are refused by the Python entry points, before any launch."""
import pytest
import torch

from test_cache_budget_gpu import BF, fa   # noqa: F401

pytestmark = pytest.mark.gpu

REFUSED = "strides"


def z(*s, t=BF):
    return torch.zeros(*s, dtype=t, device="cuda")


def test_expanded_keys_values_and_queries(fa):   # noqa: F811
    m, cuda = fa
    k, one, row = z(4, 64, 2, 128), z(4, 64, 1, 128).expand(4, 64, 2, 128), z(1, 64, 2, 128).expand(4, 64, 2, 128)
    bt, sl, q = torch.arange(4, device="cuda", dtype=torch.int32).reshape(2, 2), torch.full((2,), 128, device="cuda", dtype=torch.int32), z(2, 1, 4, 128)
    pages, lens = bt[:, None].expand(2, 2, 2).contiguous(), sl[:, None].expand(2, 2).contiguous()
    w = z(2, 2, 128, t=torch.float32)
    for bad in (one, row):
        for kk, vv in ((bad, k), (k, bad)):
            for call in (lambda: m.sparse_attn_with_kvcache(q, kk, vv, pages, lens),
                         lambda: m.flash_attn_with_kvcache_weights(q, kk, vv, sl, bt, w),
                         lambda: m.flash_attn_with_kvcache(q, kk, vv, cache_seqlens=sl, block_table=bt, causal=True)):
                with pytest.raises(RuntimeError, match=REFUSED):
                    call()
        cu = torch.tensor([0, 3, 6], dtype=torch.int32, device="cuda")
        with pytest.raises(RuntimeError, match=REFUSED):
            m.attn_token_weights(z(6, 4, 128), bad, z(4, 6, t=torch.float32), cu, 3, sl, bt, w)
        with pytest.raises(RuntimeError, match=REFUSED):
            m.attn_token_weights(z(6, 1, 128).expand(6, 4, 128), k, z(4, 6, t=torch.float32), cu, 3, sl, bt, w)
        # these read the pool by its strides
        m.kvcache_page_bounds(bad, bt, sl)
    x = z(2, 64, 4, 128)
    for q3, k3, v3 in ((x, x[:1].expand(2, 64, 4, 128), x), (x, x, x[:, :, :1].expand(2, 64, 4, 128)), (z(2, 1, 4, 128).expand(2, 64, 4, 128), x, x)):
        with pytest.raises(RuntimeError, match=REFUSED):
            m.flash_attn_func(q3, k3, v3, causal=True)
    torch.cuda.synchronize()
    assert cuda.device_status() == 0


def test_weights_that_overlap(fa):   # noqa: F811
    """Rows of the output that are one row, and an output that is the input moved by a key."""
    m, cuda = fa
    k, q = z(4, 64, 2, 128), z(2, 1, 4, 128)
    bt, sl = torch.arange(4, device="cuda", dtype=torch.int32).reshape(2, 2), torch.full((2,), 128, device="cuda", dtype=torch.int32)
    cu, lse = torch.tensor([0, 3, 6], dtype=torch.int32, device="cuda"), z(4, 6, t=torch.float32)
    w, flat = z(2, 2, 128, t=torch.float32), z(2 * 2 * 128 + 1, t=torch.float32)
    calls = (lambda a, b: m.flash_attn_with_kvcache_weights(q, k, k, sl, bt, a, token_weights_out=b),
             lambda a, b: m.attn_token_weights(z(6, 4, 128), k, lse, cu, 3, sl, bt, a, token_weights_out=b),
             lambda a, b: m.kvcache_evict(k, k, bt, sl, a, 100, token_weights_out=b))
    for call in calls:
        for rows in (w[:1].expand(2, 2, 128), w[:, :1].expand(2, 2, 128)):
            for b in (rows, None) if call is not calls[2] else (rows,):
                with pytest.raises(RuntimeError, match="stride"):
                    call(rows, b)
        with pytest.raises(RuntimeError, match="overlap"):
            call(flat[:-1].view(2, 2, 128), flat[1:].view(2, 2, 128))
        call(w[:1].expand(2, 2, 128), z(2, 2, 128, t=torch.float32))     # an input may repeat
        call(w, w)
    for bad in (z(4, 64, 1, 128).expand(4, 64, 2, 128), z(1, 64, 2, 128).expand(4, 64, 2, 128)):
        for kk, vv in ((bad, k), (k, bad)):
            with pytest.raises(RuntimeError, match="stride"):
                m.kvcache_evict(kk, vv, bt, sl, w, 100)
    torch.cuda.synchronize()
    assert cuda.device_status() == 0
