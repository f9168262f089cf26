"""GPU: scratch of the bounded-cache calls."""
import pytest
import torch

from test_cache_budget_gpu import BF, fa   # noqa: F401

pytestmark = pytest.mark.gpu


def test_large_scratch_goes_back(fa):   # noqa: F811
    """Scores of 8 sequences, 32 heads and a table of 262144 positions are 268 MB: not held after the call, and not shared with what
    another stream computes meanwhile."""
    m, cuda = fa
    g = torch.Generator(device="cuda").manual_seed(61)
    k = torch.randn(64, 64, 4, 128, device="cuda", generator=g).to(BF)
    table = torch.full((8, 4096), -1, dtype=torch.int32, device="cuda")
    table[:, :8] = torch.arange(64, device="cuda", dtype=torch.int32).reshape(8, 8)
    sl = torch.tensor([512, 3, 0, 511, 64, 65, 300, 448], dtype=torch.int32, device="cuda")
    qs = [torch.randn(8, 1, 32, 128, device="cuda", generator=g).to(BF) for _ in range(2)]
    w = torch.zeros(8, 4, 512, device="cuda")
    narrow = [m.flash_attn_with_kvcache_weights(q, k, k, sl, table[:, :8].contiguous(), None, token_weights_out=w.clone())[1] for q in qs]
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    before = torch.cuda.memory_allocated()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    outs = [[torch.zeros_like(w) for _ in range(6)] for _ in range(2)]
    torch.cuda.synchronize()
    for i in range(6):
        for x in (0, 1):
            with torch.cuda.stream(streams[x]):
                got[x].append(m.flash_attn_with_kvcache_weights(qs[x], k, k, sl, table, None, token_weights_out=outs[x][i])[1])
    torch.cuda.synchronize()
    for x in (0, 1):
        for y in got[x]:
            assert (y - narrow[x]).abs().max() <= 1e-5 * narrow[x].abs().max()
            assert torch.equal(y, got[x][0])
    del got, outs, y
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated() - before <= 2 * (64 << 20)
    assert cuda.device_status() == 0
