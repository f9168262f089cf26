"""CPU: strides that the kernels cannot take are refused on the host, before any launch."""
import ctypes

import pytest

from test_cache_budget_cpu import binding  # noqa: F401

STRIDE = 5


def fill(p, **kw):
    for k, v in kw.items():
        setattr(p, k, v)
    return p


PTR = 4096   # looked at by no launch: the calls below end before one


def decode(c, **kw):
    p = fill(c.DecodeParams(), q=PTR, k_cache=PTR, v_cache=PTR, out=PTR, block_table=PTR, cache_seqlens=PTR, softmax_lse=PTR, d=128, dtype=1,
             out_dtype=1, b=1, h=4, h_k=2, seqlen_q=1, page_size=64, num_blocks=8, max_blocks_per_seq=4, q_batch_stride=512, q_row_stride=512,
             q_head_stride=128, o_batch_stride=512, o_row_stride=512, o_head_stride=128, k_block_stride=16384, k_row_stride=256, k_head_stride=128,
             v_block_stride=16384, v_row_stride=256, v_head_stride=128, workspace=PTR, workspace_bytes=1 << 40)
    return fill(p, **kw)


def test_an_axis_that_repeats_memory_has_no_tensor_map(binding):   # noqa: F811
    """Expanded keys, values or queries: the loads of a tile would go by another stride, past the end of the memory at worst."""
    lib = binding.lib()
    e = binding.DecodeBudgetParams()
    calls = (lambda **kw: lib.fa_b200_decode_paged(ctypes.byref(decode(binding, **kw)), None),
             lambda **kw: lib.fa_b200_decode_budget(ctypes.byref(decode(binding, **kw)), ctypes.byref(e), None))
    for call in calls:
        for name in ("k_head_stride", "k_row_stride", "k_block_stride"):   # K's map is made first; V's needs a driver before it
            assert call(**{name: 0}) == STRIDE, name

    def prompt(**kw):
        p = fill(binding.TokenWeightsParams(), q=PTR, q_row_stride=512, q_head_stride=128, softmax_lse=PTR, lse_head_stride=20, cu_seqlens_q=PTR,
                 k_cache=PTR, k_block_stride=16384, k_row_stride=256, k_head_stride=128, block_table=PTR, cache_seqlens=PTR, weights_out=PTR,
                 weights_capacity=256, weights_out_batch_stride=512, weights_out_head_stride=256, total_q=20, b=1, max_seqlen_q=20, h=4, h_k=2,
                 d=128, page_size=64, num_blocks=8, max_blocks_per_seq=4, dtype=1)
        return lib.fa_b200_token_weights(ctypes.byref(fill(p, **kw)), None)

    for name in ("q_row_stride", "q_head_stride"):
        assert prompt(**{name: 0}) == STRIDE, name

    def dense(**kw):
        p = fill(binding.FwdParams(), q=PTR, k=PTR, v=PTR, out=PTR, softmax_lse=PTR, b=2, seqlen_q=64, seqlen_k=64, h=4, h_k=2, d=128, dtype=1,
                 out_dtype=1, softmax_scale=0.1, window_left=-1, window_right=-1)
        for n, h in (("q", 4), ("k", 2), ("v", 2), ("o", 4)):
            fill(p, **{n + "_batch_stride": 64 * h * 128, n + "_row_stride": h * 128, n + "_head_stride": 128})
        return lib.fa_b200_fwd(ctypes.byref(fill(p, **kw)), None)

    for axis in ("batch", "row", "head"):
        assert dense(**{f"q_{axis}_stride": 0}) == STRIDE, axis


def test_rows_of_the_weights_that_share_memory(binding):   # noqa: F811
    """Every (sequence, kv head) writes its own row."""
    lib = binding.lib()
    ok = dict(weights_in_batch_stride=0, weights_in_head_stride=0, weights_out_batch_stride=512, weights_out_head_stride=256, weights_capacity=256)
    none = 1   # a null pointer that the call needs: the strides are in order

    def decode_(b=2, **kw):
        e = fill(binding.DecodeBudgetParams(), weights_out=PTR, decay=1.0, **{**ok, **kw})
        return lib.fa_b200_decode_budget(ctypes.byref(decode(binding, b=b, q=None)), ctypes.byref(e), None)

    base = dict(b=2, h_k=2, d=128, page_size=64, num_blocks=100, max_blocks_per_seq=40, dtype=1, block_table=PTR, cache_seqlens=PTR, k_cache=PTR,
                weights_out=PTR, k_block_stride=16384, k_row_stride=256, k_head_stride=128)

    def prompt(**kw):
        p = fill(binding.TokenWeightsParams(), h=8, max_seqlen_q=10, total_q=20, q=PTR, softmax_lse=PTR, cu_seqlens_q=PTR, q_row_stride=1024,
                 q_head_stride=128, **{**base, **ok, **kw})
        return lib.fa_b200_token_weights(ctypes.byref(p), None)

    assert decode_() == none
    for call in (decode_, prompt):
        assert call(weights_out_batch_stride=0) == STRIDE and call(weights_out_head_stride=0) == STRIDE
        assert call(weights_out_batch_stride=0, b=1) != STRIDE and call(weights_out_head_stride=0, weights_capacity=0) != STRIDE

    def evict(**kw):
        p = fill(binding.KvEvictParams(), budget=100, sink_tokens=4, recent_tokens=30, v_cache=PTR, weights_in=PTR, kept_index=PTR, seqlens_out=PTR,
                 **{**base, "v_block_stride": 16384, "v_row_stride": 256, "v_head_stride": 128, **ok, **kw})
        return lib.fa_b200_kv_evict(ctypes.byref(p), None)

    for name in ("weights_out_batch_stride", "weights_out_head_stride", "k_block_stride", "k_row_stride", "k_head_stride", "v_block_stride",
                 "v_row_stride", "v_head_stride"):
        assert evict(**{name: 0}) == STRIDE, name
