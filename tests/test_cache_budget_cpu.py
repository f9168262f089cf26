"""CPU: refusals of the bounded-cache entry points, on the host, before any launch; struct mirrors; workspace sizes."""
import ctypes
import os
import re

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def binding():
    import importlib.util
    spec = importlib.util.spec_from_file_location("_fa_build", os.path.join(ROOT, "flash-attention-das_b200", "build.py"))
    b = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(b)
    b.build()
    import flash_attn_2_cuda
    return flash_attn_2_cuda


def structs(c):
    return (("fa_b200_page_bounds_params", c.PageBoundsParams), ("fa_b200_page_select_params", c.PageSelectParams),
            ("fa_b200_decode_budget_params", c.DecodeBudgetParams), ("fa_b200_token_weights_params", c.TokenWeightsParams),
            ("fa_b200_kv_evict_params", c.KvEvictParams))


def test_structs_mirror_the_header(binding):
    hdr = open(os.path.join(ROOT, "include", "fa_b200.h")).read()
    for name, cls in structs(binding):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), hdr, re.S).group(1)
        body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
        fields = [re.findall(r"(\w+)\s*$", x.strip())[0] for stmt in body.split(";") if stmt.strip() for x in stmt.split(",")]
        assert fields == [f[0] for f in cls._fields_], name


def test_a_struct_of_another_size_is_refused(binding):
    lib = binding.lib()
    one = {"PageBoundsParams": lib.fa_b200_page_bounds, "PageSelectParams": lib.fa_b200_page_select,
           "TokenWeightsParams": lib.fa_b200_token_weights, "KvEvictParams": lib.fa_b200_kv_evict}
    for cls_name, fn in one.items():
        cls = getattr(binding, cls_name)
        assert fn(None, None) == 1
        p = cls()
        p.struct_size -= 8
        assert fn(ctypes.byref(p), None) == 16
    d, e = binding.DecodeParams(), binding.DecodeBudgetParams()
    assert lib.fa_b200_decode_budget(ctypes.byref(d), None, None) == 1
    e.struct_size += 8
    assert lib.fa_b200_decode_budget(ctypes.byref(d), ctypes.byref(e), None) == 16
    assert lib.fa_b200_decode_budget_workspace_bytes(ctypes.byref(d), ctypes.byref(e)) == 0


def select(binding, **kw):
    p = binding.PageSelectParams()
    v = dict(b=2, seqlen_q=1, h=8, h_k=2, d=128, page_size=64, num_blocks=100, max_blocks_per_seq=40, num_pages=8, sink_pages=1,
             recent_pages=1, dtype=1)
    for k, x in {**v, **kw}.items():
        setattr(p, k, x)
    return binding.lib().fa_b200_page_select(ctypes.byref(p), None)


def test_select_refusals(binding):
    assert select(binding) == 1                                   # null pointers: everything else is in order
    assert select(binding, d=96) == 3 and select(binding, dtype=2) == 2
    assert select(binding, h=9) == 4 and select(binding, seqlen_q=5) == 4 and select(binding, h=64) == 4
    assert select(binding, page_size=48) == 7 and select(binding, num_pages=0) == 6 and select(binding, seqlen_q=0) == 6
    assert select(binding, sink_pages=-1) == 6 and select(binding, b=70000) == 6
    # the pages that are always taken have to fit
    assert select(binding, num_pages=2) == 1 and select(binding, num_pages=1) == 6
    assert select(binding, sink_pages=3, recent_pages=6) == 6 and select(binding, sink_pages=0, recent_pages=8) == 1
    assert select(binding, seqlen_q=4, sink_pages=0, recent_pages=0, num_pages=1) == 6   # four tokens can lie in two pages
    assert select(binding, max_blocks_per_seq=1 << 26) == 13
    assert select(binding, b=0) == 0


def test_bounds_evict_and_weights_refusals(binding):
    lib = binding.lib()

    def call(cls, fn, base, **kw):
        p = cls()
        for k, x in {**base, **kw}.items():
            setattr(p, k, x)
        return fn(ctypes.byref(p), None)

    base = dict(b=2, h_k=2, d=128, page_size=64, num_blocks=100, max_blocks_per_seq=40, dtype=1, bounds_dtype=1)
    f = lambda **kw: call(binding.PageBoundsParams, lib.fa_b200_page_bounds, base, **kw)   # noqa: E731
    assert f() == 1 and f(d=80) == 3 and f(dtype=3) == 2 and f(bounds_dtype=0) == 2 and f(dtype=4, bounds_dtype=2) == 2
    assert f(new_tokens=-1) == 6 and f(page_size=24) == 7 and f(b=0) == 0 and f(dtype=2, bounds_dtype=0) == 1
    base = dict(b=2, h_k=2, d=128, page_size=64, num_blocks=100, max_blocks_per_seq=40, dtype=1, budget=100, sink_tokens=4,
                recent_tokens=30, weights_capacity=2560)
    f = lambda **kw: call(binding.KvEvictParams, lib.fa_b200_kv_evict, base, **kw)   # noqa: E731
    assert f() == 1 and f(budget=0) == 6 and f(sink_tokens=71) == 6 and f(recent_tokens=-1) == 6 and f(d=32) == 3 and f(dtype=3) == 2
    assert f(page_size=8) == 7 and f(b=0) == 0 and f(budget=2 ** 31 - 1) == 13
    base = dict(b=2, h=8, h_k=2, d=128, page_size=64, num_blocks=100, max_blocks_per_seq=40, dtype=1, max_seqlen_q=10, total_q=20)
    f = lambda **kw: call(binding.TokenWeightsParams, lib.fa_b200_token_weights, base, **kw)   # noqa: E731
    assert f() == 1 and f(dtype=2) == 2 and f(h=258) == 4 and f(h=9) == 4 and f(total_q=-1) == 6 and f(page_size=65) == 7
    assert f(max_blocks_per_seq=200000) == 13 and f(b=0) == 0


def test_decode_budget_refusals_and_workspace(binding):
    lib = binding.lib()
    d, e = binding.DecodeParams(), binding.DecodeBudgetParams()
    d.d, d.dtype, d.out_dtype, d.b, d.h, d.h_k, d.page_size, d.max_blocks_per_seq = 128, 1, 1, 2, 8, 2, 64, 4
    size = lambda: lib.fa_b200_decode_budget_workspace_bytes(ctypes.byref(d), ctypes.byref(e))   # noqa: E731
    call = lambda: lib.fa_b200_decode_budget(ctypes.byref(d), ctypes.byref(e), None)             # noqa: E731
    assert size() == lib.fa_b200_decode_workspace_bytes(ctypes.byref(d)) == 0
    e.weights_out = 4096
    assert size() == 2 * 8 * 256 * 4            # scores of 2 x 8 rows of 256 keys
    assert call() == 1                          # no log-sum-exp to relate the weights to
    d.softmax_lse = 4096
    e.per_kv_head = 1
    assert call() == 9                          # page lists per kv head have no common positions to count weights for
    e.per_kv_head, d.o_partial_out = 0, 4096
    assert call() == 9
    d.o_partial_out, e.weights_out_head_stride = None, -1
    assert call() == 5


def test_python_refusals(binding):
    """Checks of the tensors before anything is launched: CPU tensors are refused as such."""
    import flash_attn as fa
    z = lambda *s, t=torch.bfloat16: torch.zeros(*s, dtype=t)   # noqa: E731
    k, bt, sl = z(4, 64, 2, 128), z(2, 2, t=torch.int32), z(2, t=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        fa.kvcache_page_bounds(k, bt, sl)
    with pytest.raises(ValueError, match="new_tokens"):
        fa.kvcache_page_bounds(k, bt, sl, new_tokens=0)
    with pytest.raises(RuntimeError, match="CUDA"):
        fa.kvcache_select_pages(z(2, 1, 8, 128), z(4, 2, 2, 128), bt, sl, 64, 4)
    with pytest.raises(RuntimeError, match="page_table"):
        fa.sparse_attn_with_kvcache(z(2, 1, 8, 128), k, k, bt, sl)
    with pytest.raises(RuntimeError):
        fa.flash_attn_with_kvcache_weights(z(2, 1, 8, 128), k, k, sl, bt, z(2, 2, 128, t=torch.float32))
    with pytest.raises(RuntimeError, match="token_weights"):
        fa.flash_attn_with_kvcache_weights(z(2, 1, 8, 128), k, k, sl, bt, None)
    with pytest.raises(ValueError, match="budget"):
        fa.kvcache_evict(k, k, bt, sl, z(2, 2, 128, t=torch.float32), 10, 8, 3)
    with pytest.raises(RuntimeError, match="CUDA"):
        fa.kvcache_evict(k, k, bt, sl, z(2, 2, 128, t=torch.float32), 10)
    grad = z(2, 1, 8, 128).requires_grad_()
    with pytest.raises(NotImplementedError, match="forward only"):
        fa.sparse_attn_with_kvcache(grad, k, k, z(2, 2, 2, t=torch.int32), z(2, 2, t=torch.int32))


def test_binding_argument_errors(binding):
    """The compiled host part: wrong counts and kinds of arguments are Python errors, before anything else."""
    k, i = torch.zeros(4, 64, 2, 128, dtype=torch.bfloat16), torch.zeros(2, 2, dtype=torch.int32)
    with pytest.raises(TypeError, match="expected 5"):
        binding.page_bounds(k, i)
    with pytest.raises(TypeError, match="k_cache must be a tensor"):
        binding.page_bounds(None, i, i, k, 0)
    with pytest.raises(TypeError, match="new_block_table must be a tensor"):
        binding.kv_evict(k, k, i, i[0], k.float(), 10, 0, 0, 3, None)
    with pytest.raises(RuntimeError, match="token_weights is required"):
        binding.kv_evict(k, k, i, i[0], None, 10, 0, 0, None, None)
    with pytest.raises(RuntimeError, match="addresses"):
        binding._host.bind((1, 2))
    with pytest.raises(NotImplementedError, match="forward only"):
        binding.page_bounds(k.clone().requires_grad_(), i, i[0], k, 0)
