"""Decode with a bounded KV cache, beside flash_attn_with_kvcache: either read only the pages that matter for the new
tokens, or keep only the keys that matter at all.

Read less.  ``kvcache_page_bounds`` keeps the smallest and largest key value of every page; ``kvcache_select_pages`` bounds
with them the score that any key of a page can have and lists the best pages of every kv head;
``sparse_attn_with_kvcache`` attends to the listed pages::

    fa.kvcache_page_bounds(k_cache, block_table, lens, page_bounds=bounds)                # once after the prompt
    ...                                                                                   # every step: append k, v
    fa.kvcache_page_bounds(k_cache, block_table, lens, new_tokens=1, page_bounds=bounds)
    pages, sel_lens, _ = fa.kvcache_select_pages(q, bounds, block_table, lens, page_size, num_pages)
    out = fa.sparse_attn_with_kvcache(q, k_cache, v_cache, pages, sel_lens)

Keep less.  ``attn_token_weights`` (prompt) and ``flash_attn_with_kvcache_weights`` (decode) accumulate the attention weight
that every cached key receives; ``kvcache_evict`` cuts every kv head to the heaviest keys and moves them together.

Forward only.  Pools are (num_blocks, page_block_size, nheads_k, d) with any strides that are multiples of 16 bytes, but not
zero (a (num_blocks, nheads_k, page_block_size, d) pool is passed as its ``permute(0, 2, 1, 3)``), page_block_size 16, 32 or a
multiple of 64, d 128, or 64 / 192 / 256 with fp16 / bf16 pools.  Every call runs on the current stream of the tensors'
device and can be captured into a CUDA graph; rows of padded batches have length 0.
"""
from typing import Optional

import torch

import flash_attn_2_cuda as flash_attn_cuda


def kvcache_page_bounds(
    k_cache,
    block_table,
    cache_seqlens,
    new_tokens: Optional[int] = None,
    *,
    page_bounds: Optional[torch.Tensor] = None,
    dtype: Optional[torch.dtype] = None,
):
    """Smallest and largest value of every channel over the keys of each page: page_bounds (num_blocks, nheads_k, 2, d),
    [..., 0, :] the smallest.  Written are the pages that hold the last ``new_tokens`` tokens of every sequence (None: all of
    its pages), each from all of its rows below cache_seqlens; other pages keep what they have.  A page that sequences share
    has to be full in all of them.  ``page_bounds`` None: a new tensor, zero in the pages of no sequence, of ``dtype`` (default:
    the cache's type, bf16 for an fp8 cache)."""
    if new_tokens is not None and new_tokens <= 0:
        raise ValueError("new_tokens must be positive (None: every page)")
    if page_bounds is None:
        if dtype is None:
            dtype = torch.bfloat16 if k_cache.element_size() == 1 else k_cache.dtype
        nb, _, h_k, d = k_cache.shape
        page_bounds = torch.zeros((nb, h_k, 2, d), dtype=dtype, device=k_cache.device)
    elif dtype is not None and dtype != page_bounds.dtype:
        raise ValueError("dtype is the type of a new page_bounds: pass one or the other")
    return flash_attn_cuda.page_bounds(k_cache, block_table, cache_seqlens, page_bounds, new_tokens or 0)


def kvcache_select_pages(
    q,
    page_bounds,
    block_table,
    cache_seqlens,
    page_size: int,
    num_pages: int,
    sink_pages: int = 1,
    recent_pages: int = 1,
):
    """The pages that the new tokens' queries may attend to most, for every (sequence, kv head).  q: (batch, seqlen_q, nheads,
    d) fp16 / bf16, the last seqlen_q tokens of each sequence (seqlen_q x heads per kv head <= 16); page_bounds: of q's type.

    A page's score is the largest, over the queries and the heads of the group, of the sum over the channels of q_c times the
    page's largest value (q_c >= 0) or smallest value (q_c < 0): no key of the page has a larger q . k.  The first
    ``sink_pages``, the last ``recent_pages`` and the pages of the new tokens are always taken, then the highest scores, of
    equal ones the lowest page; a NaN score counts as the highest.  Scores are compared as 64-bit sums in a fixed order: pages
    with equal bounds are equal, and scores closer than 2^-48 of the sum of |q_c| |bound_c| may be taken in either order.

    Returns (page_table, seqlens, page_index): page_table int32 (batch, nheads_k, num_pages) the physical pages in the order of
    the sequence, -1 behind them; seqlens int32 (batch, nheads_k) the tokens in them; page_index their positions in the
    sequence.  The first two are what ``sparse_attn_with_kvcache`` takes.  A sequence of at most num_pages pages keeps all."""
    return flash_attn_cuda.page_select(q, page_bounds, block_table, cache_seqlens, page_size,
                                       num_pages, sink_pages, recent_pages)


def sparse_attn_with_kvcache(
    q,
    k_cache,
    v_cache,
    page_table,
    seqlens,
    softmax_scale=None,
    causal=False,
    s_aux=None,
    return_softmax_lse=False,
    *,
    out=None,
    q_descale=None,
    k_descale=None,
    v_descale=None,
):
    """flash_attn_with_kvcache over a list of pages for every kv head: page_table int32 (batch, nheads_k, n), seqlens int32
    (batch, nheads_k), the tokens in the listed pages (only the last listed page can be partly filled).  Types, sinks and
    descales as there; with several query tokens and ``causal`` the last listed tokens are taken for the new ones, as
    ``kvcache_select_pages`` provides.  Returns out, or (out, softmax_lse (batch, nheads, seqlen_q)): the softmax is that of the
    listed pages; a head without tokens returns 0 and an lse of +inf."""
    if softmax_scale is None:
        softmax_scale = q.shape[-1] ** (-0.5)
    if page_table.dim() != 3:
        raise RuntimeError("page_table must have shape (batch, nheads_k, n)")
    out, lse, _ = flash_attn_cuda.decode_budget(q, k_cache, v_cache, page_table, seqlens, softmax_scale, causal, out,
                                                s_aux, -1, None, None, 1.0, q_descale, k_descale, v_descale,
                                                return_softmax_lse)
    return (out, lse) if return_softmax_lse else out


def flash_attn_with_kvcache_weights(
    q,
    k_cache,
    v_cache,
    cache_seqlens,
    block_table,
    token_weights,
    softmax_scale=None,
    causal=False,
    window_size=(-1, -1),  # -1 means infinite context window
    s_aux=None,
    return_softmax_lse=False,
    *,
    decay=1.0,
    out=None,
    token_weights_out=None,
    q_descale=None,
    k_descale=None,
    v_descale=None,
):
    """flash_attn_with_kvcache that also accumulates the attention weight of every key: for t below a sequence's length

        token_weights_out[b, hk, t] = decay * token_weights[b, hk, t] + sum of the probabilities of key t over the query
                                      tokens and the heads of kv head hk's group

    token_weights: fp32 (batch, nheads_k, capacity), indexed by the position in the cache; None with ``token_weights_out``
    given: from zero.  Without ``token_weights_out`` it is updated in place; an output of its own must not overlap it.  Entries at
    and behind the length are left as they are; keys at and behind ``capacity`` are attended to and their weight is dropped.
    seqlen_q x heads per kv head <= 16 (prompts: ``attn_token_weights``).  A sink (s_aux) takes part in the softmax and in no
    key's weight.  Returns (out, token_weights_out), or (out, softmax_lse, token_weights_out).

    Scratch: 4 bytes per (sequence, query head, query token, position that block_table covers), so pass a table no wider than the
    longest sequence; up to 64 MB of it are kept for the stream's next calls."""
    if softmax_scale is None:
        softmax_scale = q.shape[-1] ** (-0.5)
    if block_table.dim() != 2:
        raise RuntimeError("block_table must have shape (batch, max_num_blocks_per_seq)")
    if q.shape[1] > 1 and not causal and window_size[1] >= 0:
        raise NotImplementedError("a right window bound with several decode tokens is outside the B200 hot path of this build")
    if token_weights is None and token_weights_out is None:
        raise RuntimeError("token_weights or token_weights_out is required")
    out, lse, w = flash_attn_cuda.decode_budget(q, k_cache, v_cache, block_table, cache_seqlens, softmax_scale, causal,
                                                out, s_aux, window_size[0], token_weights, token_weights_out,
                                                decay, q_descale, k_descale, v_descale, True)
    return (out, lse, w) if return_softmax_lse else (out, w)


def attn_token_weights(
    q,
    k_cache,
    softmax_lse,
    cu_seqlens_q,
    max_seqlen_q: int,
    cache_seqlens,
    block_table,
    token_weights,
    softmax_scale=None,
    causal=True,
    *,
    decay=1.0,
    token_weights_out=None,
):
    """The attention weight that the queries of a prompt (or its last queries: an observation window) gave to every cached key:
    for t below a sequence's length

        token_weights_out[b, hk, t] = decay * token_weights[b, hk, t] + sum over the queries that see key t and the heads of
                                      kv head hk's group of exp(softmax_scale q . k_t - softmax_lse)

    q: (total_q, nheads, d) fp16 / bf16 packed by cu_seqlens_q int32 (batch + 1), each sequence's queries being its last
    positions (causal: bottom-right aligned); softmax_lse fp32 (nheads, total_q): what flash_attn_varlen_func(...,
    return_softmax_lse=True) returned for them; k_cache: the paged keys, of q's type.  token_weights as in
    ``flash_attn_with_kvcache_weights``.  max_seqlen_q: an upper bound on the sequences' queries.  Returns token_weights_out."""
    if softmax_scale is None:
        softmax_scale = q.shape[-1] ** (-0.5)
    return flash_attn_cuda.token_weights(q, k_cache, softmax_lse, cu_seqlens_q, max_seqlen_q, cache_seqlens,
                                         block_table, token_weights, softmax_scale, causal, decay, token_weights_out)


def kvcache_evict(
    k_cache,
    v_cache,
    block_table,
    cache_seqlens,
    token_weights,
    budget: int,
    sink_tokens: int = 4,
    recent_tokens: Optional[int] = None,
    *,
    new_block_table=None,
    token_weights_out=None,
):
    """Cuts every sequence of more than ``budget`` tokens to ``budget`` tokens, for every kv head its own: the first
    ``sink_tokens``, the last ``recent_tokens`` (default: a quarter of what the sinks leave of the budget) and, of the others,
    those with the highest token_weights (equal ones: the lowest position; a NaN counts as the highest).

    Keys, values and weights of the kept tokens move, in their order, to positions 0, 1, ..: in place, every page belonging to
    one sequence then, or into the pages of ``new_block_table`` int32 (batch, n), none of which may be in block_table (shorter
    sequences are copied whole).  Keys keep the rotary position that they were written with.  The weights (in place, or into
    ``token_weights_out`` of the same capacity) become zero from the new to the old length.  Page bounds of the pages written
    have to be made anew.

    token_weights has to cover the lengths (capacity >= cache_seqlens; shorter ones cut the sequence, which device_status
    reports).

    Returns (kept_index, new_seqlens): kept_index int32 (batch, nheads_k, budget) the kept positions, ascending, -1 behind
    them; new_seqlens int32 (batch,) = min(cache_seqlens, budget)."""
    if recent_tokens is None:
        recent_tokens = max(0, budget - sink_tokens) // 4
    if sink_tokens < 0 or recent_tokens < 0 or sink_tokens + recent_tokens > budget:
        raise ValueError("sink_tokens and recent_tokens must not be negative and have to fit the budget")
    return flash_attn_cuda.kv_evict(k_cache, v_cache, block_table, cache_seqlens, token_weights, budget, sink_tokens,
                                    recent_tokens, new_block_table, token_weights_out)
