"""Decode with a bounded KV cache: six operators beside the paged attention entry points, as cases that can be timed and
compared with their plain form in elementary torch operations.

    bounds    kvcache_page_bounds              smallest and largest key value of every page, per kv head and channel
    select    kvcache_select_pages             the pages whose score bound for the new tokens' queries is highest
    sparse    sparse_attn_with_kvcache         attention of the new tokens over the selected pages
    weights   flash_attn_with_kvcache_weights  attention over the whole cache that also accumulates every key's weight
    prompt    attn_token_weights               the weight that a prompt's queries gave to every cached key
    evict     kvcache_evict                    keeps the heaviest keys of every kv head, in new pages

A case names its operator in ``op``.  Lengths of a ragged batch follow from the case alone (``_lens``); an idle slot of a
padded batch has length zero.  Pools are stored (blocks, page, kv heads, d), or (blocks, kv heads, page, d) where
``bhsd`` is true, and are handed over as the first with strides, as the framework's entry points take them.
"""
import math
import os
import sys

import torch

own = False

# the package's folder, as its own tests put it on the path
_PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flash-attention-das_b200")
if _PACKAGE not in sys.path:
    sys.path.insert(0, _PACKAGE)

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn}


def _case(name, op, b, L, h, hk, d=128, page=64, q="bf16", kv=None, ragged=False, bhsd=False, **more):
    c = {"op": op, "b": b, "L": L, "h": h, "hk": hk, "d": d, "page": page, "q": q, "kv": kv or q, "ragged": ragged, "bhsd": bhsd}
    c.update(more)
    if name is not None:
        c["name"] = name
    return c


def listed():
    return [
        # one step of a serving batch has appended a token to every sequence: the pages that hold the new tokens
        _case("bounds-step", "bounds", 64, 8192, 32, 8, ragged=True, new=1),
        # a batch of long prompts has just been written: every page
        _case("bounds-prompt", "bounds", 8, 32768, 32, 8, new=0),
        # one user's chat, middle length
        _case("select-chat", "select", 1, 16384, 32, 8, sq=1, k=32),
        # a serving batch at long context, small pages' worth of keys kept
        _case("select-batch-long", "select", 32, 131072, 32, 8, sq=1, k=128),
        # a handful of users, fp16, 4096 of 16384 tokens read
        _case("sparse-chat", "sparse", 4, 16384, 32, 8, q="f16", sq=1, k=64),
        # a full serving batch over an e4m3 cache with bf16 queries, 4096 of 8192 tokens read
        _case("sparse-batch-fp8", "sparse", 64, 8192, 32, 8, kv="e4m3", sq=1, k=64),
        # one sequence, an odd group of heads and an odd length
        _case("weights-one", "weights", 1, 4099, 40, 8, sq=1),
        # a ragged serving batch at long context
        _case("weights-batch-long", "weights", 16, 32768, 32, 8, page=256, ragged=True, sq=1),
        # the last 32 queries of each prompt look at the prompt (observation window)
        _case("prompt-window", "prompt", 4, 16384, 32, 8, q="f16", sq=32),
        # every query of one prompt
        _case("prompt-full", "prompt", 1, 8192, 32, 8, sq=8192),
        # two sequences just over their budget, odd sizes, head dimension 64
        _case("evict-two", "evict", 2, 5003, 24, 8, d=64, q="f16", budget=4096, sink=4, recent=256),
        # a serving batch at the end of its prompts, cut to a quarter
        _case("evict-batch", "evict", 32, 16384, 32, 8, ragged=True, budget=4096, sink=16, recent=512),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["bounds", "select", "sparse", "weights", "prompt", "evict"])
    hk = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 4, 5, 8])
    d = rng.choice([128, 128, 64, 192, 256])
    q = rng.choice(["bf16", "f16"])
    kv = q
    if op in ("bounds", "sparse", "weights") and d == 128 and rng.random() < 0.3:
        kv = "e4m3"
    page = rng.choice([16, 32, 64, 64, 128, 256])
    c = _case(None, op, _log(rng, 1, 64), 0, hk * group, hk, d, page, q, kv, rng.random() < 0.5, rng.random() < 0.3)
    # elements of K that the operator may go over: the largest listed case of each kind
    room = {"bounds": 8 * 32768, "select": 32 * 131072, "sparse": 64 * 8192, "weights": 12 * 32768, "prompt": 4 * 16384, "evict": 20 * 16384}[op] * 1024
    top = max(2, min(131072, room // (c["b"] * hk * d)))
    c["L"] = _log(rng, 1, top)
    sq = rng.randint(1, max(1, min(4, 16 // group)))
    if op == "bounds":
        c["new"] = rng.choice([0, 1, _log(rng, 1, c["L"])])
    elif op in ("select", "sparse"):
        c["sq"] = min(sq, c["L"])
        c["k"] = _log(rng, 4, max(4, min(512, -(-c["L"] // page) + 2)))
        if op == "sparse":
            c["sq"] = 1
    elif op == "weights":
        c["sq"] = min(sq, c["L"])
    elif op == "prompt":
        c["b"] = min(c["b"], 8)
        c["sq"] = _log(rng, 1, c["L"])
        while c["b"] * c["h"] * c["sq"] * c["L"] > 32 * 8192 * 4096:
            c["sq"] = max(1, c["sq"] // 2)
            c["L"] = max(c["sq"], c["L"] * 3 // 4)
    else:
        c["budget"] = _log(rng, 1, max(1, c["L"]))
        c["sink"] = min(rng.choice([0, 4, 16]), c["budget"])
        c["recent"] = rng.randint(0, c["budget"] - c["sink"])
    return c


def _lens(c):
    """The sequences' lengths: all L, or spread by the golden ratio over [1, L] with the longest first and, from four
    sequences on, an idle slot at the end."""
    if not c["ragged"]:
        return [c["L"]] * c["b"]
    n = [c["L"] if i == 0 else 1 + int((c["L"] - 1) * ((i * 0.6180339887498949) % 1.0)) for i in range(c["b"])]
    if c["b"] >= 4:
        n[-1] = 0
    return n


def _pages(c):
    return [-(-n // c["page"]) for n in _lens(c)]


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _pool(c, blocks, g):
    """A pool of keys or values: unit noise over a few channels that are far from zero in every token of a head."""
    hk, d, page = c["hk"], c["d"], c["page"]
    shape = (blocks, hk, page, d) if c["bhsd"] else (blocks, page, hk, d)
    x = torch.empty(shape, dtype=torch.bfloat16 if c["kv"] == "e4m3" else _TYPES[c["kv"]], device="cuda").normal_(generator=g)
    offset = 4.0 * torch.randn(hk, d, device="cuda", generator=g) * (torch.rand(hk, d, device="cuda", generator=g) < 0.03)
    x += (offset[:, None, :] if c["bhsd"] else offset).to(x.dtype)
    if c["kv"] == "e4m3":
        x = x.to(torch.float8_e4m3fn)
    return x.permute(0, 2, 1, 3) if c["bhsd"] else x


def _table(c, g, first=0, pages=None):
    """Block table over a random order of the pool's pages, -1 behind each sequence's last page."""
    pages = pages or _pages(c)
    order = torch.randperm(sum(pages), device="cuda", generator=g).to(torch.int32) + first
    table = torch.full((c["b"], max(max(pages), 1)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(pages):
        table[i, :n] = order[at:at + n]
        at += n
    return table


def prepare(case, seed):
    c, g = case, _generator(seed)
    s = {"case": c, "lens": torch.tensor(_lens(c), dtype=torch.int32, device="cuda"), "scale": c["d"] ** -0.5}
    b, h, hk, d, page = c["b"], c["h"], c["hk"], c["d"], c["page"]
    blocks = sum(_pages(c))
    s["table"] = _table(c, g)
    qt = _TYPES[c["q"]]
    op = c["op"]
    if op == "select":
        # bounds of pages of 64 tokens: about +- 2.4 around the channel's own offset
        mid = 0.3 * torch.randn(blocks, hk, 1, d, device="cuda", generator=g)
        half = 2.4 + 0.4 * torch.randn(blocks, hk, 2, d, device="cuda", generator=g)
        sign = torch.tensor([-1.0, 1.0], device="cuda")[:, None]
        s["bounds"] = (mid + sign * half.abs()).to(qt)
    else:
        s["k"] = _pool(c, blocks, g) if op != "evict" else None
    if op in ("select", "sparse", "weights"):
        s["q"] = (1.5 * torch.randn(b, c["sq"], h, d, device="cuda", generator=g)).to(qt)
    if op == "bounds":
        s["bounds"] = torch.zeros(blocks, hk, 2, d, dtype=qt, device="cuda")
    if op in ("sparse", "weights"):
        s["v"] = _pool(c, blocks, g)
        s["kd"] = s["vd"] = None
        if c["kv"] == "e4m3":
            s["kd"] = torch.full((1,), 0.9, device="cuda")
            s["vd"] = torch.full((1,), 1.1, device="cuda")
    if op == "sparse":
        # a selection of each kv head: the last page and others in ascending order
        pages = torch.tensor(_pages(c), device="cuda")
        score = torch.rand(b, hk, s["table"].shape[1], device="cuda", generator=g)
        at = torch.arange(s["table"].shape[1], device="cuda")
        score = torch.where(at < pages[:, None, None], score, -1.0)
        score = torch.where(at == (pages - 1)[:, None, None], 2.0, score)
        k = min(c["k"], s["table"].shape[1])
        top, index = score.topk(k, -1)
        index = torch.where(top >= 0, index, 1 << 30).sort(-1).values
        full = torch.full((b, hk, c["k"]), -1, dtype=torch.int32, device="cuda")
        full[..., :k] = torch.where(index < (1 << 30), s["table"][:, None].expand(b, hk, -1).gather(-1, index.clamp(max=s["table"].shape[1] - 1)), -1)
        s["pages"] = full
        n = torch.minimum(pages, torch.tensor(c["k"], device="cuda"))
        short = (page - s["lens"] % page) % page
        s["sel_lens"] = (n * page - short).clamp(min=0).to(torch.int32)[:, None].expand(b, hk).contiguous()
    if op in ("weights", "prompt", "evict"):
        cap = s["table"].shape[1] * page
        w = torch.randn(b, hk, cap, device="cuda", generator=g).mul_(2).exp_()
        # keys that no query has looked at yet carry no weight: equal values in numbers
        s["w"] = torch.where(torch.rand(b, hk, cap, device="cuda", generator=g) < 0.1, 0.0, w)
        s["w_out"] = torch.zeros_like(s["w"])
    if op == "prompt":
        n = [min(c["sq"], x) for x in _lens(c)]
        s["cu"] = torch.tensor([sum(n[:i]) for i in range(b + 1)], dtype=torch.int32, device="cuda")
        s["q"] = (1.5 * torch.randn(sum(n), h, d, device="cuda", generator=g)).to(qt)
        s["n"], s["max_q"] = n, max(n)
        s["lse"] = _lse(s)
    if op == "evict":
        kept = [-(-min(x, c["budget"]) // page) for x in _lens(c)]
        s["new_table"] = _table(c, g, first=blocks, pages=kept)
        s["first_new"] = blocks
        s["k"], s["v"] = _pool(c, blocks + sum(kept), g), _pool(c, blocks + sum(kept), g)
    return s


def _lse(s):
    """Log-sum-exp of every query of a prompt over the keys that it sees, as the attention call of the prompt returned it."""
    c = s["case"]
    out = torch.empty(c["h"], s["q"].shape[0], device="cuda")
    at = 0
    for i, (n, length) in enumerate(zip(s["n"], _lens(c))):
        if n == 0:
            continue
        pages = s["table"][i, :-(-length // c["page"])].long()
        hidden = torch.arange(length, device="cuda")[None, :] > (torch.arange(n, device="cuda") + length - n)[:, None]
        for x in range(c["hk"]):
            keys = s["k"][pages][:, :, x].reshape(-1, c["d"])[:length].float()
            for y in range(x * c["h"] // c["hk"], (x + 1) * c["h"] // c["hk"]):
                score = s["q"][at:at + n, y].float() @ keys.T * s["scale"]
                out[y, at:at + n] = torch.logsumexp(score.masked_fill_(hidden, -math.inf), -1)
        at += n
    return out


# ---------------------------------------------------------------------------------------------- plain forms

def _rows(pool, table):
    """The rows of a pool's pages in the table's order, in 32 bits: table (b, n) -> (b, kv heads, n * page, d)."""
    b, n = table.shape
    x = pool.view(torch.uint8) if pool.element_size() == 1 else pool
    x = x[table.clamp(min=0).long()]
    x = x.view(pool.dtype) if pool.element_size() == 1 else x
    return x.float().reshape(b, -1, *pool.shape[2:]).transpose(1, 2)


def _rows_by_head(pool, table):
    """The same with a table (b, kv heads, n) for each kv head."""
    b, hk, n = table.shape
    x = pool.view(torch.uint8) if pool.element_size() == 1 else pool
    x = x.transpose(1, 2)[table.clamp(min=0).long(), torch.arange(hk, device=table.device)[None, :, None]]
    x = x.view(pool.dtype) if pool.element_size() == 1 else x
    return x.float().reshape(b, hk, n * pool.shape[1], pool.shape[3])


def _attention(s, keys, values, lens):
    """Softmax attention of the last sq tokens: (out, log-sum-exp, weight of each key).  lens (b, kv heads or 1)."""
    c = s["case"]
    b, sq, h, d = s["q"].shape
    hk, group = c["hk"], h // c["hk"]
    q = s["q"].float().reshape(b, sq, hk, group, d).permute(0, 2, 3, 1, 4)
    scale = s["scale"] * (s["kd"] if s["kd"] is not None else 1.0)
    score = (q.reshape(b, hk, group * sq, d) @ keys.transpose(-1, -2) * scale).reshape(b, hk, group, sq, -1)
    at = torch.arange(keys.shape[2], device=keys.device)
    behind = sq - 1 - torch.arange(sq, device=keys.device)
    seen = at < (lens[:, :, None, None] - behind[:, None])          # (b, hk or 1, sq, keys)
    score = torch.where(seen[:, :, None], score, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, 1.0)
    out = p.reshape(b, hk, group * sq, -1) @ values * (s["vd"] if s["vd"] is not None else 1.0)
    out = out.reshape(b, hk, group, sq, d).permute(0, 3, 1, 2, 4).reshape(b, sq, h, d).to(s["q"].dtype)
    lse = torch.where(total > 0, top + torch.log(total), math.inf).reshape(b, h, sq)
    return out, lse, p.sum((2, 3))


def _plain_bounds(s):
    c = s["case"]
    page, width = c["page"], s["table"].shape[1]
    n = (s["lens"] + page - 1) // page
    first = torch.zeros_like(n) if c["new"] == 0 else (s["lens"] - c["new"]).clamp(min=0) // page
    m = width if c["new"] == 0 else min(width, (c["new"] - 1) // page + 2)         # pages that new tokens can lie in
    slot = first[:, None] + torch.arange(m, device="cuda")
    ids = s["table"].gather(1, slot.clamp(max=width - 1).long())
    x = _rows(s["k"], ids).reshape(c["b"], c["hk"], m, page, c["d"])
    there = slot[:, :, None] * page + torch.arange(page, device="cuda") < s["lens"][:, None, None]
    there = there[:, None, :, :, None]
    low = torch.where(there, x, math.inf).amin(3)
    high = torch.where(there, x, -math.inf).amax(3)
    both = torch.stack([low, high], 3).transpose(1, 2)                              # (b, m, hk, 2, d)
    touched = slot < n[:, None]
    s["bounds"][ids[touched].long()] = both[touched].to(s["bounds"].dtype)
    return s["bounds"]


def _plain_select(s):
    c = s["case"]
    b, sq, h, d = s["q"].shape
    hk, page, k = c["hk"], c["page"], c["k"]
    x = s["bounds"][s["table"].clamp(min=0).long()].double().permute(0, 2, 1, 3, 4)   # (b, hk, pages, 2, d): 64 bits, the choice has a border
    q = s["q"].double().reshape(b, sq, hk, h // hk, d).transpose(1, 2).reshape(b, hk, -1, d)
    score = q.clamp(max=0) @ x[..., 0, :].transpose(-1, -2) + q.clamp(min=0) @ x[..., 1, :].transpose(-1, -2)
    score = score.amax(2)                                                              # (b, hk, pages)
    at = torch.arange(score.shape[-1], device="cuda")
    n = ((s["lens"] + page - 1) // page)[:, None, None]
    open_from = ((s["lens"] - sq).clamp(min=0) // page)[:, None, None]                 # the pages that hold the new tokens
    score = torch.where((at < 1) | (at >= torch.minimum(n - 1, open_from)), math.inf, score)
    score = torch.where(at < n, score, -math.inf)
    order = score.sort(dim=-1, descending=True, stable=True).indices[..., :k]
    order = torch.where(order < n, order, 1 << 30).sort(-1).values
    index = torch.full((b, hk, k), -1, dtype=torch.int32, device="cuda")
    index[..., :order.shape[-1]] = torch.where(order < (1 << 30), order, -1).to(torch.int32)
    pages = torch.where(index >= 0, s["table"][:, None].expand(b, hk, -1).gather(-1, index.clamp(min=0).long()), -1)
    short = ((page - s["lens"] % page) % page)[:, None]
    lens = ((index >= 0).sum(-1) * page - short).clamp(min=0).to(torch.int32)
    return pages, lens, index


def _plain_sparse(s):
    out, lse, _ = _attention(s, _rows_by_head(s["k"], s["pages"]), _rows_by_head(s["v"], s["pages"]), s["sel_lens"])
    return out, lse


def _plain_weights(s):
    out, lse, w = _attention(s, _rows(s["k"], s["table"]), _rows(s["v"], s["table"]), s["lens"][:, None])
    at = torch.arange(w.shape[-1], device="cuda")
    s["w_out"].copy_(torch.where(at < s["lens"][:, None, None], s["w"] + w, s["w_out"]))
    return out, lse, s["w_out"]


def _plain_prompt(s):
    c = s["case"]
    hk, group, d, b = c["hk"], c["h"] // c["hk"], c["d"], c["b"]
    top = s["max_q"]
    n = s["cu"][1:] - s["cu"][:-1]
    row = torch.arange(top, device="cuda")
    packed = (s["cu"][:-1, None] + row).clamp(max=max(s["q"].shape[0] - 1, 0)).long()
    q = s["q"][packed].float().reshape(b, top, hk, group, d).permute(0, 2, 3, 1, 4)            # (b, hk, group, top, d)
    lse = s["lse"][:, packed].reshape(hk, group, b, top).permute(2, 0, 1, 3)
    keys = _rows(s["k"], s["table"])
    score = q.reshape(b, hk, group * top, d) @ keys.transpose(-1, -2)
    score = score.mul_(s["scale"]).reshape(b, hk, group, top, -1).sub_(lse[..., None]).exp_()
    at = torch.arange(keys.shape[2], device="cuda")
    seen = (at <= (row[:, None] + (s["lens"] - n)[:, None, None])) & (row[:, None] < n[:, None, None])
    score.masked_fill_(~seen[:, None, None], 0.0)
    s["w_out"].copy_(torch.where(at < s["lens"][:, None, None], s["w"] + score.sum((2, 3)), s["w_out"]))
    return s["w_out"]


def _plain_evict(s):
    c = s["case"]
    b, hk, budget, page = c["b"], c["hk"], c["budget"], c["page"]
    cap = s["w"].shape[-1]
    at = torch.arange(cap, device="cuda")
    n = s["lens"][:, None, None]
    value = torch.where((at < c["sink"]) | (at >= n - c["recent"]), math.inf, s["w"])
    value = torch.where(at < n, value, -math.inf)
    order = value.sort(dim=-1, descending=True, stable=True).indices[..., :budget]
    order = torch.where(order < n, order, 1 << 30).sort(-1).values
    kept = torch.full((b, hk, budget), -1, dtype=torch.int32, device="cuda")
    kept[..., :order.shape[-1]] = torch.where(order < (1 << 30), order, -1).to(torch.int32)
    new_lens = torch.clamp(s["lens"], max=budget)
    there = kept >= 0
    i, j, to = there.nonzero(as_tuple=True)
    src = kept[there].long()
    from_page, to_page = s["table"][i, src // page].long(), s["new_table"][i, to // page].long()
    s["k"][to_page, to % page, j] = s["k"][from_page, src % page, j]
    s["v"][to_page, to % page, j] = s["v"][from_page, src % page, j]
    s["w_out"][i, j, to] = s["w"][i, j, src]
    behind = (at >= new_lens[:, None, None]) & (at < n)
    s["w_out"].masked_fill_(behind, 0.0)
    return kept, new_lens, s["k"][s["first_new"]:], s["v"][s["first_new"]:], s["w_out"]


_PLAIN = {"bounds": _plain_bounds, "select": _plain_select, "sparse": _plain_sparse, "weights": _plain_weights,
          "prompt": _plain_prompt, "evict": _plain_evict}


# ------------------------------------------------------------------------------------- the framework's calls

def _own(s):
    import flash_attn as fa
    c = s["case"]
    op = c["op"]
    if op == "bounds":
        return fa.kvcache_page_bounds(s["k"], s["table"], s["lens"], new_tokens=c["new"] or None, page_bounds=s["bounds"])
    if op == "select":
        return fa.kvcache_select_pages(s["q"], s["bounds"], s["table"], s["lens"], c["page"], c["k"], sink_pages=1, recent_pages=1)
    if op == "sparse":
        return fa.sparse_attn_with_kvcache(s["q"], s["k"], s["v"], s["pages"], s["sel_lens"], s["scale"], causal=True,
                                           return_softmax_lse=True, k_descale=s["kd"], v_descale=s["vd"])
    if op == "weights":
        return fa.flash_attn_with_kvcache_weights(s["q"], s["k"], s["v"], s["lens"], s["table"], s["w"], s["scale"], causal=True,
                                                  return_softmax_lse=True, token_weights_out=s["w_out"], k_descale=s["kd"],
                                                  v_descale=s["vd"])
    if op == "prompt":
        return fa.attn_token_weights(s["q"], s["k"], s["lse"], s["cu"], s["max_q"], s["lens"], s["table"], s["w"], s["scale"],
                                     causal=True, token_weights_out=s["w_out"])
    kept, lens = fa.kvcache_evict(s["k"], s["v"], s["table"], s["lens"], s["w"], c["budget"], sink_tokens=c["sink"],
                                  recent_tokens=c["recent"], new_block_table=s["new_table"], token_weights_out=s["w_out"])
    return kept, lens, s["k"][s["first_new"]:], s["v"][s["first_new"]:], s["w_out"]


def run(state):
    if own:
        return _own(state)
    return _PLAIN[state["case"]["op"]](state)


def work(case):
    c = case
    lens, es, qs = _lens(c), 1 if case["kv"] == "e4m3" else 2, 2
    b, h, hk, d, page = c["b"], c["h"], c["hk"], c["d"], c["page"]
    op = c["op"]
    tokens = sum(lens)
    if op == "bounds":
        rows = pages = 0
        for n in lens:
            first = 0 if c["new"] == 0 else max(0, n - c["new"]) // page * page
            rows += n - first if n else 0
            pages += -(-n // page) - first // page if n else 0
        return {"bytes": rows * hk * d * es + pages * (hk * 2 * d * qs + 4) + 4 * b, "flops": 2 * rows * hk * d}
    if op == "select":
        pages = sum(_pages(c))
        return {"bytes": pages * (hk * 2 * d * qs + 4) + b * (c["sq"] * h * d * qs + hk * (8 * c["k"] + 4) + 4),
                "flops": pages * c["sq"] * h * 4 * d}
    if op == "sparse":
        keys = sum(max(0, min(n, c["k"]) * page - (page - x % page) % page) for n, x in zip(_pages(c), lens))
        return {"bytes": keys * hk * d * 2 * es + b * c["sq"] * h * (2 * d * qs + 4) + b * hk * (4 * c["k"] + 4),
                "flops": 4 * keys * c["sq"] * h * d}
    if op == "weights":
        return {"bytes": tokens * hk * (d * 2 * es + 8) + b * c["sq"] * h * (2 * d * qs + 4) + 4 * sum(_pages(c)) + 4 * b,
                "flops": 4 * tokens * c["sq"] * h * d}
    if op == "prompt":
        n = [min(c["sq"], x) for x in lens]
        pairs = sum(x * y - x * (x - 1) // 2 for x, y in zip(n, lens))
        return {"bytes": sum(n) * h * (d * qs + 4) + tokens * hk * (d * es + 8) + 4 * sum(_pages(c)), "flops": 2 * pairs * h * d}
    kept = sum(min(x, c["budget"]) for x in lens)
    return {"bytes": kept * hk * (4 * d * es + 8) + tokens * hk * 4 + b * hk * c["budget"] * 4, "flops": tokens * hk}


# ------------------------------------------------------------------------------------------ in 64 bits, by definition

def _sequence(s, pool, i, head, length, table=None):
    """Rows of one sequence and kv head in 64 bits."""
    pages = (s["table"][i] if table is None else table)[:-(-length // s["case"]["page"])].long()
    x = pool[:, :, head].float() if pool.element_size() == 1 else pool[:, :, head]
    return x[pages].reshape(-1, pool.shape[-1])[:length].double()


def _exact_attention(s, i, x, keys, values):
    """Out (sq, group, d), log-sum-exp (group, sq) and the weight of each key, of one sequence and kv head."""
    c = s["case"]
    group, sq = c["h"] // c["hk"], c["sq"]
    q = s["q"][i, :, x * group:(x + 1) * group].double()
    length = keys.shape[0]
    scale = s["scale"] * (float(s["kd"]) if s["kd"] is not None else 1.0)
    score = torch.einsum("sgd,td->gst", q, keys) * scale
    for t in range(sq):
        score[:, t, max(0, length - (sq - 1 - t)):] = -math.inf
    lse = torch.logsumexp(score, -1) if length else torch.full((group, sq), -math.inf, device="cuda", dtype=torch.float64)
    p = torch.where(lse[..., None] > -math.inf, torch.exp(score - lse[..., None]), 0.0)
    out = torch.einsum("gst,td->sgd", p, values) * (float(s["vd"]) if s["vd"] is not None else 1.0)
    return out, torch.where(lse > -math.inf, lse, math.inf), p.sum((0, 1))


def exact(case, seed):
    c, s = case, prepare(case, seed)
    lens, b, hk, page, op = _lens(c), c["b"], c["hk"], c["page"], c["op"]
    group = c["h"] // hk
    if op == "bounds":
        out, pool = s["bounds"].double(), s["k"].float()
        for i, n in enumerate(lens):
            first = (0 if c["new"] == 0 else max(0, n - c["new"])) // page
            ids = s["table"][i, first:-(-n // page)].long()
            if n == 0:
                continue
            x = pool[ids].double()
            out[ids, :, 0], out[ids, :, 1] = x.amin(1), x.amax(1)
            last = x[-1, :n - (-(-n // page) - 1) * page]
            out[ids[-1], :, 0], out[ids[-1], :, 1] = last.amin(0), last.amax(0)
        return out
    if op == "select":
        table = torch.full((b, hk, c["k"]), -1, dtype=torch.int32, device="cuda")
        index, sel = table.clone(), torch.zeros(b, hk, dtype=torch.int32, device="cuda")
        for i, n in enumerate(_pages(c)):
            for x in range(hk):
                if n == 0:
                    continue
                q = s["q"][i, :, x * group:(x + 1) * group].double().reshape(-1, 1, c["d"])
                box = s["bounds"][s["table"][i, :n].long(), x].double()
                value = torch.stack([torch.maximum(y * box[:, 0], y * box[:, 1]).sum(-1) for y in q]).amax(0)
                value[0] = math.inf
                value[min(n - 1, max(0, lens[i] - c["sq"]) // page):] = math.inf
                best = value.sort(descending=True, stable=True).indices[:c["k"]].sort().values
                index[i, x, :len(best)] = best.to(torch.int32)
                table[i, x, :len(best)] = s["table"][i, best]
                sel[i, x] = len(best) * page - (n * page - lens[i])
        return table, sel, index
    if op in ("sparse", "weights"):
        out = torch.zeros(b, c["sq"], c["h"], c["d"], dtype=torch.float64, device="cuda")
        lse = torch.zeros(b, c["h"], c["sq"], dtype=torch.float64, device="cuda")
        w = s["w_out"].double() if op == "weights" else None
        pools = [x.float() if c["kv"] == "e4m3" else x for x in (s["k"], s["v"])]
        for i in range(b):
            for x in range(hk):
                n = lens[i] if op == "weights" else int(s["sel_lens"][i, x])
                table = s["table"][i] if op == "weights" else s["pages"][i, x]
                keys, values = (_sequence(s, y, i, x, n, table) for y in pools)
                out[i, :, x * group:(x + 1) * group], lse[i, x * group:(x + 1) * group], more = _exact_attention(s, i, x, keys, values)
                if w is not None:
                    w[i, x, :n] = s["w"][i, x, :n].double() + more
        return (out, lse) if w is None else (out, lse, w)
    if op == "prompt":
        w, at = s["w_out"].double(), 0
        for i, n in enumerate(lens):
            m = s["n"][i]
            for x in range(hk):
                keys = _sequence(s, s["k"], i, x, n)
                total = s["w"][i, x, :n].double()
                hidden = torch.arange(n, device="cuda")[None, :] > (torch.arange(m, device="cuda") + n - m)[:, None]
                for y in range(x * group, (x + 1) * group):
                    score = s["q"][at:at + m, y].double() @ keys.T * s["scale"] - s["lse"][y, at:at + m].double()[:, None]
                    total += score.masked_fill_(hidden, -math.inf).exp_().sum(0)
                w[i, x, :n] = total
            at += m
        return w
    kept = torch.full((b, hk, c["budget"]), -1, dtype=torch.int32, device="cuda")
    k, v, w = s["k"].clone(), s["v"].clone(), s["w_out"].clone()
    for i, n in enumerate(lens):
        m = min(n, c["budget"])
        rows = torch.arange(m, device="cuda")
        to = s["new_table"][i, rows // page].long()
        for x in range(hk):
            forced = torch.zeros(n, dtype=torch.bool, device="cuda")
            forced[:c["sink"]] = True
            forced[max(0, n - c["recent"]):] = True
            rest = (~forced).nonzero().flatten()
            best = rest[s["w"][i, x, rest].sort(descending=True, stable=True).indices[:max(0, m - int(forced.sum()))]]
            chosen = torch.cat([forced.nonzero().flatten(), best]).sort().values[:m]
            kept[i, x, :m] = chosen.to(torch.int32)
            at = s["table"][i, chosen // page].long()
            k[to, rows % page, x], v[to, rows % page, x] = s["k"][at, chosen % page, x], s["v"][at, chosen % page, x]
            w[i, x, m:n] = 0.0
            w[i, x, :m] = s["w"][i, x, chosen]
    return kept, torch.clamp(s["lens"], max=c["budget"]), k[s["first_new"]:].double(), v[s["first_new"]:].double(), w.double()
