"""CPU restatement, in 64 bits, of the operators of a bounded KV cache: page bounds, choice of pages, attention over
listed pages, key weights and eviction.  Plain loops over sequences and heads, from the definitions."""
import math

import torch


def rows(pool, table, head, length):
    """Keys or values of one sequence and kv head: (length, d) float64."""
    page = pool.shape[1]
    n = -(-length // page)
    ids = table[:n].long()
    return pool[:, :, head].float()[ids].reshape(-1, pool.shape[3])[:length].double()


def page_bounds_ref(k_cache, block_table, lens, bounds, new_tokens=None):
    out, page = bounds.clone(), k_cache.shape[1]
    for i, n in enumerate(lens.tolist()):
        first = 0 if new_tokens is None else max(0, n - new_tokens) // page
        for j in range(first, -(-n // page)):
            x = k_cache[int(block_table[i, j])].float()[:min(page, n - j * page)]
            out[int(block_table[i, j]), :, 0] = x.amin(0).to(out.dtype)
            out[int(block_table[i, j]), :, 1] = x.amax(0).to(out.dtype)
    return out


def select_pages_ref(q, bounds, block_table, lens, page, k, sink_pages=1, recent_pages=1):
    b, sq, h, d = q.shape
    hk = bounds.shape[1]
    index = torch.full((b, hk, k), -1, dtype=torch.int32)
    table, sel = index.clone(), torch.zeros(b, hk, dtype=torch.int32)
    for i, length in enumerate(lens.tolist()):
        n = -(-length // page)
        open_from = max(0, length - sq) // page
        forced = torch.tensor([j < sink_pages or j >= n - recent_pages or j >= open_from for j in range(n)], dtype=torch.bool)
        for x in range(hk):
            if n == 0:
                continue
            qs = q[i, :, x * (h // hk):(x + 1) * (h // hk)].double().reshape(-1, 1, d)
            box = bounds[block_table[i, :n].long(), x].double()
            score = torch.where(qs < 0, qs * box[None, :, 0], qs * box[None, :, 1]).sum(-1)
            score = score.amax(0)                       # a NaN wins, as in the definition
            order = sorted(range(n), key=lambda j: (not forced[j], not math.isnan(score[j]),
                                                    0.0 if math.isnan(score[j]) else -float(score[j]), j))
            chosen = sorted(order[:k])
            m = len(chosen)
            index[i, x, :m] = torch.tensor(chosen, dtype=torch.int32)
            table[i, x, :m] = block_table[i, chosen]
            sel[i, x] = m * page - (n * page - length)
    return table, sel, index


def attention_ref(q, keys, values, scale, causal, window_left=-1, sink=None):
    """One sequence and kv head: q (sq, group, d) float64 -> out (sq, group, d), lse (group, sq), key weights."""
    sq, group, _ = q.shape
    n = keys.shape[0]
    score = torch.einsum("sgd,td->gst", q, keys) * scale
    t = torch.arange(n)
    for s in range(sq):
        pos = n - sq + s
        if causal:
            score[:, s, t > pos] = -math.inf
        if window_left >= 0:
            score[:, s, t < pos - window_left] = -math.inf
    full = score if sink is None else torch.cat([score, sink.double()[:, None, None].expand(group, sq, 1)], -1)
    lse = torch.logsumexp(full, -1) if full.shape[-1] else torch.full((group, sq), -math.inf, dtype=torch.float64)
    p = torch.where(lse[..., None] > -math.inf, torch.exp(score - lse[..., None]), 0.0)
    p = torch.where(score == -math.inf, 0.0, p)
    return torch.einsum("gst,td->sgd", p, values), torch.where(lse > -math.inf, lse, math.inf), p.sum((0, 1))


def decode_ref(q, k_cache, v_cache, table, lens, scale, causal=True, window_left=-1, sink=None, k_scale=1.0, v_scale=1.0):
    """table (b, n) with lens (b), or (b, hk, n) with lens (b, hk): out, lse, list of weights[b][hk] (float64)."""
    b, sq, h, d = q.shape
    hk = k_cache.shape[2]
    group = h // hk
    out = torch.zeros(b, sq, h, d, dtype=torch.float64)
    lse = torch.zeros(b, h, sq, dtype=torch.float64)
    weights = []
    for i in range(b):
        weights.append([])
        for x in range(hk):
            t = table[i, x] if table.dim() == 3 else table[i]
            n = int(lens[i, x]) if table.dim() == 3 else int(lens[i])
            hs = slice(x * group, (x + 1) * group)
            o, l, w = attention_ref(q[i, :, hs].double(), rows(k_cache, t, x, n) * k_scale, rows(v_cache, t, x, n) * v_scale, scale, causal,
                                    window_left, None if sink is None else sink[hs])
            out[i, :, hs], lse[i, hs] = o, l
            weights[i].append(w)
    return out, lse, weights


def token_weights_ref(q, k_cache, lse, cu, table, lens, w, scale, causal=True, decay=1.0):
    out = w.double().clone()
    hk = k_cache.shape[2]
    group = q.shape[1] // hk
    for i, n in enumerate(lens.tolist()):
        a, e = int(cu[i]), int(cu[i + 1])
        for x in range(hk):
            keys = rows(k_cache, table[i], x, n)
            total = w[i, x, :n].double() * decay
            for y in range(x * group, (x + 1) * group):
                p = torch.exp(q[a:e, y].double() @ keys.T * scale - lse[y, a:e].double()[:, None])
                if causal:
                    p[torch.arange(n)[None, :] > (torch.arange(e - a) + n - (e - a))[:, None]] = 0.0
                total = total + p.sum(0)
            out[i, x, :n] = total
    return out


def evict_ref(k_cache, v_cache, table, lens, w, budget, sink, recent, new_table=None, w_out=None):
    """(kept, new lens, k, v, weights)."""
    b, hk, page = table.shape[0], k_cache.shape[2], k_cache.shape[1]
    kept = torch.full((b, hk, budget), -1, dtype=torch.int32)
    k, v, out = k_cache.clone(), v_cache.clone(), (w if w_out is None else w_out).clone()
    dst = table if new_table is None else new_table
    for i, n in enumerate(lens.tolist()):
        m = min(n, budget)
        for x in range(hk):
            forced = [t for t in range(n) if t < sink or t >= n - recent]
            rest = [t for t in range(n) if not (t < sink or t >= n - recent)]
            value = w[i, x].tolist()
            rest.sort(key=lambda t: (not math.isnan(value[t]), 0.0 if math.isnan(value[t]) else -value[t], t))
            chosen = list(range(n)) if n <= budget else sorted(forced + rest[:m - len(forced)])
            for to, t in enumerate(chosen):
                kept[i, x, to] = t
                sp, dp = int(table[i, t // page]), int(dst[i, to // page])
                k[dp, to % page, x], v[dp, to % page, x] = k_cache[sp, t % page, x], v_cache[sp, t % page, x]
            out[i, x, m:n] = 0.0
            out[i, x, :m] = w[i, x, chosen]
    return kept, torch.clamp(lens, max=budget), k, v, out
