"""The definition of `ops.paged_prefix_attention` in float64 on the CPU, with a bound of its rounding: that of paged_oracle.attention_by_sequence over the keys of prefix
and sequence together, and one more chain of partial results."""

import math

import torch


def attention(q, k_pages, v_pages, page_table, cu, ctx, prefix_table, prefix_len, group_seqs, causal, scale):
    """(o, bound of its error, whether the token belongs to a sequence) per token"""
    t, nq, d = q.shape
    half = torch.finfo(q.dtype).eps / 2
    page, nkv, n_pages = k_pages.shape[1], k_pages.shape[2], k_pages.shape[0]
    rep = nq // nkv
    owned = torch.zeros(t, dtype=torch.bool)
    out, bound = torch.full((t, nq, d), math.nan, dtype=torch.float64), torch.full((t, nq, d), math.nan, dtype=torch.float64)

    def keys(row, length):
        """(length, K, V, |K|, |V|), each [KV head, key, feature]"""
        length = max(0, min(length, len(row) * page))
        ids = row[:-(-length // page)].long().clamp(0, n_pages - 1)
        k, v = (x[ids].reshape(-1, nkv, d)[:length].double().transpose(0, 1).contiguous() for x in (k_pages, v_pages))
        return length, k, v, k.abs(), v.abs()
    group = None
    for b in range(len(ctx)):
        n, rows = cu[b + 1] - cu[b], slice(cu[b], cu[b + 1])
        owned[rows] = True
        if n == 0:
            continue
        of = [g for g in range(len(prefix_len)) if group_seqs[g] <= b < group_seqs[g + 1]]
        if b == 0 or of != group:                          # (sequences of a group are neighbours)
            group = of
            prefix = keys(prefix_table[of[0]], prefix_len[of[0]]) if of else keys(page_table[b], 0)
        own = keys(page_table[b], ctx[b])
        shared, mine = prefix[0], own[0]
        limit = (max(ctx[b], 0) - n + 1 + torch.arange(n)).clamp(0, mine) if causal else torch.full((n,), mine)
        limit = (shared + limit).repeat_interleave(rep)[:, None]
        length = shared + mine
        hidden = torch.arange(length) >= limit
        if length == 0:
            out[rows] = bound[rows] = 0.0
            continue
        # all heads together, [KV head, row, ...]
        qs = q[rows].double().view(n, nkv, rep, d).transpose(0, 1).reshape(nkv, n * rep, d)
        scores = lambda x, i: torch.cat([torch.bmm(x, part[i].transpose(1, 2)) for part in (prefix, own)], 2) * scale
        weighted = lambda p, i: torch.bmm(p[:, :, :shared], prefix[i]) + torch.bmm(p[:, :, shared:], own[i])
        p = torch.nan_to_num(torch.softmax(scores(qs, 1).masked_fill(hidden, -math.inf), 2))
        o, size = weighted(p, 2), weighted(p, 4)
        score = scores(qs.abs(), 3).masked_fill(hidden, 0.0).amax(2, keepdim=True)
        relative = half + 2 * (d + 8) * 2.0 ** -24 * score + (length / 32 + 192) * 2.0 ** -24
        tiny = 2.0 ** -25 * (weighted((~hidden).double().expand(nkv, -1, -1), 4) + 1) if q.dtype == torch.float16 else 0.0
        b_rows = (half * o.abs() + (1 + half) * (relative * size + tiny)) * (1 + 2.0 ** -20)
        b_rows.masked_fill_((limit == 0), 0.0)
        heads = lambda x: x.view(nkv, n, rep, d).transpose(0, 1).reshape(n, nq, d)
        out[rows], bound[rows] = heads(o), heads(b_rows)
    return out, bound, owned
