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
        length = max(0, min(length, len(row) * page))
        ids = row[:-(-length // page)].long().clamp(0, n_pages - 1)
        return length, [x[ids].reshape(-1, nkv, d)[:length].double() for x in (k_pages, v_pages)]
    for b in range(len(ctx)):
        n, rows = cu[b + 1] - cu[b], slice(cu[b], cu[b + 1])
        owned[rows] = True
        if n == 0:
            continue
        group = [g for g in range(len(prefix_len)) if group_seqs[g] <= b < group_seqs[g + 1]]
        shared, (shared_k, shared_v) = keys(prefix_table[group[0]], prefix_len[group[0]]) if group else keys(page_table[b], 0)
        mine, (own_k, own_v) = keys(page_table[b], ctx[b])
        k, v = torch.cat((shared_k, own_k)), torch.cat((shared_v, own_v))
        limit = (max(ctx[b], 0) - n + 1 + torch.arange(n)).clamp(0, mine) if causal else torch.full((n,), mine)
        limit = (shared + limit).repeat_interleave(rep)[:, None]
        length = shared + mine
        hidden = torch.arange(length) >= limit
        for g in range(nkv):
            at = slice(g * rep, (g + 1) * rep)
            if length == 0:
                out[rows, at] = bound[rows, at] = 0.0
                continue
            qs = q[rows, at].double().reshape(n * rep, d)
            p = torch.nan_to_num(torch.softmax((qs @ k[:, g].T * scale).masked_fill(hidden, -math.inf), 1))
            o, size = p @ v[:, g], p @ v[:, g].abs()
            score = (qs.abs() @ k[:, g].abs().T * scale).masked_fill(hidden, 0.0).amax(1, keepdim=True)
            relative = half + 2 * (d + 8) * 2.0 ** -24 * score + (length / 32 + 192) * 2.0 ** -24
            tiny = 2.0 ** -25 * ((~hidden).double() @ v[:, g].abs() + 1) if q.dtype == torch.float16 else 0.0
            b_rows = (half * o.abs() + (1 + half) * (relative * size + tiny)) * (1 + 2.0 ** -20)
            b_rows[(limit == 0)[:, 0]] = 0.0
            out[rows, at], bound[rows, at] = o.view(n, rep, d), b_rows.view(n, rep, d)
    return out, bound, owned
