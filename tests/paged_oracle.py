"""The definitions of `ops.norm_rotary`, `ops.paged_append` and `ops.paged_attention` in float64 on the CPU, with the magnitudes that bound their rounding."""

import math

import torch


def rotation(cos, sin, ids, d, interleaved):
    """(matrix-free) R and its transpose of rows [tokens, heads, d]: y_i = x_i c_i + x_partner(i) f_i."""
    i = torch.arange(d)
    c, f = torch.ones(len(ids), d, dtype=torch.float64), torch.zeros(len(ids), d, dtype=torch.float64)
    ids = ids.clamp(0, cos.shape[0] - 1)
    cr, sr = cos.double()[ids], sin.double()[ids]
    if interleaved:
        partner = i ^ 1
        c, f = cr.repeat_interleave(2, 1), sr.repeat_interleave(2, 1) * torch.where(i % 2 == 0, -1.0, 1.0)
    else:
        r = cos.shape[1]
        partner = torch.where(i < r, (i + r // 2) % r, i)
        c[:, :r], f[:, :r] = cr, sr * torch.where(i[:r] < r // 2, -1.0, 1.0)

    def apply(x, back=False, magnitude=False):
        by = f[:, partner] if back else f
        a, b = (c.abs(), by.abs()) if magnitude else (c, by)
        return x * a[:, None] + x[..., partner] * b[:, None]
    return apply


def no_rotation(x, back=False, magnitude=False):
    return x


def norm(x, weight, bias, eps, layer_norm):
    """xh, 1 / deviation, xh w + b, and the magnitude of what is summed for the last"""
    x = x.double()
    mean = x.mean(-1, keepdim=True) if layer_norm else torch.zeros_like(x[..., :1])
    centred = x - mean
    rstd = 1.0 / torch.sqrt((centred * centred).mean(-1, keepdim=True) + eps)
    xh = centred * rstd
    w = weight.double()
    b = torch.zeros_like(w) if bias is None else bias.double()
    size = (x.abs() + (x.abs().mean(-1, keepdim=True) if layer_norm else 0)) * rstd * w.abs() + b.abs()
    return xh, rstd, xh * w + b, size


def norm_rotary(x, weight, bias, eps, layer_norm, rotate):
    """(y, magnitude)"""
    _, _, y, size = norm(x, weight, bias, eps, layer_norm)
    return rotate(y), rotate(size, magnitude=True)


def norm_rotary_grad(x, weight, eps, layer_norm, rotate, dy):
    """((dx, magnitude), (dweight, magnitude), (dbias, magnitude))"""
    xh, rstd, _, _ = norm(x, weight, None, eps, layer_norm)
    x = x.double()
    dn, dn_size = rotate(dy.double(), back=True), rotate(dy.double().abs(), back=True, magnitude=True)
    g, g_size = dn * weight.double(), dn_size * weight.double().abs()
    xh_size = (x.abs() + (x.abs().mean(-1, keepdim=True) if layer_norm else 0)) * rstd
    dx = g - xh * (g * xh).mean(-1, keepdim=True)
    size = g_size + xh_size * (g_size * xh_size).mean(-1, keepdim=True)
    if layer_norm:
        dx = dx - g.mean(-1, keepdim=True)
        size = size + g_size.mean(-1, keepdim=True)
    return (dx * rstd, size * rstd), ((dn * xh).sum((0, 1)), (dn_size * xh_size).sum((0, 1))), (dn.sum((0, 1)), dn_size.sum((0, 1)))


def slots(page_table, cu, ctx, page, n_pages, n_tokens):
    """per token (page, row), or None where it is not stored"""
    out = [None] * n_tokens
    for b in range(len(ctx)):
        for t in range(cu[b], cu[b + 1]):
            at = ctx[b] - (cu[b + 1] - t)
            if 0 <= at < page_table.shape[1] * page and 0 <= int(page_table[b, at // page]) < n_pages:
                out[t] = (int(page_table[b, at // page]), at % page)
    return out


def attention(q, k_pages, v_pages, page_table, cu, ctx, causal, scale):
    """(o, bound of its error, whether the token belongs to a sequence) per token.

    Roundings of a result: its own; each probability to the type (half a step, of float16 below 2^-14 at most 2^-25 where the largest is 1 or more); scores,
    whose d products and sums and scaling are each 2^-24 of what is summed, and which enter numerator and denominator; exponentials, sums over the
    keys in chains of at most n / 32, wavefronts, splits and the division, each 2^-24."""
    t, nq, d = q.shape
    half = torch.finfo(q.dtype).eps / 2
    page, nkv = k_pages.shape[1], k_pages.shape[2]
    n_pages = k_pages.shape[0]
    owned = torch.zeros(t, dtype=torch.bool)
    out, bound = torch.full((t, nq, d), math.nan, dtype=torch.float64), torch.full((t, nq, d), math.nan, dtype=torch.float64)
    for b in range(len(ctx)):
        n = cu[b + 1] - cu[b]
        length = max(0, min(ctx[b], page_table.shape[1] * page))
        ids = [min(max(int(i), 0), n_pages - 1) for i in page_table[b, :-(-length // page)]]
        k = k_pages[ids].reshape(-1, nkv, d)[:length].double()
        v = v_pages[ids].reshape(-1, nkv, d)[:length].double()
        for i in range(n):
            limit = max(0, min(length, max(ctx[b], 0) - n + i + 1)) if causal else length
            row = cu[b] + i
            owned[row] = True
            for h in range(nq):
                g = h // (nq // nkv)
                if limit == 0:
                    out[row, h] = bound[row, h] = 0.0
                    continue
                s = k[:limit, g] @ q[row, h].double() * scale
                p = torch.softmax(s, 0)
                o, size = p @ v[:limit, g], p @ v[:limit, g].abs()
                score = float((k[:limit, g].abs() @ q[row, h].double().abs() * scale).max())
                relative = half + 2 * (d + 8) * 2.0 ** -24 * score + (length / 32 + 96) * 2.0 ** -24
                tiny = 2.0 ** -25 * (v[:limit, g].abs().sum(0) + 1) if q.dtype == torch.float16 else 0.0
                out[row, h], bound[row, h] = o, (half * o.abs() + (1 + half) * (relative * size + tiny)) * (1 + 2.0 ** -20)
    return out, bound, owned


def attention_by_sequence(q, k_pages, v_pages, page_table, cu, ctx, causal, scale):
    """What `attention` gives, with the rows of a sequence and KV head together: for calls of thousands of rows."""
    t, nq, d = q.shape
    half = torch.finfo(q.dtype).eps / 2
    page, nkv, n_pages = k_pages.shape[1], k_pages.shape[2], k_pages.shape[0]
    rep = nq // nkv
    owned = torch.zeros(t, dtype=torch.bool)
    out, bound = torch.full((t, nq, d), math.nan, dtype=torch.float64), torch.full((t, nq, d), math.nan, dtype=torch.float64)
    for b in range(len(ctx)):
        n, rows = cu[b + 1] - cu[b], slice(cu[b], cu[b + 1])
        length = max(0, min(ctx[b], page_table.shape[1] * page))
        owned[rows] = True
        if n == 0:
            continue
        ids = page_table[b, :-(-length // page)].long().clamp(0, n_pages - 1)
        k, v = (x[ids].reshape(-1, nkv, d)[:length].double() for x in (k_pages, v_pages))
        limit = (max(ctx[b], 0) - n + 1 + torch.arange(n)).clamp(0, length) if causal else torch.full((n,), length)
        hidden = torch.arange(length) >= limit.repeat_interleave(rep)[:, None]
        for g in range(nkv):
            qs = q[rows, g * rep:(g + 1) * rep].double().reshape(n * rep, d)
            if length == 0:
                out[rows, g * rep:(g + 1) * rep] = bound[rows, g * rep:(g + 1) * rep] = 0.0
                continue
            p = torch.nan_to_num(torch.softmax((qs @ k[:, g].T * scale).masked_fill(hidden, -math.inf), 1))     # rows without keys: zeros
            o, size = p @ v[:, g], p @ v[:, g].abs()
            score = (qs.abs() @ k[:, g].abs().T * scale).masked_fill(hidden, 0.0).amax(1, keepdim=True)
            relative = half + 2 * (d + 8) * 2.0 ** -24 * score + (length / 32 + 96) * 2.0 ** -24
            tiny = 2.0 ** -25 * ((~hidden).double() @ v[:, g].abs() + 1) if q.dtype == torch.float16 else 0.0
            b_rows = (half * o.abs() + (1 + half) * (relative * size + tiny)) * (1 + 2.0 ** -20)
            b_rows[limit.repeat_interleave(rep) == 0] = 0.0
            out[rows, g * rep:(g + 1) * rep], bound[rows, g * rep:(g + 1) * rep] = o.view(n, rep, d), b_rows.view(n, rep, d)
    return out, bound, owned
