"""The definition of `ops.sample_rows` in float64 on the CPU, by sorting the row.

A kernel's sums differ from these by rounding, and where the number drawn lies that close to a border between two tokens (or a running sum to what top-p asks for) the
token on the other side is right as well.  Weights are whole multiples of 2^-F there, F >= 30 + clz(vocab) capped at 51, each off by half of one and an
exponential in 64 bits; sums of at most `vocab` of them, relative to a largest weight of 1, by vocab * 2^-(F + 1) <= 2^-22 * 2^-8 at the worst vocabulary and
2^-30 * 2^-... at 2^17: `slack` below, with what sums in 64 bits of other orders differ by."""

import math

import torch


def slack(vocab):
    """(F is 39 for 2^22 tokens and 44 for 2^17, which makes the first part 2^-18 and 2^-28.)"""
    bits = min(51, 30 + 32 - vocab.bit_length())
    return vocab * 2.0 ** -(bits + 1) + vocab * 2.0 ** -50


def row(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(id, log-probability, ids that rounding may lead to) of one row; parameters as float32 numbers."""
    as32 = lambda v: float(torch.tensor(v, dtype=torch.float32))
    x, u, temperature, top_p, min_p = x.double(), as32(u), as32(temperature), as32(top_p), as32(min_p)
    x = torch.where(torch.isnan(x), -math.inf, x) + 0.0
    vocab = x.numel()
    order = torch.sort(x, descending=True, stable=True)[1]
    order = order[x[order] > -math.inf]
    if order.numel() == 0:
        return 0, -math.inf, {0}
    v = x[order]
    if not temperature > 0:
        return int(order[0]), 0.0, {int(order[0])}
    u = 0.0 if math.isnan(u) else min(max(u, 0.0), 1.0 - 2.0 ** -24)
    z = torch.where(v == v[0], 0.0, (v - v[0]) / temperature) if not math.isinf(float(v[0])) else torch.where(v == v[0], 0.0, -math.inf).double()
    w = torch.exp(z)
    S = w.cumsum(0)
    n_k = min(top_k, len(w)) if top_k > 0 else len(w)
    tol = slack(vocab) * max(1.0, float(S[-1]) * 2.0 ** -20)

    def first(goal, upto, strict):
        """the first place up to which the sum is (more than, at least) goal"""
        reached = S[:upto] > goal if strict else S[:upto] >= goal
        return int(reached.nonzero()[0]) if bool(reached.any()) else upto - 1
    ends = [n_k]
    if top_p < 1:
        goal = top_p * float(S[n_k - 1])
        ends = [first(goal + d, n_k, False) + 1 for d in (0.0, -tol, tol)]
    if min_p > 0:
        heavy = max(1, int((w >= min_p).sum()))
        ends = [min(e, heavy) for e in ends]
        close = (w / min_p - 1).abs() < 2.0 ** -40        # an exponential may come out on either side of min_p
        if bool(close.any()):
            ends += [min(ends[0], max(1, heavy + d)) for d in (-int(close.sum()), int(close.sum()))]
    ids, answer = set(), None
    for end in ends:
        for d in (0.0, -tol, tol):
            j = first(u * float(S[end - 1]) + d, end, True)
            while j > 0 and w[j] == 0:
                j -= 1
            ids.add(int(order[j]))
            if answer is None:
                answer = int(order[j]), float(z[j]) - math.log(float(S[end - 1]))
    return answer[0], answer[1], ids


def rows(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """([(id, log-probability, allowed ids)] of rows; parameters: numbers or a value per row"""
    of = lambda value, i: value[i] if isinstance(value, (list, tuple)) else value
    return [row(x[i], u[i], of(temperature, i), of(top_k, i), of(top_p, i), of(min_p, i)) for i in range(x.shape[0])]
