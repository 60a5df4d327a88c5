"""The definition of `ops.paged_step`, page by page and token by token, on lists."""


def step(new, lengths, table, free, count, status, page, tokens, max_ctx=None, offset=None):
    """(ctx_len, table, free, count, status, cu, positions, slots, sequences, last); lists, of which none is changed"""
    table, free, room = [list(r) for r in table], list(free), len(table[0]) * page
    max_ctx = room if max_ctx is None else max_ctx
    lengths = [min(max(n, 0), room) for n in lengths]
    count = min(max(count, 0), len(free))
    for b, n in enumerate(new):
        if n < 0:
            for i in reversed(range(-(-lengths[b] // page))):
                if count < len(free):
                    free[count] = table[b][i]
                    count += 1
            lengths[b] = 0
    new = [max(n, 0) for n in new]
    too_long = any(n > 0 and length + n > max_ctx for n, length in zip(new, lengths))
    wanted = sum(-(-(length + n) // page) - -(-length // page) for n, length in zip(new, lengths) if not (n > 0 and length + n > max_ctx))
    now = (1 if wanted > count else 0) | (2 if too_long else 0) | (4 if sum(new) > tokens else 0)
    if now:
        new = [0] * len(new)
    positions, slots, sequences, last, cu, ctx = [], [], [], [], [0], []
    for b, n in enumerate(new):
        for at in range(lengths[b], lengths[b] + n):
            if at % page == 0:
                count -= 1
                table[b][at // page] = free[count]
            positions.append(at + (offset[b] if offset else 0))
            slots.append(table[b][at // page] * page + at % page)
            sequences.append(b)
        last.append(len(positions) - 1 if n else 0)
        cu.append(len(positions))
        ctx.append(lengths[b] + n)
    rest = tokens - len(positions)
    return ctx, table, free, count, status | now, cu, positions + [0] * rest, slots + [-1] * rest, sequences + [0] * rest, last
