"""Operators of the loop that samples several answers to each of a few prompts, as a server runs it without the host between its steps:

  sample_rows              `ops.sample_rows`: a token of every row of logits, by temperature, top-k, top-p and min-p, from given random numbers
  paged_step               `ops.paged_step`: pages, positions and slots of the next step's tokens, from lengths that lie on the GPU
  paged_prefix_attention   `ops.paged_prefix_attention`: attention over a paged cache for sequences that share a long prefix, group by group

With `own` false, `run` computes them in their plain form, in elementary torch operations; with `own` true it makes the calls a user makes.
"""

import math
import random

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}


# ---- cases ---------------------------------------------------------------------------------------------------------
def sample_rows(name=None, *, rows, vocab, dtype, temperature, top_k=0, top_p=1.0, min_p=0.0, mixed=False, masked=0.0, spread=2.5):
    """mixed: parameters of each row's own around the given ones, some rows greedy.  masked: that share of the vocabulary is not allowed (-inf).  spread: standard
    deviation of the logits."""
    return _named(dict(op="sample_rows", rows=rows, vocab=vocab, dtype=dtype, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p, mixed=mixed,
                       masked=masked, spread=spread), name)


def paged_step(name=None, *, batch, new_min, new_max, ctx_max, page, ends=0.0, idle=0.0):
    """new_min .. new_max new tokens of each sequence, which then has up to ctx_max; that share of the sequences ends, another brings nothing."""
    return _named(dict(op="paged_step", batch=batch, new_min=new_min, new_max=new_max, ctx_max=ctx_max, page=page, ends=ends, idle=idle), name)


def paged_prefix_attention(name=None, *, groups, batch, new_min, new_max, own_max, prefix_min, prefix_max, heads, kv_heads, dim, page, dtype):
    """batch sequences in groups of about one size; new_min .. new_max new tokens each, up to own_max keys of their own with them."""
    return _named(dict(op="paged_prefix_attention", groups=groups, batch=batch, new_min=new_min, new_max=new_max, own_max=own_max, prefix_min=prefix_min,
                       prefix_max=prefix_max, heads=heads, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype), name)


def _named(case, name):
    if name is not None:
        case["name"] = name
    return case


def listed():
    return [
        # One user's next token, as chat front ends ask for it.
        sample_rows("sample_1_bf16", rows=1, vocab=32000, dtype="bfloat16", temperature=0.75, top_k=50, top_p=0.9375),
        # A batch that decodes with an 8B-class decoder's vocabulary, nucleus sampling.
        sample_rows("sample_32_nucleus", rows=32, vocab=128256, dtype="bfloat16", temperature=1.0, top_p=0.9),
        # Users with parameters of their own, a vocabulary of odd size, float32 logits.
        sample_rows("sample_7_mixed_f32", rows=7, vocab=49999, dtype="float32", temperature=0.9, top_k=200, top_p=0.95, min_p=0.01, mixed=True),
        # Answers that have to follow a grammar, float16, no truncation but min-p.
        sample_rows("sample_60_masked_f16", rows=60, vocab=64000, dtype="float16", temperature=1.25, min_p=0.05, masked=0.75),
        # First tokens of many answers at once, as rollouts for training take them.
        sample_rows("sample_256_mixed", rows=256, vocab=128256, dtype="bfloat16", temperature=1.0, top_k=1000, top_p=0.95, mixed=True),
        # The next token of 32 users.
        paged_step("step_decode_32", batch=32, new_min=1, new_max=1, ctx_max=4096, page=64),
        # Many users, some of whom are done and some of whom wait.
        paged_step("step_decode_1000", batch=1000, new_min=1, new_max=1, ctx_max=2048, page=16, ends=0.05, idle=0.1),
        # Prompts and chunks of prompts, beside sequences that have nothing to add.
        paged_step("step_prompts_65k", batch=48, new_min=500, new_max=2048, ctx_max=8192, page=64, idle=0.1),
        # Eight answers to one prompt.
        paged_prefix_attention("prefix_8x1500", groups=1, batch=8, new_min=1, new_max=1, own_max=200, prefix_min=1500, prefix_max=1500, heads=32, kv_heads=8,
                               dim=128, page=16, dtype="bfloat16"),
        # Many answers to a few prompts, float16 with narrow heads.
        paged_prefix_attention("prefix_4_groups_f16", groups=4, batch=50, new_min=1, new_max=1, own_max=900, prefix_min=700, prefix_max=6000, heads=16,
                               kv_heads=4, dim=64, page=32, dtype="float16"),
        # Users of one long system prompt and document, drafts of a few tokens each.
        paged_prefix_attention("prefix_drafts_32x8192", groups=1, batch=32, new_min=3, new_max=7, own_max=1000, prefix_min=8192, prefix_max=8192, heads=32,
                               kv_heads=8, dim=128, page=64, dtype="bfloat16"),
        # Many answers to one long document.
        paged_prefix_attention("prefix_128x16384", groups=1, batch=128, new_min=1, new_max=1, own_max=1024, prefix_min=16384, prefix_max=16384, heads=32,
                               kv_heads=8, dim=128, page=64, dtype="bfloat16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_sample(rng):
    return sample_rows(rows=_log_int(rng, 1, 256), vocab=_log_int(rng, 500, 160000), dtype=rng.choice(("bfloat16", "bfloat16", "float16", "float32")),
                       temperature=rng.choice((0.5, 0.75, 1.0, 1.0, 1.5)), top_k=rng.choice((0, 0, _log_int(rng, 1, 5000))),
                       top_p=rng.choice((1.0, 1.0, round(rng.uniform(0.3, 0.99), 3))), min_p=rng.choice((0.0, 0.0, round(rng.uniform(0.001, 0.3), 3))),
                       mixed=rng.random() < 0.4, masked=rng.choice((0.0, 0.0, round(rng.uniform(0.1, 0.99), 2))), spread=rng.choice((1.0, 2.5, 2.5, 4.0)))


def _draw_step(rng):
    new_max = 1 if rng.random() < 0.5 else _log_int(rng, 2, 2048)
    batch = _log_int(rng, 1, min(2048, 65536 // new_max))
    return paged_step(batch=batch, new_min=rng.randint(1, new_max), new_max=new_max, ctx_max=rng.randint(new_max, 16384), page=rng.choice((16, 32, 48, 64, 128, 256)),
                      ends=rng.choice((0.0, 0.0, round(rng.uniform(0.0, 0.5), 2))), idle=rng.choice((0.0, round(rng.uniform(0.0, 0.5), 2))))


_HEADS = ((4, 4), (8, 8), (12, 12), (16, 16), (16, 4), (32, 8), (12, 3), (32, 4), (20, 4))


def _draw_prefix(rng):
    heads, kv_heads = rng.choice(_HEADS)
    batch = _log_int(rng, 2, 160)
    new_max = 1 if rng.random() < 0.6 else _log_int(rng, 2, max(2, 1024 // batch))
    prefix_max = _log_int(rng, 30, 20000)
    return paged_prefix_attention(groups=_log_int(rng, 1, max(1, batch // 2)), batch=batch, new_min=rng.randint(1, new_max), new_max=new_max,
                                  own_max=max(new_max, _log_int(rng, 2, 2000)), prefix_min=rng.randint(1, prefix_max), prefix_max=prefix_max, heads=heads,
                                  kv_heads=kv_heads, dim=rng.choice((32, 64, 64, 96, 128, 128)), page=rng.choice((16, 16, 32, 48, 64, 64, 128, 256)),
                                  dtype=rng.choice(("bfloat16", "bfloat16", "float16")))


def draw(rng: random.Random):
    """Sizes over the whole range of the listed cases; no more work than the largest of each operator."""
    most = {c["op"]: work(c)["bytes"] for c in listed()}
    flops = max(work(c)["flops"] for c in listed())
    while True:
        case = rng.choice((_draw_sample, _draw_step, _draw_prefix, _draw_prefix))(rng)
        if case["op"] == "paged_step" and sum(max(n, 0) for n in _step_lengths(case)[0]) > 70000:
            continue
        if work(case)["bytes"] <= most[case["op"]] * (2 if case["op"] == "paged_step" else 1) and work(case)["flops"] <= flops:
            return case


def _seeded(case, *names):
    return random.Random(" ".join(str(case[n]) for n in names))


def _step_lengths(case):
    """(new tokens, -1: ends; cached tokens before) per sequence; of the case's values alone."""
    rng = _seeded(case, "batch", "new_min", "new_max", "ctx_max", "ends", "idle")
    new, lengths = [], []
    for _ in range(case["batch"]):
        what = rng.random()
        n = rng.randint(case["new_min"], case["new_max"])
        new.append(-1 if what < case["ends"] else 0 if what < case["ends"] + case["idle"] else n)
        lengths.append(rng.randint(0, case["ctx_max"] - n))
    if max(new) < 1:
        new[0] = case["new_min"]
    return new, lengths


def _prefix_lengths(case):
    """(sequences per group, prefix length per group, new tokens and own keys with them per sequence); of the case's values alone."""
    rng = _seeded(case, "groups", "batch", "new_min", "new_max", "own_max", "prefix_min", "prefix_max")
    sizes = [case["batch"] // case["groups"]] * case["groups"]
    for i in range(case["batch"] - sum(sizes)):
        sizes[i] += 1
    if case["groups"] > 1:                                 # one sequence more here, one less there
        sizes[0], sizes[-1] = sizes[0] + 1, sizes[-1] - 1
    new = [rng.randint(case["new_min"], case["new_max"]) for _ in range(case["batch"])]
    return sizes, [rng.randint(case["prefix_min"], case["prefix_max"]) for _ in sizes], new, [rng.randint(n, case["own_max"]) for n in new]


def _pages(case, length):
    return -(-length // case["page"])


def work(case):
    """Inputs read once, outputs written once; products and sums of the attention, a few operations an element elsewhere."""
    if case["op"] == "sample_rows":
        elements = case["rows"] * case["vocab"]
        return {"bytes": elements * DTYPES[case["dtype"]].itemsize + 32 * case["rows"], "flops": 4 * elements}
    if case["op"] == "paged_step":
        new, lengths = _step_lengths(case)
        taken = sum(_pages(case, length + n) - _pages(case, length) for n, length in zip(new, lengths) if n > 0)
        tokens = sum(n for n in new if n > 0)
        # new, lengths, ctx_len, cu_seqlens, last; pages taken and given back; positions, slots and sequences
        return {"bytes": 24 * case["batch"] + 8 * taken + 8 * sum(_pages(case, length) for n, length in zip(new, lengths) if n < 0) + 24 * tokens,
                "flops": 10 * case["batch"] + 10 * tokens}
    sizes, prefix, new, keys = _prefix_lengths(case)
    e, d, first, pairs = DTYPES[case["dtype"]].itemsize, case["dim"], 0, 0
    for size, shared in zip(sizes, prefix):
        for n, length in zip(new[first:first + size], keys[first:first + size]):
            pairs += n * (shared + length) - n * (n - 1) // 2
        first += size
    return {"bytes": 2 * sum(new) * case["heads"] * d * e + 2 * (sum(prefix) + sum(keys)) * case["kv_heads"] * d * e
            + 4 * sum(_pages(case, length) for length in prefix + keys), "flops": 4 * d * case["heads"] * pairs}


# ---- inputs --------------------------------------------------------------------------------------------------------
def _randn(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device=DEVICE) * scale).to(dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _prepare_sample_rows(case, gen, dtype):
    rows, vocab = case["rows"], case["vocab"]
    logits = torch.randn(rows, vocab, generator=gen, device=DEVICE) * case["spread"]
    likely = torch.randint(0, vocab, (rows, 3), generator=gen, device=DEVICE)            # a few tokens that the text asks for
    logits.scatter_add_(1, likely, torch.rand(rows, 3, generator=gen, device=DEVICE) * 2.0 * case["spread"])
    if case["masked"] > 0:
        hidden = torch.rand(rows, vocab, generator=gen, device=DEVICE) < case["masked"]
        hidden.scatter_(1, likely[:, :1], False)
        logits.masked_fill_(hidden, -math.inf)
    state = dict(logits=logits.to(dtype), uniforms=torch.rand(rows, generator=gen, device=DEVICE))
    for name in ("temperature", "top_k", "top_p", "min_p"):
        state[name] = case[name]
    if case["mixed"]:
        def around(value, factor, kind):
            return (value * torch.exp2((torch.rand(rows, generator=gen, device=DEVICE) * 2 - 1) * factor)).to(kind)
        state["temperature"] = around(case["temperature"], 0.5, torch.float32)
        state["temperature"][torch.rand(rows, generator=gen, device=DEVICE) < 0.1] = 0.0  # greedy
        state["top_k"] = around(max(case["top_k"], 20), 3.0, torch.int32)
        state["top_p"] = 1.0 - around(max(1.0 - case["top_p"], 0.02), 2.0, torch.float32)
        state["min_p"] = around(max(case["min_p"], 0.002), 2.0, torch.float32)
    return state


def _prepare_paged_step(case, gen):
    new, lengths = _step_lengths(case)
    width = _pages(case, case["ctx_max"])
    held = [_pages(case, length) for length in lengths]
    taken = sum(_pages(case, length + n) - h for n, length, h in zip(new, lengths, held) if n > 0)
    n_pages = sum(held) + taken + 5
    order = torch.randperm(n_pages, generator=gen, device=DEVICE).to(torch.int32)
    table, at = torch.zeros(len(new), width, dtype=torch.int32, device=DEVICE), 0
    columns, h = torch.arange(width, device=DEVICE)[None, :], _ints(held).long()
    index = (h.cumsum(0) - h)[:, None] + columns
    table = torch.where(columns < h[:, None], order[index.clamp(max=n_pages - 1)], 0).to(torch.int32).contiguous()
    at = sum(held)
    free = torch.zeros(n_pages, dtype=torch.int32, device=DEVICE)
    free[:n_pages - at] = order[at:]
    return dict(new=_ints(new), lengths=_ints(lengths), page_table=table, free_pages=free, state=_ints([n_pages - at, 0]), tokens=sum(n for n in new if n > 0),
                ctx_len=_ints([0] * len(new)), state_out=_ints([0, 0]))


def _prepare_prefix(case, gen, dtype):
    sizes, prefix, new, keys = _prefix_lengths(case)
    nq, nkv, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    needed = [_pages(case, length) for length in prefix + keys]
    n_pages = sum(needed) + 3
    order = torch.randperm(n_pages, generator=gen, device=DEVICE).to(torch.int32)
    rows, used = [], 0
    for n in needed:
        rows.append(order[used:used + n])
        used += n

    def table(pieces):
        out = torch.zeros(len(pieces), max(len(p) for p in pieces) + 1, dtype=torch.int32, device=DEVICE)
        for i, p in enumerate(pieces):
            out[i, :len(p)] = p
        return out
    k_pages, v_pages = (_randn(gen, (n_pages, nkv, page, d), dtype).transpose(1, 2) for _ in range(2))   # a page's keys of one head lie together
    tokens = sum(new)
    state = dict(k_pages=k_pages, v_pages=v_pages, page_table=table(rows[len(sizes):]), prefix_table=table(rows[:len(sizes)]), sizes=sizes, prefix=prefix, new=new,
                 keys=keys, prefix_len=_ints(prefix), ctx_len=_ints(keys), cu_seqlens=_ints([0] + [sum(new[:i + 1]) for i in range(len(new))]),
                 group_seqs=_ints([0] + [sum(sizes[:i + 1]) for i in range(len(sizes))]), q=_randn(gen, (tokens, nq, d), dtype, 1.5))
    if own:
        from scaling_amd import ops
        state["workspace"] = ops.paged_prefix_workspace(len(new), len(sizes), tokens, nq, nkv, d, torch.device(DEVICE, torch.cuda.current_device()))
    return state


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    if case["op"] == "paged_step":
        state = _prepare_paged_step(case, gen)
    else:
        state = (_prepare_sample_rows if case["op"] == "sample_rows" else _prepare_prefix)(case, gen, DTYPES[case["dtype"]])
    state["case"] = case
    return state


# ---- one pass ------------------------------------------------------------------------------------------------------
def run(state):
    return (_RUN_OWN if own else _RUN_PLAIN)[state["case"]["op"]](state)


def _own_sample_rows(s):
    from scaling_amd import ops
    return ops.sample_rows(s["logits"], s["uniforms"], s["temperature"], s["top_k"], s["top_p"], s["min_p"], return_logprobs=True)


def _own_paged_step(s):
    from scaling_amd import ops
    step = ops.paged_step(s["new"], s["lengths"], s["page_table"], s["free_pages"], s["state"], s["case"]["page"], s["tokens"], ctx_len=s["ctx_len"],
                          state_out=s["state_out"])
    return step.cu_seqlens, s["ctx_len"], step.position_ids, step.slots, step.sequences, step.last, s["page_table"], s["free_pages"], s["state_out"]


def _own_prefix(s):
    from scaling_amd import ops
    return ops.paged_prefix_attention(s["q"], s["k_pages"], s["v_pages"], s["page_table"], s["cu_seqlens"], s["ctx_len"], s["prefix_table"], s["prefix_len"],
                                      s["group_seqs"], max_q_len=max(s["new"]), workspace=s["workspace"])


_RUN_OWN = {"sample_rows": _own_sample_rows, "paged_step": _own_paged_step, "paged_prefix_attention": _own_prefix}


# ---- plain form ----------------------------------------------------------------------------------------------------
def _column(value, rows, dtype):
    """A parameter of all rows, or of each, as [rows, 1]."""
    if torch.is_tensor(value):
        return value.to(dtype)[:, None]
    return torch.full((rows, 1), value, dtype=torch.float32 if dtype.is_floating_point else dtype, device=DEVICE).to(dtype)


@torch.no_grad()
def _plain_sample_rows(s):
    """Weights exp((x - max) / T) of the row in descending order (equal ones by index); top-k, top-p and min-p each keep the first so many; of those the first
    whose running sum exceeds u times the whole.  In 64 bits: u lies next to a border now and then."""
    rows, vocab = s["logits"].shape
    value, index = torch.sort(s["logits"].float(), dim=1, descending=True, stable=True)
    temperature = _column(s["temperature"], rows, torch.float64)
    greedy = temperature <= 0
    weight = torch.exp((value.double() - value[:, :1].double()) / torch.where(greedy, 1.0, temperature))
    rank = torch.arange(vocab, device=DEVICE)[None, :]
    top_k = _column(s["top_k"], rows, torch.int64)
    weight = torch.where((rank < torch.where(top_k > 0, top_k, vocab)) & ~(greedy & (rank > 0)), weight, 0.0)
    total = weight.cumsum(dim=1)
    before = total - weight
    top_p = _column(s["top_p"], rows, torch.float64)
    kept = (rank == 0) | (((top_p >= 1) | (before < top_p * total[:, -1:])) & (weight >= _column(s["min_p"], rows, torch.float64)) & (weight > 0))
    weight = torch.where(kept, weight, 0.0)
    total = weight.cumsum(dim=1)
    at = (total <= s["uniforms"].double()[:, None] * total[:, -1:]).sum(dim=1, keepdim=True)
    at = torch.minimum(at, (weight > 0).sum(dim=1, keepdim=True) - 1)
    chosen = weight.gather(1, at) / total[:, -1:]
    return index.gather(1, at)[:, 0], chosen.log().float()[:, 0]


@torch.no_grad()
def _plain_paged_step(s):
    page, batch, width, tokens = s["case"]["page"], s["new"].numel(), s["page_table"].shape[1], s["tokens"]
    new, lengths, free, table = s["new"].long(), s["lengths"].long(), s["free_pages"], s["page_table"]
    ends, count = new < 0, s["state"][0].long()
    columns = torch.arange(width, device=DEVICE)[None, :]
    # pages of the sequences that end go onto the stack, sequence by sequence, last page first
    given = torch.where(ends, (lengths + page - 1) // page, 0)
    slot = count + given.cumsum(0)[:, None] - 1 - columns
    spare = torch.cat((free, free.new_zeros(1)))
    spare.scatter_(0, torch.where(columns < given[:, None], slot, free.numel()).flatten(), table.flatten())
    free.copy_(spare[:-1])
    count = count + given.sum()
    before = torch.where(ends, 0, lengths)
    new = new.clamp(min=0)
    after = before + new
    held = (before + page - 1) // page
    wanted = (after + page - 1) // page - held
    fits = (wanted.sum() <= count) & (after.max() <= width * page) & (new.sum() <= tokens)
    status = torch.where(wanted.sum() > count, 1, 0) + torch.where(after.max() > width * page, 2, 0) + torch.where(new.sum() > tokens, 4, 0)
    new, wanted, after = torch.where(fits, new, 0), torch.where(fits, wanted, 0), torch.where(fits, after, before)
    # taken from the top, sequence by sequence
    source = count - 1 - ((wanted.cumsum(0) - wanted)[:, None] + columns - held[:, None])
    table.copy_(torch.where((columns >= held[:, None]) & (columns < (held + wanted)[:, None]), free[source.clamp(0, free.numel() - 1)], table))
    upto = new.cumsum(0)
    cu = torch.cat((upto.new_zeros(1), upto))
    row = torch.arange(tokens, device=DEVICE)
    owned = row < cu[-1]
    sequence = torch.where(owned, (row[:, None] >= upto[None, :]).sum(dim=1), 0)
    position = torch.where(owned, after[sequence] - cu[sequence + 1] + row, 0)
    slots = torch.where(owned, table[sequence, position // page].long() * page + position % page, -1)
    last = torch.where(new > 0, upto - 1, 0)
    s["ctx_len"].copy_(after)
    s["state_out"].copy_(torch.stack((count - wanted.sum(), s["state"][1].long() | status)))
    return cu.to(torch.int32), s["ctx_len"], position, slots, sequence, last, table, free, s["state_out"]


@torch.no_grad()
def _plain_prefix(s):
    case = s["case"]
    nq, nkv, d = case["heads"], case["kv_heads"], case["dim"]
    n_rep, scale = nq // nkv, 1.0 / math.sqrt(d)
    out, token, b = torch.empty_like(s["q"]), 0, 0
    for g, size in enumerate(s["sizes"]):
        ids = s["prefix_table"][g, :_pages(case, s["prefix"][g])].long()
        shared = [s[name][ids].flatten(0, 1)[:s["prefix"][g]].float().transpose(0, 1) for name in ("k_pages", "v_pages")]      # [nkv, length, d]
        for _ in range(size):
            n, length = s["new"][b], s["keys"][b]
            ids = s["page_table"][b, :_pages(case, length)].long()
            k, v = (torch.cat((x, s[name][ids].flatten(0, 1)[:length].float().transpose(0, 1)), dim=1) for x, name in zip(shared, ("k_pages", "v_pages")))
            q = s["q"][token:token + n].float().view(n, nkv, n_rep, d).permute(1, 2, 0, 3)                                      # [nkv, n_rep, n, d]
            sees = s["prefix"][g] + torch.arange(length - n, length, device=DEVICE)
            hidden = torch.arange(s["prefix"][g] + length, device=DEVICE)[None, :] > sees[:, None]
            for h in range(nkv):
                scores = torch.matmul(q[h].reshape(n_rep * n, d), k[h].t()).view(n_rep, n, -1) * scale
                scores.masked_fill_(hidden, -math.inf)
                scores = torch.exp(scores - scores.amax(dim=-1, keepdim=True))
                o = torch.matmul(scores.view(n_rep * n, -1), v[h]).view(n_rep, n, d) / scores.sum(dim=-1, keepdim=True)
                out[token:token + n, h * n_rep:(h + 1) * n_rep] = o.transpose(0, 1).to(out.dtype)
            token, b = token + n, b + 1
    return out


_RUN_PLAIN = {"sample_rows": _plain_sample_rows, "paged_step": _plain_paged_step, "paged_prefix_attention": _plain_prefix}


# ---- the definition, in float64 ------------------------------------------------------------------------------------
def _exact_sample_rows(s):
    """Row by row over its distinct values, largest first: each stands for `count` tokens of one weight."""
    def of(value, row):
        return float(value[row]) if torch.is_tensor(value) else float(torch.tensor(value, dtype=torch.float32))
    ids, logprobs = [], []
    for row in range(s["logits"].shape[0]):
        x = s["logits"][row].double()
        values, counts = torch.unique(x[x > -math.inf], return_counts=True)
        values, counts = values.flip(0), counts.flip(0).double()
        temperature, k = of(s["temperature"], row), int(of(s["top_k"], row))
        if temperature <= 0:
            temperature, k = 1.0, 1
        if k > 0:                                          # whole values, and what is left of the last one
            counts = torch.minimum(counts, (k - (counts.cumsum(0) - counts)).clamp(min=0))
        weights = torch.exp((values - values[0]) / temperature)
        p = of(s["top_p"], row)
        if p < 1:                                          # the fewest tokens with p of the weight: n of a value w behind a sum S make S + n w >= goal
            goal = p * (weights * counts).sum()
            in_front = (weights * counts).cumsum(0) - weights * counts
            counts = torch.minimum(counts, torch.ceil((goal - in_front) / weights).clamp(min=0))
            counts[0] = counts[0].clamp(min=1)
        keep = weights >= of(s["min_p"], row)
        keep[0] = True
        counts = torch.where(keep, counts, 0.0)
        mass = weights * counts
        goal = s["uniforms"][row].double() * mass.sum()
        j = int((mass.cumsum(0) <= goal).sum().clamp(max=int((mass > 0).sum()) - 1))
        nth = int(((goal - (mass.cumsum(0)[j] - mass[j])) / weights[j]).floor().clamp(0, counts[j] - 1))
        ids.append((x == values[j]).nonzero()[nth, 0])
        logprobs.append(torch.log(weights[j] / mass.sum()))
    return torch.stack(ids), torch.stack(logprobs)


def _exact_paged_step(s):
    """In Python, page by page and token by token."""
    page, (new, lengths), table = s["case"]["page"], _step_lengths(s["case"]), s["page_table"].tolist()
    free, (count, status) = s["free_pages"].tolist(), s["state"].tolist()
    for b, n in enumerate(new):
        if n < 0:
            for i in reversed(range(-(-lengths[b] // page))):
                free[count] = table[b][i]
                count += 1
    cu, after, position, slots, sequence, last = [0], [], [], [], [], []
    for b, n in enumerate(new):
        length = 0 if n < 0 else lengths[b]
        for at in range(length, length + max(n, 0)):
            if at % page == 0:
                count -= 1
                table[b][at // page] = free[count]
            position.append(at)
            slots.append(table[b][at // page] * page + at % page)
            sequence.append(b)
        last.append(len(position) - 1 if n > 0 else 0)
        cu.append(len(position))
        after.append(length + max(n, 0))
    longs = [torch.tensor(x, dtype=torch.int64, device=DEVICE) for x in (position, slots, sequence, last)]
    return _ints(cu), _ints(after), *longs, _ints(table), _ints(free), _ints([count, status])


def _exact_prefix(s):
    case, start, b, parts = s["case"], 0, 0, []
    n_rep = case["heads"] // case["kv_heads"]

    def keys_of(name, row, length):
        return torch.cat([s[name][i] for i in row[:_pages(case, length)]])[:length].double()
    own_rows, shared_rows = s["page_table"].tolist(), s["prefix_table"].tolist()
    for g, size in enumerate(s["sizes"]):
        shared_k, shared_v = (keys_of(name, shared_rows[g], s["prefix"][g]) for name in ("k_pages", "v_pages"))
        for _ in range(size):
            n, length = s["new"][b], s["keys"][b]
            own_k, own_v = (keys_of(name, own_rows[b], length) for name in ("k_pages", "v_pages"))
            q, heads = s["q"][start:start + n].double(), []
            mask = torch.full((n, length), -math.inf, dtype=torch.float64, device=DEVICE).triu(length - n + 1)
            for h in range(case["heads"]):
                kv = h // n_rep
                logits = torch.cat((q[:, h] @ shared_k[:, kv].t().contiguous(), q[:, h] @ own_k[:, kv].t().contiguous() + mask), dim=1) / math.sqrt(case["dim"])
                p = torch.softmax(logits, dim=-1)
                heads.append(p[:, :s["prefix"][g]] @ shared_v[:, kv].contiguous() + p[:, s["prefix"][g]:] @ own_v[:, kv].contiguous())
            parts.append(torch.stack(heads, dim=1))
            start, b = start + n, b + 1
    return torch.cat(parts)


_EXACT = {"sample_rows": _exact_sample_rows, "paged_step": _exact_paged_step, "paged_prefix_attention": _exact_prefix}


@torch.no_grad()
def exact(case, seed):
    return _EXACT[case["op"]](prepare(case, seed))
