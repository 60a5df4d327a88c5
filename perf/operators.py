"""Operators between the projections of an attention block, as a training step and a server of ragged batches use them:

  norm_rotary      `ops.norm_rotary`: norms of queries and keys over each head with the rotary embedding in the same pass, forward and backward
  paged_append     `ops.paged_append`: the same of a batch of new tokens, with keys and values stored into the pages of a cache
  paged_attention  `ops.paged_attention`: attention of ragged chunks of new tokens (one token and more per sequence) over those pages

With `own` false, `run` computes them in their plain form, in elementary torch operations; with `own` true it makes the calls a user makes.
"""

import math
import random

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
EPS = 1e-5


# ---- cases ---------------------------------------------------------------------------------------------------------
def norm_rotary(name=None, *, tokens, heads, kv_heads, dim, rot, dtype, layer_norm=False, interleaved=False, one_tensor=False):
    """rot: rotated features per head.  one_tensor: q and k are slices of one projection's output."""
    return _named(dict(op="norm_rotary", tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim, rot=rot, dtype=dtype, layer_norm=layer_norm,
                       interleaved=interleaved, one_tensor=one_tensor), name)


def paged_append(name=None, *, batch, new_min, new_max, ctx_min, ctx_max, heads, kv_heads, dim, page, dtype, norm=True, layer_norm=False,
                 interleaved=False):
    """new_min .. new_max new tokens per sequence, which brings its cache to ctx_min .. ctx_max."""
    return _named(dict(op="paged_append", batch=batch, new_min=new_min, new_max=new_max, ctx_min=ctx_min, ctx_max=ctx_max, heads=heads,
                       kv_heads=kv_heads, dim=dim, page=page, dtype=dtype, norm=norm, layer_norm=layer_norm, interleaved=interleaved), name)


def paged_attention(name=None, *, batch, new_min, new_max, ctx_min, ctx_max, heads, kv_heads, dim, page, dtype, singles=0, causal=True):
    """singles: that many of the sequences bring one token, whatever new_min and new_max say."""
    return _named(dict(op="paged_attention", batch=batch, new_min=new_min, new_max=new_max, ctx_min=ctx_min, ctx_max=ctx_max, heads=heads,
                       kv_heads=kv_heads, dim=dim, page=page, dtype=dtype, singles=singles, causal=causal), name)


def _named(case, name):
    if name is not None:
        case["name"] = name
    return case


def listed():
    return [
        # Training with key_query_norm: the q and k of one layer of an 8B-class decoder on 8192 tokens.
        norm_rotary("norm_rotary_8k_bf16", tokens=8192, heads=32, kv_heads=8, dim=128, rot=128, dtype="bfloat16"),
        # The default architecture block (LayerNorm, one QKV projection) of a small model, an odd number of tokens, half of each head rotated.
        norm_rotary("norm_rotary_partial_f16", tokens=4083, heads=16, kv_heads=16, dim=64, rot=32, dtype="float16", layer_norm=True, one_tensor=True),
        # float32, the default precision, of a toy model with the interleaved rotary.
        norm_rotary("norm_rotary_tiny_f32", tokens=255, heads=4, kv_heads=4, dim=64, rot=64, dtype="float32", interleaved=True),
        # One layer of a decode step of 32 users: the latency of one launch.
        paged_append("append_decode_32", batch=32, new_min=1, new_max=1, ctx_min=500, ctx_max=4096, heads=32, kv_heads=8, dim=128, page=64,
                     dtype="bfloat16"),
        # Prompts of a few users, chunk by chunk.
        paged_append("append_chunks_f16", batch=7, new_min=300, new_max=2048, ctx_min=2048, ctx_max=6000, heads=16, kv_heads=4, dim=64, page=16,
                     dtype="float16", layer_norm=True, interleaved=True),
        # Serving one user.
        paged_attention("attend_decode_1", batch=1, new_min=1, new_max=1, ctx_min=1500, ctx_max=1500, heads=32, kv_heads=8, dim=128, page=16,
                        dtype="bfloat16"),
        # Serving many users with prompts and answers of all lengths.
        paged_attention("attend_decode_32", batch=32, new_min=1, new_max=1, ctx_min=200, ctx_max=8192, heads=32, kv_heads=8, dim=128, page=64,
                        dtype="bfloat16"),
        # A few long documents, in float16 with narrow heads.
        paged_attention("attend_decode_long_f16", batch=3, new_min=1, new_max=1, ctx_min=20000, ctx_max=32768, heads=16, kv_heads=4, dim=64, page=256,
                        dtype="float16"),
        # A few tokens per user at once, as checking a draft asks for them.
        paged_attention("attend_draft_8", batch=8, new_min=3, new_max=9, ctx_min=900, ctx_max=5000, heads=32, kv_heads=8, dim=128, page=32,
                        dtype="bfloat16"),
        # The next chunk of one long prompt.
        paged_attention("attend_chunk_512", batch=1, new_min=512, new_max=512, ctx_min=8192, ctx_max=8192, heads=32, kv_heads=8, dim=128, page=64,
                        dtype="bfloat16"),
        # A mixed batch: chunks of two prompts beside sequences that decode.
        paged_attention("attend_mixed_f16", batch=18, singles=16, new_min=400, new_max=1000, ctx_min=1000, ctx_max=6000, heads=16, kv_heads=16, dim=64,
                        page=16, dtype="float16"),
        # Four long prompts, 2048 tokens of each at a time.
        paged_attention("attend_prefill_4x2048", batch=4, new_min=2048, new_max=2048, ctx_min=4096, ctx_max=16384, heads=32, kv_heads=8, dim=128, page=128,
                        dtype="bfloat16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_HEADS = ((4, 4), (8, 8), (12, 12), (16, 16), (16, 4), (32, 8), (12, 3), (32, 4), (20, 4))


def _draw_norm_rotary(rng):
    heads, kv_heads = rng.choice(_HEADS)
    dim = rng.choice((32, 64, 64, 96, 128, 128))
    interleaved = rng.random() < 0.4
    one_tensor = rng.random() < 0.3
    return norm_rotary(tokens=_log_int(rng, 1, 8192), heads=heads, kv_heads=heads if one_tensor else kv_heads, dim=dim,
                       rot=dim if interleaved else rng.choice((dim, dim, dim // 2)), dtype=rng.choice(tuple(DTYPES)), layer_norm=rng.random() < 0.4,
                       interleaved=interleaved, one_tensor=one_tensor)


def _draw_paged(rng):
    heads, kv_heads = rng.choice(_HEADS)
    batch = _log_int(rng, 1, 48)
    ctx_max = _log_int(rng, 16, 20000)
    new_max = 1 if rng.random() < 0.4 else min(ctx_max, _log_int(rng, 2, 2048))
    ctx_min = rng.randint(new_max, ctx_max)
    return dict(batch=batch, new_min=rng.randint(1, new_max), new_max=new_max, ctx_min=ctx_min, ctx_max=ctx_max, heads=heads, kv_heads=kv_heads,
                dim=rng.choice((32, 64, 64, 96, 128, 128)), page=rng.choice((16, 16, 32, 48, 64, 64, 128, 256)), dtype=rng.choice(("bfloat16", "bfloat16", "float16")))


def _cache_bytes(case):
    return 4 * case["kv_heads"] * case["dim"] * sum(_pages(case, length) * case["page"] for length in _lengths(case)[1])


def draw(rng: random.Random):
    """Sizes over the whole range of the listed cases; no more work than the largest of them."""
    most = work(listed()[-1])["flops"]
    while True:
        op = rng.choice(("norm_rotary", "paged_append", "paged_attention", "paged_attention"))
        if op == "norm_rotary":
            return _draw_norm_rotary(rng)
        case = _draw_paged(rng)
        if op == "paged_append":
            case = paged_append(norm=rng.random() < 0.7, layer_norm=rng.random() < 0.4, interleaved=rng.random() < 0.4, **case)
        else:
            case = paged_attention(singles=rng.choice((0, 0, case["batch"] // 2)), causal=rng.random() < 0.85, **case)
        if work(case)["flops"] <= most and _cache_bytes(case) <= 2 << 30 and sum(_lengths(case)[0]) <= 8192:
            return case


def _lengths(case):
    """(new tokens, cached tokens with them) per sequence; of the case's values alone."""
    rng = random.Random("lengths %d %d %d %d %d" % (case["batch"], case["new_min"], case["new_max"], case["ctx_min"], case["ctx_max"]))
    new, ctx = [], []
    for i in range(case["batch"]):
        new.append(1 if i < case.get("singles", 0) else rng.randint(case["new_min"], case["new_max"]))
        ctx.append(rng.randint(case["ctx_min"], case["ctx_max"]))
    order = list(range(case["batch"]))
    rng.shuffle(order)
    return [new[i] for i in order], [ctx[i] for i in order]


def _pages(case, length):
    return -(-length // case["page"])


def work(case):
    """Inputs read once, outputs written once; products and sums of the attention, some ten operations an element elsewhere."""
    e = DTYPES[case["dtype"]].itemsize
    d = case["dim"]
    if case["op"] == "norm_rotary":
        elements = case["tokens"] * (case["heads"] + case["kv_heads"]) * d
        tables = min(case["tokens"], 8192) * case["rot"] * (4 if case["interleaved"] else 2 * e)
        return {"bytes": 5 * elements * e + 2 * (tables + 8 * case["tokens"]), "flops": 30 * elements}
    new, ctx = _lengths(case)
    tokens = sum(new)
    if case["op"] == "paged_append":
        elements = tokens * (case["heads"] + 2 * case["kv_heads"]) * d
        return {"bytes": 2 * elements * e + tokens * (8 + d * (4 if case["interleaved"] else 2 * e)) + 4 * sum(_pages(case, n) for n in new),
                "flops": 12 * elements}
    pairs = 0
    for n, length in zip(new, ctx):
        pairs += n * length - (n * (n - 1) // 2 if case["causal"] else 0)
    return {"bytes": 2 * tokens * case["heads"] * d * e + 2 * sum(ctx) * case["kv_heads"] * d * e + 4 * sum(_pages(case, length) for length in ctx),
            "flops": 4 * d * case["heads"] * pairs}


# ---- inputs --------------------------------------------------------------------------------------------------------
def _randn(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device=DEVICE) * scale).to(dtype)


def _tables(rows, rot, dtype, interleaved):
    """cos / sin as the framework's rotary modules keep them: [rows, rot] in the tensors' type, or float32 [rows, rot / 2] for interleaved pairs."""
    angle = torch.arange(rows, device=DEVICE, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, rot, 2, device=DEVICE, dtype=torch.float64) / rot)
    if interleaved:
        return angle.cos().float(), angle.sin().float()
    angle = torch.cat((angle, angle), dim=1)
    return angle.cos().to(dtype), angle.sin().to(dtype)


def _norm_weights(gen, case, dtype):
    names = ("q_weight", "k_weight") + (("q_bias", "k_bias") if case["layer_norm"] else ())
    return {n: _randn(gen, (case["dim"],), dtype, 0.2) + (1 if "weight" in n else 0) for n in names}


def _prepare_norm_rotary(case, gen, dtype):
    t, nq, nkv, d = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
    if case["one_tensor"]:                                 # per head q, then k, then v
        qkv = _randn(gen, (t, nq, 3 * d), dtype)
        q, k = qkv[..., :d], qkv[..., d:2 * d]
    else:
        q, k = _randn(gen, (t, nq, d), dtype), _randn(gen, (t, nkv, d), dtype)
    rows = 8192
    cos, sin = _tables(rows, case["rot"], dtype, case["interleaved"])
    position_ids = torch.arange(t, device=DEVICE)          # packed documents: positions start anew
    starts = torch.randint(0, t, (3,), generator=gen, device=DEVICE)
    position_ids = position_ids - torch.where(starts[None, :] <= position_ids[:, None], starts[None, :], 0).amax(dim=1)
    weights = _norm_weights(gen, case, dtype)
    for x in (q, k, *weights.values()):
        x.requires_grad_(True)
    return dict(q=q, k=k, dq=_randn(gen, (t, nq, d), dtype), dk=_randn(gen, (t, nkv, d), dtype), rotary=(cos, sin, position_ids), **weights)


def _prepare_paged(case, gen, dtype):
    new, ctx = _lengths(case)
    nq, nkv, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    needed = [_pages(case, length) for length in ctx]
    n_pages = sum(needed) + 3
    order = torch.randperm(n_pages, generator=gen, device=DEVICE).to(torch.int32)
    page_table = torch.zeros(len(ctx), max(needed) + 1, dtype=torch.int32, device=DEVICE)
    used = 0
    for b, n in enumerate(needed):
        page_table[b, :n] = order[used:used + n]
        used += n
    tokens = sum(new)
    k_pages, v_pages = (_randn(gen, (n_pages, nkv, page, d), dtype).transpose(1, 2) for _ in range(2))   # a page's keys of one head lie together
    state = dict(k_pages=k_pages, v_pages=v_pages, page_table=page_table, new=new, ctx=ctx,
                 cu_seqlens=torch.tensor([0] + [sum(new[:i + 1]) for i in range(len(new))], dtype=torch.int32, device=DEVICE),
                 ctx_len=torch.tensor(ctx, dtype=torch.int32, device=DEVICE))
    if case["op"] == "paged_append":
        qkv = _randn(gen, (tokens, (nq + 2 * nkv) * d), dtype)     # the output of one projection
        state["q"] = qkv[:, :nq * d].view(tokens, nq, d)
        state["k"] = qkv[:, nq * d:(nq + nkv) * d].view(tokens, nkv, d)
        state["v"] = qkv[:, (nq + nkv) * d:].view(tokens, nkv, d)
        cos, sin = _tables(case["ctx_max"], d, dtype, case["interleaved"])
        position_ids = torch.cat([torch.arange(length - n, length, device=DEVICE) for n, length in zip(new, ctx)])
        state["rotary"] = (cos, sin, position_ids)
        if case["norm"]:
            state.update(_norm_weights(gen, case, dtype))
    else:
        state["q"] = _randn(gen, (tokens, nq, d), dtype, 1.5)
        if own:
            from scaling_amd import ops
            state["workspace"] = ops.paged_workspace(len(new), tokens, nq, nkv, d, torch.device(DEVICE, torch.cuda.current_device()))
    return state


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    state = _prepare_norm_rotary(case, gen, dtype) if case["op"] == "norm_rotary" else _prepare_paged(case, gen, dtype)
    state["case"] = case
    return state


# ---- one pass ------------------------------------------------------------------------------------------------------
def run(state):
    return (_RUN_OWN if own else _RUN_PLAIN)[state["case"]["op"]](state)


def _own_norm_rotary(s):
    from scaling_amd import ops
    case = s["case"]
    q, k = ops.norm_rotary(s["q"], s["k"], s["q_weight"], s["k_weight"], EPS, s.get("q_bias"), s.get("k_bias"), layer_norm=case["layer_norm"],
                           rotary=s["rotary"], interleaved=case["interleaved"])
    names = ("q_weight", "k_weight") + (("q_bias", "k_bias") if case["layer_norm"] else ())
    return (q, k) + torch.autograd.grad((q, k), (s["q"], s["k"]) + tuple(s[n] for n in names), (s["dq"], s["dk"]))


def _own_paged_append(s):
    from scaling_amd import ops
    case = s["case"]
    q = ops.paged_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["page_table"], s["cu_seqlens"], s["ctx_len"], q=s["q"], q_weight=s.get("q_weight"),
                         k_weight=s.get("k_weight"), eps=EPS, q_bias=s.get("q_bias"), k_bias=s.get("k_bias"), layer_norm=case["layer_norm"],
                         rotary=s["rotary"], interleaved=case["interleaved"])
    return q, s["k_pages"], s["v_pages"]


def _own_paged_attention(s):
    from scaling_amd import ops
    return ops.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["page_table"], s["cu_seqlens"], s["ctx_len"], causal=s["case"]["causal"],
                               max_q_len=max(s["new"]), workspace=s["workspace"])


_RUN_OWN = {"norm_rotary": _own_norm_rotary, "paged_append": _own_paged_append, "paged_attention": _own_paged_attention}


# ---- plain form: float32, rounded once -----------------------------------------------------------------------------
def _plain_norm(x, weight, bias, layer_norm):
    """(normed, rstd, scaled and shifted) of x over its last dimension"""
    x = x.float()
    if layer_norm:
        x = x - x.mean(dim=-1, keepdim=True)
    rstd = torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + EPS)
    normed = x * rstd
    y = normed * weight.float()
    return normed, rstd, y if bias is None else y + bias.float()


def _plain_rotate(x, cos, sin, position_ids, interleaved, back=False):
    c, s = cos[position_ids].float()[:, None, :], sin[position_ids].float()[:, None, :]
    if back:
        s = -s
    if interleaved:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack((a * c - b * s, b * c + a * s), dim=-1).flatten(-2)
    rot = c.shape[-1]
    half = rot // 2
    a, b = x[..., :half], x[..., half:rot]
    return torch.cat((a * c[..., :half] - b * s[..., :half], b * c[..., half:] + a * s[..., half:], x[..., rot:]), dim=-1)


@torch.no_grad()
def _plain_norm_rotary(s):
    case, (cos, sin, ids) = s["case"], s["rotary"]
    rotated, gradients, of_weights, of_biases = [], [], [], []
    for name in ("q", "k"):
        x, weight, bias, dy = s[name], s[name + "_weight"], s.get(name + "_bias"), s["d" + name]
        normed, rstd, y = _plain_norm(x, weight, bias, case["layer_norm"])
        rotated.append(_plain_rotate(y, cos, sin, ids, case["interleaved"]).to(x.dtype))
        dn = _plain_rotate(dy.float(), cos, sin, ids, case["interleaved"], back=True)
        g = dn * weight.float()
        dx = g - normed * (g * normed).mean(dim=-1, keepdim=True)
        if case["layer_norm"]:
            dx = dx - g.mean(dim=-1, keepdim=True)
            of_biases.append(dn.sum(dim=(0, 1), dtype=torch.float64).to(x.dtype))
        gradients.append((dx * rstd).to(x.dtype))
        of_weights.append((dn * normed).sum(dim=(0, 1), dtype=torch.float64).to(x.dtype))
    return tuple(rotated + gradients + of_weights + of_biases)


def _slots(s):
    """(page, row in it) of every new token"""
    page = s["case"]["page"]
    pages, rows = [], []
    for b, (n, length) in enumerate(zip(s["new"], s["ctx"])):
        at = torch.arange(length - n, length, device=DEVICE)
        pages.append(s["page_table"][b][at // page].long())
        rows.append(at % page)
    return torch.cat(pages), torch.cat(rows)


@torch.no_grad()
def _plain_paged_append(s):
    case, (cos, sin, ids) = s["case"], s["rotary"]
    out = []
    for name in ("q", "k"):
        x = s[name]
        y = _plain_norm(x, s[name + "_weight"], s.get(name + "_bias"), case["layer_norm"])[2] if case["norm"] else x.float()
        out.append(_plain_rotate(y, cos, sin, ids, case["interleaved"]).to(x.dtype))
    pages, rows = _slots(s)
    s["k_pages"][pages, rows] = out[1]
    s["v_pages"][pages, rows] = s["v"]
    return out[0], s["k_pages"], s["v_pages"]


@torch.no_grad()
def _plain_paged_attention(s):
    case = s["case"]
    nq, nkv, d = case["heads"], case["kv_heads"], case["dim"]
    n_rep, scale = nq // nkv, 1.0 / math.sqrt(d)
    out, first = torch.empty_like(s["q"]), 0
    for b, (n, length) in enumerate(zip(s["new"], s["ctx"])):
        ids = s["page_table"][b, :_pages(case, length)].long()
        k, v = (s[name][ids].flatten(0, 1)[:length].float().transpose(0, 1) for name in ("k_pages", "v_pages"))       # [nkv, length, d]
        q = s["q"][first:first + n].float().view(n, nkv, n_rep, d).permute(1, 2, 0, 3)                                   # [nkv, n_rep, n, d]
        hidden = None
        if case["causal"]:
            hidden = torch.arange(length, device=DEVICE)[None, :] > torch.arange(length - n, length, device=DEVICE)[:, None]
        for h in range(nkv):
            scores = torch.matmul(q[h].reshape(n_rep * n, d), k[h].t()).view(n_rep, n, length) * scale
            if hidden is not None:
                scores.masked_fill_(hidden, -math.inf)
            scores = torch.exp(scores - scores.amax(dim=-1, keepdim=True))
            o = torch.matmul(scores.view(n_rep * n, length), v[h]).view(n_rep, n, d) / scores.sum(dim=-1, keepdim=True)
            out[first:first + n, h * n_rep:(h + 1) * n_rep] = o.transpose(0, 1).to(out.dtype)
        first += n
    return out


_RUN_PLAIN = {"norm_rotary": _plain_norm_rotary, "paged_append": _plain_paged_append, "paged_attention": _plain_paged_attention}


# ---- the definition, in float64 ------------------------------------------------------------------------------------
def _rotation(cos, sin, position_ids, dim, interleaved):
    """x [tokens, heads, dim] -> its rotation by the positions' angles (transposed: by minus them), as sums of x and of x with its pairs swapped."""
    index = torch.arange(dim, device=DEVICE)
    c, s = torch.ones(len(position_ids), dim, dtype=torch.float64, device=DEVICE), torch.zeros(len(position_ids), dim, dtype=torch.float64, device=DEVICE)
    cr, sr = cos.double()[position_ids], sin.double()[position_ids]
    if interleaved:
        partner, sign = index ^ 1, torch.where(index % 2 == 0, -1.0, 1.0)
        c, s = cr.repeat_interleave(2, dim=1), sr.repeat_interleave(2, dim=1)
    else:
        rot = cos.shape[1]
        partner = torch.where(index < rot, (index + rot // 2) % rot, index)
        sign = torch.where(index < rot // 2, -1.0, 1.0)
        c[:, :rot], s[:, :rot] = cr, sr
    forth = s * sign                                       # y_i = x_i c_i + x_partner forth_i, so x_i also reaches y_partner by forth_partner

    def rotate(x, transposed=False):
        by = forth[:, partner] if transposed else forth
        return x * c[:, None, :] + x[..., partner] * by[:, None, :]
    return rotate


def _exact_norm(x, layer_norm):
    x = x.detach().double()
    centred = x - x.mean(dim=-1, keepdim=True) if layer_norm else x
    deviation = (centred.square().sum(dim=-1, keepdim=True) / x.shape[-1] + EPS).sqrt()
    return centred / deviation, deviation


def _exact_norm_rotary(s):
    case = s["case"]
    rotate = _rotation(*s["rotary"], case["dim"], case["interleaved"])
    out, dx, dw, db = [], [], [], []
    for name in "qk":
        unit, deviation = _exact_norm(s[name], case["layer_norm"])
        weight = s[name + "_weight"].detach().double()
        shifted = unit * weight + (s[name + "_bias"].detach().double() if case["layer_norm"] else 0.0)
        out.append(rotate(shifted))
        upstream = rotate(s["d" + name].double(), transposed=True)
        dw.append((upstream * unit).sum(dim=1).sum(dim=0))
        db.append(upstream.sum(dim=1).sum(dim=0))
        inner = upstream * weight
        projected = inner - unit * ((inner * unit).sum(dim=-1, keepdim=True) / case["dim"])
        dx.append((projected - inner.mean(dim=-1, keepdim=True) if case["layer_norm"] else projected) / deviation)
    return tuple(out + dx + dw + (db if case["layer_norm"] else []))


def _exact_paged_append(s):
    case = s["case"]
    rotate = _rotation(*s["rotary"], case["dim"], case["interleaved"])
    rotated = {}
    for name in "qk":
        x = s[name].double()
        if case["norm"]:
            x = _exact_norm(s[name], case["layer_norm"])[0] * s[name + "_weight"].double() + (s[name + "_bias"].double() if case["layer_norm"] else 0.0)
        rotated[name] = rotate(x)
    k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
    table, page, token = s["page_table"].tolist(), case["page"], 0
    for b, (n, length) in enumerate(zip(s["new"], s["ctx"])):
        at = length - n
        while at < length:                                 # page by page
            rows = min(length - at, page - at % page)
            to = slice(at % page, at % page + rows)
            k_pages[table[b][at // page], to] = rotated["k"][token:token + rows]
            v_pages[table[b][at // page], to] = s["v"][token:token + rows].double()
            at, token = at + rows, token + rows
    return rotated["q"], k_pages, v_pages


def _exact_paged_attention(s):
    case = s["case"]
    n_rep = case["heads"] // case["kv_heads"]
    table, page, start, parts = s["page_table"].tolist(), case["page"], 0, []
    for b, (n, length) in enumerate(zip(s["new"], s["ctx"])):
        pages = table[b][:_pages(case, length)]
        k = torch.cat([s["k_pages"][i] for i in pages])[:length].double()
        v = torch.cat([s["v_pages"][i] for i in pages])[:length].double()
        q = s["q"][start:start + n].double()
        heads = []
        for h in range(case["heads"]):
            logits = q[:, h] @ k[:, h // n_rep].t().contiguous() / math.sqrt(case["dim"])
            if case["causal"]:
                logits += torch.full((n, length), -math.inf, dtype=torch.float64, device=DEVICE).triu(length - n + 1)
            heads.append(torch.softmax(logits, dim=-1) @ v[:, h // n_rep].contiguous())
        parts.append(torch.stack(heads, dim=1))
        start += n
    return torch.cat(parts)


_EXACT = {"norm_rotary": _exact_norm_rotary, "paged_append": _exact_paged_append, "paged_attention": _exact_paged_attention}


@torch.no_grad()
def exact(case, seed):
    return _EXACT[case["op"]](prepare(case, seed))
