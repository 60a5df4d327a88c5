"""Norms of queries and keys over a head with the rotary embedding in one pass, forward and backward, against float64."""

import pytest
import torch

from scaling_amd import ops
from tests import paged_oracle as oracle
from tests.kernels import launched

pytestmark = pytest.mark.gpu
DEV = "cuda"

# Roundings of float32 on the way to a result, each 2^-24 of what is summed: a row's mean and mean of squares (at most 64 additions in a lane's slots and six
# exchanges, twice for LayerNorm), the reciprocal root (2), products with weight and tables and their sums (8).
ROUNDINGS = 160
SMALLEST = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}    # half a step of subnormals


def _close(name, got, ref, size, roundings=ROUNDINGS):
    t = got.dtype
    bound = torch.finfo(t).eps / 2 * ref.abs() + (1 + torch.finfo(t).eps) * roundings * 2.0 ** -24 * size + SMALLEST[t]
    diff = (got.detach().cpu().double() - ref).abs()
    over = (diff - bound).max() if diff.numel() else torch.tensor(-1.0)
    print(f"{name}: max error / bound {float((diff / bound).max()) if diff.numel() else 0:.2f}", flush=True)
    assert bool((diff <= bound).all()), f"{name}: over the bound by {float(over):.3e}"


def _tables(rows, r, dtype, interleaved, table_dtype=None):
    ang = torch.outer(torch.arange(rows).double(), 10000.0 ** (-torch.arange(0, r, 2).double() / r))
    if interleaved:
        return ang.cos().float(), ang.sin().float()
    ang = torch.cat((ang, ang), 1)
    return ang.cos().to(table_dtype or dtype), ang.sin().to(table_dtype or dtype)


def _inputs(t, nq, nkv, d, dtype, layer_norm, seed, layout="plain"):
    g = torch.Generator().manual_seed(seed)

    def rand(*shape):
        return torch.randn(*shape, generator=g)
    if layout == "one":                                    # per head q, then k, then v
        qkv = rand(t, nq, 3 * d).to(dtype)
        q, k = qkv[..., :d], qkv[..., d:2 * d]
    elif layout == "odd":                                  # rows that are not whole vectors
        q, k = rand(t, nq, d + 1).to(dtype)[..., 1:], rand(t, nkv, d + 3).to(dtype)[..., :d]
    elif layout == "heads":                                # heads outermost
        q, k = rand(nq, t, d).to(dtype).transpose(0, 1), rand(nkv, t, d).to(dtype).transpose(0, 1)
    else:
        q, k = rand(t, nq, d).to(dtype), rand(t, nkv, d).to(dtype)
    if t > 2:
        q[1] *= 100.0                                      # rows of very different sizes
        k[2] *= 1e-3
        q[0, 0] = 0.0                                      # a row of zeros
    w = [(1 + 0.3 * rand(d)).to(dtype) for _ in range(2)] + ([(0.2 * rand(d)).to(dtype) for _ in range(2)] if layer_norm else [None, None])
    dy = [rand(t, nq, d).to(dtype), rand(t, nkv, d).to(dtype)]
    ids = torch.randint(0, 64, (t,), generator=g)
    return q, k, w, dy, ids


CASES = [
    # tokens, q heads, kv heads, d, rotated, interleaved, layer norm, layout, table type
    (1, 4, 2, 64, 64, False, False, "plain", None),
    (7, 4, 4, 64, 64, True, False, "one", None),
    (33, 8, 2, 128, 128, False, True, "plain", None),
    (65, 3, 1, 128, 128, True, True, "heads", None),
    (19, 5, 5, 96, 96, False, False, "plain", None),
    (19, 4, 2, 96, 48, False, True, "one", None),
    (9, 2, 2, 32, 16, False, False, "plain", torch.float32),
    (11, 3, 1, 32, 32, True, True, "plain", None),
    (13, 2, 1, 64, 20, False, False, "plain", None),          # halves that are not whole vectors
    (21, 4, 2, 64, 64, False, True, "odd", None),             # neither are rows
    (5, 2, 2, 80, 80, False, False, "plain", torch.float32),
    (6, 2, 1, 256, 256, True, False, "plain", None),
    (6, 2, 1, 250, 128, False, True, "plain", None),
    (4, 1, 1, 1, 0, False, False, "plain", None),             # a head of one feature, no rotation
    (17, 4, 4, 64, 0, False, True, "plain", None),
    (700, 32, 8, 128, 128, False, False, "plain", None),      # several rows per workgroup of the backward pass
    (1500, 9, 3, 64, 64, True, True, "one", None),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=["bf16", "f16", "f32"])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_norm_rotary_and_gradients(case, dtype):
    t, nq, nkv, d, r, interleaved, layer_norm, layout, table_dtype = case
    print(f"case {case} {dtype}", flush=True)
    if layout == "one":
        nkv = nq
    q, k, w, dy, ids = _inputs(t, nq, nkv, d, dtype, layer_norm, seed=t * 7 + d, layout=layout)
    eps = 1e-5
    rotary, rotate = None, oracle.no_rotation
    if r:
        cos, sin = _tables(64, r, dtype, interleaved, table_dtype)
        rotate = oracle.rotation(cos, sin, ids, d, interleaved)
        rotary = (cos.to(DEV), sin.to(DEV), ids.to(DEV))

    def device(x):                                         # with its strides
        return torch.empty_strided(x.shape, x.stride(), dtype=x.dtype, device=DEV).copy_(x) if layout == "heads" else x.to(DEV)
    if layout in ("one", "odd"):
        base_q, base_k = q._base.to(DEV), k._base.to(DEV)
        qd, kd = (base_q[..., :d], base_q[..., d:2 * d]) if layout == "one" else (base_q[..., 1:], base_k[..., :d])
    else:
        qd, kd = device(q), device(k)
    wd = [None if x is None else x.to(DEV).requires_grad_(True) for x in w]
    qd, kd = qd.detach().requires_grad_(True), kd.detach().requires_grad_(True)
    assert qd.stride() == q.stride()
    yq, yk = ops.norm_rotary(qd, kd, wd[0], wd[1], eps, wd[2], wd[3], layer_norm=layer_norm, rotary=rotary, interleaved=interleaved)
    with torch.no_grad():                                  # without gradients: the same bits
        for a, b in zip(ops.norm_rotary(qd, kd, wd[0], wd[1], eps, wd[2], wd[3], layer_norm=layer_norm, rotary=rotary, interleaved=interleaved), (yq, yk)):
            assert torch.equal(a, b)
    wanted = [qd, kd] + [x for x in wd if x is not None]
    grads = torch.autograd.grad((yq, yk), wanted, [x.to(DEV) for x in dy], retain_graph=True)
    again = torch.autograd.grad((yq, yk), wanted, [x.to(DEV) for x in dy])
    torch.cuda.synchronize()
    for a, b in zip(grads, again):
        assert torch.equal(a, b)                           # no order of its own to any sum
    sums = ROUNDINGS + t * max(nq, nkv) // 8 + 16 + 128    # a chain of a workgroup's rows, lanes, wavefronts, chains of partial sums
    for i, (x, y) in enumerate(((q, yq), (k, yk))):
        ref, size = oracle.norm_rotary(x, w[i], w[i + 2], eps, layer_norm, rotate)
        _close("qk"[i], y, ref, size)
        dx, dw, db = oracle.norm_rotary_grad(x, w[i], eps, layer_norm, rotate, dy[i])
        _close("d" + "qk"[i], grads[i], *dx, roundings=3 * ROUNDINGS)
        _close("dw" + "qk"[i], grads[2 + i], *dw, roundings=sums)
        if layer_norm:
            _close("db" + "qk"[i], grads[4 + i], *db, roundings=sums)


def test_gradients_against_differences():
    """float32 gradients along random directions against central differences of the float64 definition."""
    t, nq, nkv, d, eps = 9, 4, 2, 32, 1e-5
    q, k, w, dy, ids = _inputs(t, nq, nkv, d, torch.float32, True, seed=5)
    q[0, 0] = 0.5 + torch.arange(d) / d
    cos, sin = _tables(64, d, torch.float32, True)
    rotate = oracle.rotation(cos, sin, ids, d, True)
    leaves = [x.to(DEV).requires_grad_(True) for x in (q, k, *w)]
    out = ops.norm_rotary(leaves[0], leaves[1], leaves[2], leaves[3], eps, leaves[4], leaves[5], layer_norm=True,
                          rotary=(cos.to(DEV), sin.to(DEV), ids.to(DEV)), interleaved=True)
    grads = torch.autograd.grad(out, leaves, [x.to(DEV) for x in dy])

    def value(x):
        return sum((oracle.norm_rotary(x[i], x[2 + i], x[4 + i], eps, True, rotate)[0] * dy[i].double()).sum() for i in range(2))
    base = [x.double() for x in (q, k, *w)]
    g = torch.Generator().manual_seed(1)
    for i, grad in enumerate(grads):
        direction = torch.randn(base[i].shape, generator=g, dtype=torch.float64)
        scale = base[i].abs().clamp_min(0.05) if i < 2 else torch.ones_like(base[i])     # rows of every size
        direction = direction * scale
        h = 1e-5
        plus, minus = list(base), list(base)
        plus[i], minus[i] = base[i] + h * direction, base[i] - h * direction
        want = (value(plus) - value(minus)) / (2 * h)
        got = (grad.cpu().double() * direction).sum()
        size = (grad.cpu().double() * direction).abs().sum()
        # differences: h^2 / 6 of the third derivative, below 1e-6 of the terms here; gradients: float32
        assert abs(float(got - want)) <= 2e-5 * float(size), (i, float(got), float(want))


def test_one_output_used_and_no_tokens():
    t, nq, nkv, d = 12, 4, 2, 64
    q, k, w, dy, ids = _inputs(t, nq, nkv, d, torch.bfloat16, True, seed=3)
    cos, sin = _tables(64, d, torch.bfloat16, False)
    rotary = (cos.to(DEV), sin.to(DEV), ids.to(DEV))
    leaves = [x.to(DEV).requires_grad_(True) for x in (q, k, *w)]

    def call():
        return ops.norm_rotary(leaves[0], leaves[1], leaves[2], leaves[3], 1e-5, leaves[4], leaves[5], layer_norm=True, rotary=rotary)
    both = torch.autograd.grad(call(), leaves, [x.to(DEV) for x in dy])
    only_q = torch.autograd.grad(call()[0], leaves, dy[0].to(DEV), allow_unused=True)
    only_k = torch.autograd.grad(call()[1], leaves, dy[1].to(DEV), allow_unused=True)
    for i, (a, b, c) in enumerate(zip(both, only_q, only_k)):
        assert (b is None) == (i % 2 == 1) and (c is None) == (i % 2 == 0)
        got = b if i % 2 == 0 else c
        # alone a tensor may have more workgroups, and its sums another order
        assert torch.allclose(got.float(), a.float(), rtol=2 ** -7, atol=1e-5) if i >= 2 else torch.equal(got, a)
    # an expanded gradient and one with strides
    one = torch.ones((), dtype=torch.bfloat16, device=DEV)
    got = torch.autograd.grad(call()[0], leaves[0], one.expand(t, nq, d))[0]
    assert torch.equal(got, torch.autograd.grad(call()[0], leaves[0], torch.ones(t, nq, d, dtype=torch.bfloat16, device=DEV))[0])
    turned = dy[0].to(DEV).permute(2, 0, 1).contiguous().permute(1, 2, 0)
    assert torch.equal(torch.autograd.grad(call()[0], leaves[0], turned)[0], both[0])
    # no tokens
    empty = [torch.empty(0, n, d, dtype=torch.bfloat16, device=DEV, requires_grad=True) for n in (nq, nkv)]
    out = ops.norm_rotary(empty[0], empty[1], leaves[2], leaves[3], 1e-5, leaves[4], leaves[5], layer_norm=True, rotary=(*rotary[:2], rotary[2][:0]))
    assert out[0].shape == (0, nq, d) and out[1].shape == (0, nkv, d)
    grads = torch.autograd.grad(out, empty + leaves[2:], [torch.empty_like(x) for x in out])
    assert all(float(x.float().abs().sum()) == 0.0 for x in grads) and grads[0].shape == (0, nq, d)


def test_positions_outside_the_table_are_clamped():
    q, k, w, _, _ = _inputs(6, 2, 1, 64, torch.bfloat16, False, seed=9)
    cos, sin = _tables(64, 64, torch.bfloat16, False)
    ids = torch.tensor([0, -5, 63, 64, 2 ** 40, -2 ** 40])
    args = [x.to(DEV) for x in (q, k, w[0], w[1])]
    a = ops.norm_rotary(*args, rotary=(cos.to(DEV), sin.to(DEV), ids.to(DEV)))
    b = ops.norm_rotary(*args, rotary=(cos.to(DEV), sin.to(DEV), ids.clamp(0, 63).to(DEV)))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_infinities_and_nan_stay_in_their_rows():
    q, k, w, dy, ids = _inputs(9, 4, 2, 64, torch.float32, True, seed=4)
    cos, sin = _tables(64, 64, torch.float32, False)
    rotary = (cos.to(DEV), sin.to(DEV), ids.to(DEV))

    def call(q, k):
        leaves = [q.to(DEV).requires_grad_(True), k.to(DEV).requires_grad_(True)]
        y = ops.norm_rotary(leaves[0], leaves[1], w[0].to(DEV), w[1].to(DEV), 1e-5, w[2].to(DEV), w[3].to(DEV), layer_norm=True, rotary=rotary)
        return (*y, *torch.autograd.grad(y, leaves, [x.to(DEV) for x in dy]))
    clean = call(q, k)
    q2, k2 = q.clone(), k.clone()
    q2[3, 1, 5] = float("nan")
    k2[7, 0, 2] = float("inf")
    dirty = call(q2, k2)
    keep_q, keep_k = torch.ones(9, 4, dtype=torch.bool), torch.ones(9, 2, dtype=torch.bool)
    keep_q[3, 1] = False
    keep_k[7, 0] = False
    for a, b, keep in zip(clean, dirty, (keep_q, keep_k, keep_q, keep_k)):
        assert torch.equal(a.cpu()[keep], b.cpu()[keep])
        assert bool(torch.isnan(b.cpu()[~keep]).all())


def test_launches_streams_and_graphs():
    t, nq, nkv, d = 40, 8, 2, 128
    q, k, w, dy, ids = _inputs(t, nq, nkv, d, torch.bfloat16, False, seed=11)
    cos, sin = _tables(64, d, torch.bfloat16, False)
    rotary = (cos.to(DEV), sin.to(DEV), ids.to(DEV))
    wd = [x.to(DEV) for x in w[:2]]
    x = [q.to(DEV), k.to(DEV)]
    want = ops.norm_rotary(*x, *wd, rotary=rotary)
    names = launched(lambda: ops.norm_rotary(*x, *wd, rotary=rotary))
    assert len(names) == 1 and "head_rows_kernel" in names[0], names
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.norm_rotary(*x, *wd, rotary=rotary)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # a captured forward and backward pass, replayed on new inputs between eager work
    leaves = [v.clone().requires_grad_(True) for v in x] + [v.clone().requires_grad_(True) for v in wd]
    up = [v.to(DEV) for v in dy]

    def step():
        return torch.autograd.grad(ops.norm_rotary(*leaves, rotary=rotary), leaves, up)
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for i in range(3):
        with torch.no_grad():
            leaves[0].copy_(torch.randn(t, nq, d, generator=torch.Generator().manual_seed(i)).to(DEV))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, step()):
            assert torch.equal(a, b), i


def test_refusals():
    q, k, w, _, ids = _inputs(6, 4, 2, 64, torch.bfloat16, True, seed=2)
    cos, sin = (x.to(DEV) for x in _tables(64, 64, torch.bfloat16, False))
    q, k, ids = q.to(DEV), k.to(DEV), ids.to(DEV)
    w = [x.to(DEV) for x in w]
    ok = dict(rotary=(cos, sin, ids))
    for bad, kwargs in [
        ((q, k[:5], w[0], w[1]), ok),                                           # another number of tokens
        ((q, k[..., :32], w[0], w[1]), ok),                                     # another head
        ((q, k.half(), w[0], w[1]), ok),                                        # another type
        ((q, k, w[0].float(), w[1]), ok), ((q, k, w[0][:32], w[1]), ok),
        ((q, k.cpu(), w[0], w[1]), ok),
        ((q.double(), k.double(), w[0].double(), w[1].double()), {}),
        ((q.transpose(1, 2), k.transpose(1, 2), w[0], w[1]), {}),               # features apart
        ((q, k, w[0], w[1], 1e-5, w[2], w[3]), ok),                             # RMSNorm has no bias
        ((q, k, w[0], w[1], -1.0), ok),
        ((q, k, w[0], w[1]), dict(rotary=(cos, sin[:5], ids))),
        ((q, k, w[0], w[1]), dict(rotary=(cos, sin, ids[:5]))),
        ((q, k, w[0], w[1]), dict(rotary=(cos, sin, ids.int()))),
        ((q, k, w[0], w[1]), dict(rotary=(cos[:, :33].contiguous(), sin[:, :33].contiguous(), ids))),     # an odd number of features
        ((q, k, w[0], w[1]), dict(rotary=(cos.repeat(1, 2), sin.repeat(1, 2), ids))),                     # more than the head has
        ((q, k, w[0], w[1]), dict(rotary=(cos, sin, ids), interleaved=True)),                             # not float32 [rows, d / 2]
        ((q, k, w[0], w[1]), dict(rotary=(cos.half(), sin.half(), ids))),                                 # neither the rows' type nor float32
        ((torch.zeros(2, 1, 264, dtype=torch.bfloat16, device=DEV),) * 2 + (torch.ones(264, dtype=torch.bfloat16, device=DEV),) * 2, {}),
    ]:
        with pytest.raises((RuntimeError, ValueError, TypeError)):
            ops.norm_rotary(*bad, **kwargs)
    ops.norm_rotary(q, k, w[0], w[1], 1e-5, w[2], w[3], layer_norm=True, **ok)
    torch.cuda.synchronize()


def test_gradients_are_differentiated_once():
    """A pass that records a graph gives the same gradients, and differentiating those raises instead of taking them for constants."""
    g = torch.Generator().manual_seed(0)
    q, k, w = (torch.randn(*s, generator=g).to(DEV).requires_grad_() for s in ((6, 2, 64), (6, 1, 64), (64,)))
    out = ops.norm_rotary(q, k, w, w)
    dy = [torch.randn_like(o) for o in out]
    plain = torch.autograd.grad(out, (q, k, w), dy, retain_graph=True)
    recorded = torch.autograd.grad(out, (q, k, w), dy, create_graph=True)
    for a, b in zip(plain, recorded):
        assert torch.equal(a, b) and b.requires_grad
    with pytest.raises(RuntimeError):                        # torch's own: the graph of the gradients does not reach q
        torch.autograd.grad(recorded[0].sum(), q, retain_graph=True)
    with pytest.raises(RuntimeError, match="differentiated again"):
        recorded[0].sum().backward()


@pytest.mark.parametrize("nq,nkv", [(0, 2), (3, 0)])
def test_a_tensor_without_heads(nq, nkv):
    """Its weights' gradients are sums over nothing; the other tensor's are what they are."""
    t, d, dtype = 9, 64, torch.bfloat16
    q, k, w, dy, _ = _inputs(t, 3, 2, d, dtype, True, seed=13)
    q, k, dy = q[:, :nq], k[:, :nkv], [dy[0][:, :nq], dy[1][:, :nkv]]
    leaves = [x.contiguous().to(DEV).requires_grad_(True) for x in (q, k, *w)]
    full = [torch.full((d,), float("nan"), dtype=dtype, device=DEV) for _ in range(64)]          # what memory holds that nobody wrote
    del full

    def call():
        return ops.norm_rotary(leaves[0], leaves[1], leaves[2], leaves[3], 1e-5, leaves[4], leaves[5], layer_norm=True)
    out = call()
    assert out[0].shape == (t, nq, d) and out[1].shape == (t, nkv, d)
    up = [x.contiguous().to(DEV) for x in dy]
    grads = torch.autograd.grad(out, leaves, up)
    empty = 0 if nq == 0 else 1
    alone = torch.autograd.grad(call()[empty], leaves, up[empty], allow_unused=True)             # the tensor without heads alone
    for i, x in enumerate(grads):
        if i % 2 == empty:
            assert x.shape == leaves[i].shape and float(x.float().abs().sum()) == 0.0 and float(alone[i].float().abs().sum()) == 0.0, i
        else:
            assert alone[i] is None
    one = 1 - empty
    dx, dw, db = oracle.norm_rotary_grad((q, k)[one], w[one], 1e-5, True, oracle.no_rotation, dy[one])
    sums = ROUNDINGS + t * 3 // 8 + 16 + 128
    _close("dx", grads[one], *dx, roundings=3 * ROUNDINGS)
    _close("dw", grads[2 + one], *dw, roundings=sums)
    _close("db", grads[4 + one], *db, roundings=sums)


def test_one_bias_and_leaves_without_gradients():
    """A bias of one tensor alone; gradients of some of the leaves: the same as with all of them."""
    t, nq, nkv, d, dtype = 21, 4, 2, 64, torch.bfloat16
    q, k, w, dy, ids = _inputs(t, nq, nkv, d, dtype, True, seed=17)
    cos, sin = _tables(64, d, dtype, False)
    rotate, rotary = oracle.rotation(cos, sin, ids, d, False), (cos.to(DEV), sin.to(DEV), ids.to(DEV))
    up = [x.to(DEV) for x in dy]
    for given in (2, 3):
        bias = [w[2] if given == 2 else None, w[3] if given == 3 else None]
        leaves = {i: x.to(DEV).requires_grad_(True) for i, x in enumerate((q, k, w[0], w[1], *bias)) if x is not None}

        def call(wanted):
            at = [leaves[i] if i in wanted else None if i not in leaves else leaves[i].detach() for i in range(6)]
            y = ops.norm_rotary(at[0], at[1], at[2], at[3], 1e-5, at[4], at[5], layer_norm=True, rotary=rotary)
            return y, torch.autograd.grad(y, [leaves[i] for i in wanted], up)
        y, grads = call(list(leaves))
        grads = dict(zip(leaves, grads))
        sums = ROUNDINGS + t * nq // 8 + 16 + 128
        for i, x in enumerate((q, k)):
            _close("y", y[i], *oracle.norm_rotary(x, w[i], bias[i], 1e-5, True, rotate))
            dx, dw, db = oracle.norm_rotary_grad(x, w[i], 1e-5, True, rotate, dy[i])
            _close("dx", grads[i], *dx, roundings=3 * ROUNDINGS)
            _close("dw", grads[2 + i], *dw, roundings=sums)
            if bias[i] is not None:
                _close("db", grads[4 + i], *db, roundings=sums)
        for wanted in ([0], [3], [given + 2], [1, 2]):
            for i, x in zip(wanted, call(wanted)[1]):
                assert torch.equal(x, grads[i]), (wanted, i)


@pytest.mark.parametrize("nq,nkv,layer_norm", [(40, 1, True), (3, 38, False)], ids=["layernorm", "rms"])
def test_more_rows_than_the_workgroups_of_the_backward_pass(nq, nkv, layer_norm):
    """Workgroups take several items each, divided between the tensors by their rows."""
    t, d, dtype = 3500, 128, torch.bfloat16
    q, k, w, dy, ids = _inputs(t, nq, nkv, d, dtype, layer_norm, seed=23)
    cos, sin = _tables(64, d, dtype, False)
    rotate, rotary = oracle.rotation(cos, sin, ids, d, False), (cos.to(DEV), sin.to(DEV), ids.to(DEV))
    leaves = [None if x is None else x.to(DEV).requires_grad_(True) for x in (q, k, *w)]
    y = ops.norm_rotary(leaves[0], leaves[1], leaves[2], leaves[3], 1e-5, leaves[4], leaves[5], layer_norm=layer_norm, rotary=rotary)
    grads = torch.autograd.grad(y, [x for x in leaves if x is not None], [x.to(DEV) for x in dy])
    sums = ROUNDINGS + t * max(nq, nkv) // 8 + 16 + 128
    for i, x in enumerate((q, k)):
        _close("y", y[i], *oracle.norm_rotary(x, w[i], w[i + 2], 1e-5, layer_norm, rotate))
        dx, dw, db = oracle.norm_rotary_grad(x, w[i], 1e-5, layer_norm, rotate, dy[i])
        _close("dx", grads[i], *dx, roundings=3 * ROUNDINGS)
        _close("dw", grads[2 + i], *dw, roundings=sums)
        if layer_norm:
            _close("db", grads[4 + i], *db, roundings=sums)
