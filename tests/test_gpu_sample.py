"""Tokens drawn from rows of logits, against float64."""

import math

import pytest
import torch

from scaling_amd import ops
from tests import sample_oracle as oracle
from tests.kernels import launched

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
NAMES = ["bf16", "f16", "f32"]


def _parameter(value, dtype):
    return torch.tensor(value, dtype=dtype, device=DEV) if isinstance(value, (list, tuple)) else value


def _draw(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    return ops.sample_rows(x, torch.tensor(u, dtype=torch.float32, device=DEV), _parameter(temperature, torch.float32), _parameter(top_k, torch.int32),
                           _parameter(top_p, torch.float32), _parameter(min_p, torch.float32), return_logprobs=True)


def _check(x, u, **parameters):
    """Tokens are the oracle's; log-probabilities are within a float32 rounding (half a step, and what their 64-bit sum is off by)."""
    ids, logprobs = _draw(x.to(DEV) if not x.is_cuda else x, u, **parameters)
    assert ids.dtype == torch.int64 and logprobs.dtype == torch.float32 and ids.shape == logprobs.shape == (x.shape[0],)
    for i, (want, logprob, allowed) in enumerate(oracle.rows(x.cpu(), u, **parameters)):
        got = int(ids[i])
        assert got in allowed, f"row {i}: {got}, expected {want} (or {allowed}); u {u[i]} {parameters}"
        if got == want and len(allowed) == 1:
            if math.isinf(logprob):
                assert float(logprobs[i]) == logprob
            else:
                assert abs(float(logprobs[i]) - logprob) <= 2.0 ** -24 * abs(logprob) * 1.001 + 2 * oracle.slack(x.shape[1]), (i, float(logprobs[i]), logprob)
    return ids


def _logits(rows, vocab, dtype, seed, spread=2.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, vocab, generator=g) * spread).to(dtype)


def _uniforms(rows, seed):
    u = torch.rand(rows, generator=torch.Generator().manual_seed(seed)).tolist()
    u[0] = 0.0
    if rows > 1:
        u[1] = 1.0 - 2.0 ** -24
    return u


PARAMETERS = [
    dict(),
    dict(temperature=0.7, top_k=50, top_p=0.95),
    dict(top_p=0.9),
    dict(top_k=7),
    dict(min_p=0.05, temperature=1.3),
    dict(temperature=2.0, top_k=300, top_p=0.8, min_p=0.02),
    dict(temperature=30.0, top_p=0.99),
    dict(temperature=0.01),
    dict(top_p=1e-6),
    dict(top_k=1, min_p=1.0),
]


@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
@pytest.mark.parametrize("vocab", [1, 2, 3, 8, 65, 1000, 8191, 49999, 131072, 140003])
def test_parameters(vocab, dtype):
    rows = 6
    x = _logits(rows, vocab, dtype, seed=vocab)
    for i, parameters in enumerate(PARAMETERS):
        print(f"{vocab} {dtype} {parameters}", flush=True)
        _check(x, _uniforms(rows, 100 * i + vocab % 97), **parameters)


@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
def test_parameters_of_each_row(dtype):
    rows, vocab = 12, 5003
    x = _logits(rows, vocab, dtype, seed=1)
    _check(x, _uniforms(rows, 2), temperature=[0.0, 1.0, -1.0, 0.5, 3.0, 1e-30, math.inf, math.nan, 1.0, 1.0, 0.8, 100.0],
           top_k=[0, 3, 0, -5, 10, 0, 20000, 0, 5003, 1, 100, 2500], top_p=[0.5, 1.0, 1.0, 0.9, 0.0, 0.7, 0.9, 0.5, 2.0, 1.0, 0.99, 0.3],
           min_p=[0.0, 0.0, 0.5, 0.1, 0.0, 0.0, 0.0, 0.0, 5.0, 0.0, 0.001, -1.0])


@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
@pytest.mark.parametrize("offset,width", [(0, 1000), (1, 1001), (3, 1010), (5, 1008)])
def test_rows_anywhere(offset, width, dtype):
    """Rows that are no whole vectors, start on any element and lie apart."""
    whole = _logits(5, width + 9, dtype, seed=width + offset).to(DEV)
    _check(whole[:, offset:offset + 997], _uniforms(5, 3), top_p=0.9, temperature=1.5)
    _check(whole[::2, offset:offset + 5], _uniforms(3, 4))


@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
def test_masked_and_not_finite(dtype):
    vocab, low = 3001, torch.finfo(dtype).min
    x = _logits(12, vocab, dtype, seed=5)
    hidden = torch.rand(12, vocab, generator=torch.Generator().manual_seed(6)) < 0.9
    x[0:3] = x[0:3].masked_fill(hidden[0:3], -math.inf)
    x[3:6] = x[3:6].masked_fill(hidden[3:6], low)
    x[6] = -math.inf                                       # nothing to draw from
    x[7] = math.nan
    x[8, ::3], x[8, 1::3] = math.nan, -math.inf
    x[9, 5], x[9, 700] = math.inf, math.inf
    x[10] = low
    x[11] = -math.inf
    x[11, 2999] = low
    for u in (_uniforms(12, 7), [0.75] * 12):
        for parameters in (dict(), dict(top_k=40, top_p=0.9), dict(min_p=0.2), dict(temperature=0.0)):
            ids = _check(x, u, **parameters)
            assert int(ids[6]) == int(ids[7]) == 0 and int(ids[11]) == 2999 and int(ids[9]) in (5, 700)
            assert int(ids[8]) % 3 == 2


@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
def test_equal_values(dtype):
    """Ties go to the lowest index, also among zeros of both signs and more equal values than 16 bits count."""
    n = 100003
    same = torch.zeros(4, n, dtype=dtype)
    same[1, ::2] = -0.0
    same[2, : n // 2] = 1.0
    same[3, 90000:] = -2.0
    for parameters in (dict(), dict(top_k=70000), dict(top_p=0.5), dict(min_p=0.9), dict(top_k=99999, top_p=0.75, min_p=0.1)):
        for u in ([0.0, 0.25, 0.5, 0.75], [0.999, 0.9999, 0.66, 0.31]):
            _check(same, u, **parameters)
    few = torch.tensor([[3.0, 1.0, 3.0, 1.0, 3.0, 0.0, -0.0, 0.0]] * 8, dtype=dtype)
    _check(few, [i / 8 + 0.01 for i in range(8)])
    _check(few, [i / 8 + 0.01 for i in range(8)], top_k=2)
    _check(few, [i / 8 + 0.01 for i in range(8)], top_k=7, temperature=5.0)


@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
def test_shares_of_evenly_spaced_numbers(dtype):
    """Of n evenly spaced numbers a token of probability p gets p n, give or take one."""
    n, vocab = 2048, 61
    x = _logits(1, vocab, dtype, seed=9, spread=1.5).expand(n, vocab)     # rows on one another
    u = [(i + 0.5) / n for i in range(n)]
    for parameters in (dict(), dict(top_k=20, temperature=0.7), dict(top_p=0.8)):
        ids, logprobs = _draw(x.to(DEV)[:1].expand(n, vocab), u, **parameters)
        counts, p = torch.bincount(ids.cpu(), minlength=vocab), {int(i): math.exp(float(l)) for i, l in zip(ids, logprobs)}
        assert abs(sum(p.values()) - 1) < 1e-4 or len(p) < vocab
        for i in range(vocab):
            assert abs(int(counts[i]) - n * p.get(i, 0.0)) <= 1.001, (i, int(counts[i]), n * p.get(i, 0.0))


@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
@pytest.mark.parametrize("parameters", [dict(), dict(top_k=20, temperature=0.7), dict(top_p=0.8), dict(min_p=0.2), dict(top_k=40, top_p=0.9, min_p=0.1, temperature=1.5)],
                         ids=lambda p: "-".join(p) or "all")
def test_probabilities_of_what_is_kept_add_up(parameters, dtype):
    """Every token that is kept is drawn by evenly spaced numbers that lie closer than the least of their probabilities, no other is, and their probabilities together are 1."""
    n, vocab = 8192, 61
    x = _logits(1, vocab, dtype, seed=19, spread=0.8)
    w = torch.exp(torch.sort(x[0].double(), descending=True, stable=True)[0] / parameters.get("temperature", 1.0))
    w = w[:parameters.get("top_k") or vocab]
    if "top_p" in parameters:
        w = w[:int((w.cumsum(0) < parameters["top_p"] * w.sum()).sum()) + 1]
    w = w[w >= parameters.get("min_p", 0.0) * w[0]]
    assert float(w[-1] / w.sum()) * n > 2.0
    ids, logprobs = _draw(x.to(DEV).expand(n, vocab), [(i + 0.5) / n for i in range(n)], **parameters)
    p = {int(i): float(l) for i, l in zip(ids, logprobs)}
    assert len(p) == len(w)
    # a float32 rounding of each logarithm, and weights in parts of 2^51
    assert abs(sum(math.exp(l) for l in p.values()) - 1) <= max(-l for l in p.values()) * 2.0 ** -24 * 1.01 + vocab * 2.0 ** -50


@pytest.mark.parametrize("u,same", [(-0.5, 0.0), (1.0, 1 - 2.0 ** -24), (7.0, 1 - 2.0 ** -24), (math.inf, 1 - 2.0 ** -24), (-math.inf, 0.0), (math.nan, 0.0)])
def test_numbers_outside_are_the_nearest_inside(u, same):
    x = _logits(3, 777, torch.bfloat16, seed=11)
    assert torch.equal(_draw(x.to(DEV), [u] * 3)[0], _draw(x.to(DEV), [same] * 3)[0])


def test_greedy_is_argmax_and_small_top_p_too():
    x = _logits(9, 40000, torch.bfloat16, seed=12).to(DEV)
    u = _uniforms(9, 13)
    for parameters in (dict(temperature=0.0), dict(top_k=1), dict(top_p=0.0), dict(min_p=2.0)):
        ids, logprobs = _draw(x, u, **parameters)
        assert torch.equal(ids, torch.argmax(x, dim=-1)) and float(logprobs.abs().max()) == 0.0


def test_one_launch_streams_and_replays():
    x = _logits(5, 32000, torch.bfloat16, seed=14).to(DEV)
    u = torch.tensor(_uniforms(5, 15), device=DEV)
    want = ops.sample_rows(x, u, 0.9, 100, 0.9, 0.01)
    assert len(launched(lambda: ops.sample_rows(x, u, 0.9, 100, 0.9, 0.01))) == 1
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(ops.sample_rows(x, u, 0.9, 100, 0.9, 0.01), want)
    torch.cuda.current_stream().wait_stream(side)
    graph, static = torch.cuda.CUDAGraph(), x.clone()
    with torch.cuda.graph(graph):
        out = ops.sample_rows(static, u, 0.9, 100, 0.9, 0.01)
    for seed in (16, 17, 14):
        fresh = _logits(5, 32000, torch.bfloat16, seed=seed).to(DEV)
        static.copy_(fresh)
        graph.replay()
        assert torch.equal(out, ops.sample_rows(fresh, u, 0.9, 100, 0.9, 0.01))
        torch.cuda.synchronize()
    assert torch.equal(out, want)


@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
def test_min_p_far_below(dtype):
    """Temperatures at which tokens of the type's lowest value weigh more than min_p, and ones at which min_p stands for a value near zero far below the largest."""
    vocab, low = 3000, torch.finfo(dtype).min
    x = _logits(6, vocab, dtype, seed=20)
    x[:3] = x[:3].masked_fill(torch.rand(3, vocab, generator=torch.Generator().manual_seed(21)) < 0.8, low)
    x[3, ::2] = low / 2
    x[4] *= 1e-3
    x[4, 17] = 60000.0
    _check(x, [0.99, 0.5, 0.2, 0.9, 0.7, 0.999], temperature=[-low / 4, -low / 3, math.inf, -low / 2, 60000.0 / math.log(1000.0), 1.0], min_p=[1e-3, 1e-3, 0.5, 0.05, 1e-3, 1e-3])


@pytest.mark.parametrize("dtype", DTYPES, ids=NAMES)
@pytest.mark.parametrize("value", [-math.inf, "lowest", -1e4, 0.0, -0.0, 3.5, math.inf, math.nan])
def test_one_value_most_of_the_row(value, dtype):
    """Masked tokens and the like: more than 65535 of one value, beside another one that is frequent, everywhere or only at an end of the row; NaN of any payload among them."""
    vocab, value = 140003, torch.finfo(dtype).min if value == "lowest" else value
    print(f"case {value} {dtype}", flush=True)
    x = _logits(6, vocab, dtype, seed=30)
    at = torch.rand(6, vocab, generator=torch.Generator().manual_seed(31))
    x[:3] = x[:3].masked_fill(at[:3] < 0.9, value)
    x[3, 40000:130000] = value
    x[4] = value
    x[5] = x[5].masked_fill(at[5] < 0.4, value).masked_fill(at[5] > 0.6, -2.25)
    if dtype != torch.float32:
        ints = torch.int16
        payloads = (torch.arange(200, dtype=torch.int32) % 127 + (0x7f81 if dtype == torch.bfloat16 else 0x7c01)).to(ints)
        x[1, 777:977], x[2, 777:977] = payloads.view(dtype), (payloads | torch.tensor(-32768, dtype=ints)).view(dtype)
    u = [0.3, 1 - 2.0 ** -24, 0.999, 0.5, 0.77, 0.9]
    _check(x, u, temperature=[1.0, math.inf, 3e4, 1.0, 1.0, 2.0])
    _check(x, u, temperature=[1.0, math.inf, 1.0, 1.0, 1.0, 2.0], top_k=[0, 90000, 20000, 51000, 139000, 30000], top_p=[0.9, 1.0, 0.99, 0.5, 0.7, 0.8])


def test_far_rows():
    """Offsets over 2^31 elements."""
    stride = (1 << 31) // 3 + 1001
    x = torch.empty(3 * stride + 2000, dtype=torch.bfloat16, device=DEV)
    rows = x.as_strided((4, 2000), (stride, 1))
    want = _logits(4, 2000, torch.bfloat16, seed=18)
    rows.copy_(want)
    _check(rows, _uniforms(4, 19), top_p=0.95)


def test_no_rows_and_refusals():
    x, u = torch.zeros(0, 100, device=DEV), torch.zeros(0, device=DEV)
    assert ops.sample_rows(x, u).shape == (0,)
    x, u = torch.zeros(2, 100, device=DEV), torch.zeros(2, device=DEV)
    for bad in (dict(logits=x.t()), dict(logits=x[0]), dict(logits=x.double()), dict(logits=x.int()), dict(logits=x[:, :0]), dict(uniforms=u[:1]), dict(uniforms=u.double()),
                dict(uniforms=torch.zeros(2)), dict(temperature=u[:1]), dict(top_k=u), dict(top_k=1.5), dict(top_p=u.double()), dict(min_p=True), dict(temperature="1"),
                dict(temperature=math.nan), dict(top_p=torch.zeros(2)), dict(top_p=torch.zeros(4, device=DEV)[::2])):
        with pytest.raises((RuntimeError, TypeError, ValueError)):
            ops.sample_rows(**{**dict(logits=x, uniforms=u), **bad})
