"""The oracle of `ops.sample_rows` against counting, and the refusals of the C entry."""

import ctypes
import math

import pytest
import torch

from scaling_amd import _lib
from tests import sample_oracle as oracle


def test_oracle_by_counting():
    """Integer weights: logits log(count) draw token i for count_i of the numbers (j + 1/2) / total, in the order of the counts."""
    counts = [5, 1, 0, 8, 5, 2]
    x = torch.tensor([math.log(c) if c else -math.inf for c in counts])
    order = [3, 0, 4, 5, 1]
    want = [i for i in order for _ in range(counts[i])]
    assert [oracle.row(x, (j + 0.5) / 21)[0] for j in range(21)] == want
    want = [i for i in order[:3] for _ in range(counts[i])]
    assert [oracle.row(x, (j + 0.5) / 18, top_k=3)[0] for j in range(18)] == want
    assert [oracle.row(x, (j + 0.5) / 18, top_p=0.7)[0] for j in range(18)] == want          # 8, 13, 18 of 21: 0.7 * 21 is more than 13
    assert [oracle.row(x, (j + 0.5) / 18, min_p=0.5)[0] for j in range(18)] == want
    assert abs(oracle.row(x, 0.0)[1] - math.log(8 / 21)) < 1e-6
    assert oracle.row(torch.full((3,), -math.inf), 0.5)[:2] == (0, -math.inf) and oracle.row(torch.full((3,), math.nan), 0.5)[0] == 0
    assert oracle.row(torch.tensor([1.0, 2.0, 2.0]), 0.9, temperature=0.0)[:2] == (1, 0.0)
    assert oracle.row(torch.tensor([1.0, math.inf, 2.0, math.inf]), 0.6)[0] == 3


def test_entry_refuses():
    lib = _lib.load()
    assert lib.mi_sample(None) == -1
    a = _lib.MiSampleArgs()
    assert lib.mi_sample(ctypes.byref(a)) == 0                                               # no rows
    a.n_rows, a.vocab, a.row_stride = 4, 100, 100
    assert lib.mi_sample(ctypes.byref(a)) == -1
    buf = (ctypes.c_char * 64)()
    a.logits = a.uniforms = a.ids = ctypes.addressof(buf)
    for name, value in (("n_rows", -1), ("n_rows", 1 << 31), ("n_rows", 1 << 22), ("vocab", 0), ("vocab", (1 << 22) + 1), ("row_stride", -1)):
        before = getattr(a, name)
        setattr(a, name, value)
        assert lib.mi_sample(ctypes.byref(a)) == -3, name
        setattr(a, name, before)
    a.dtype = 9
    assert lib.mi_sample(ctypes.byref(a)) == -2


def test_ops_refuse_without_gpu():
    if torch.cuda.is_available():
        pytest.skip("GPU present")
    from scaling_amd import ops
    with pytest.raises(RuntimeError):
        ops.sample_rows(torch.zeros(2, 8), torch.zeros(2))
