"""Edges of the embedding operators' sizes, layouts and arguments, against plain
implementations in 64 bits where there are values to compare."""

import ctypes

import pytest
import torch

from tests.helpers import say
from tests.test_gpu_embed import BF, F32, HF, U, attention_want, attention_want_gpu, cu_of, dev_cu, inside, linear_want, norm_want, ops, rand  # noqa: F401

pytestmark = pytest.mark.gpu


# ------------------------------------------------------- pooling, wide rows --
@pytest.mark.parametrize("dim", [1025, 1536, 2500, 4096, 4100, 5000, 8192])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_pool_unit_of_wide_rms_rows(ops, dim, dtype):  # noqa: F811
    """Rows of several waves, RMS norm, unit length: sequences of 1, 2, 5 and 6
    rows take an odd number of sums before the vector's own, which goes through
    the same two places.  Right, and the same bits again."""
    say("pool unit of wide rows", dim, dtype)
    lens = [(1, 2, 5, 6, 3, 4, 0, 9)[i % 8] for i in range(640)]
    cu = cu_of(lens)
    x, w = rand((cu[-1], dim), 1, dtype, 1.0, 0.3), rand((dim,), 2, dtype, 0.2, 1.0)
    rows, err = norm_want(x, w, None, "rms")
    want, bound = torch.zeros(len(lens), dim, dtype=torch.float64), torch.zeros(len(lens), dim, dtype=torch.float64)
    for s, (a, e) in enumerate(zip(cu, cu[1:])):
        if e == a:
            continue
        y = rows[a:e].mean(0)
        # the rows are added one by one, divided by their number and weighted
        er = err[a:e].mean(0) + (e - a + 2) * 2.0 ** -24 * rows[a:e].abs().mean(0)
        n = y.norm()  # its square: 64 2^-24, as the norms' sums
        want[s], bound[s] = y / n, er / n + y.abs() / n * (er.norm() / n + 64 * 2.0 ** -24)
    x, w, c = x.cuda(), w.cuda(), dev_cu(cu)
    got = ops.pool(x, c, kind="rms", weight=w)
    inside(got, want, bound, "unit of wide rows")
    for _ in range(5):
        assert torch.equal(ops.pool(x, c, kind="rms", weight=w), got)
