"""EmbedOps.add_norm and norm_q8 of more than 128 MB, which are read past the caches:
bit by bit as parts of the same rows below that, and some rows against 64 bits."""

import pytest
import torch

from tests.helpers import say
from tests.test_gpu_embed import BF, F32, HF, U, inside, ops  # noqa: F401
from tests.test_gpu_embed_q8 import codes_fit, floor_of, normed, sum_want

pytestmark = pytest.mark.gpu

# widths that one, two, four and sixteen waves take, of one chunk and of two, whole and not
SIZES = [(120001, 384), (90001, 501), (70003, 768), (45001, 1001), (45001, 1024), (22001, 2047), (11001, 4096), (11001, 4090), (9001, 5001),
         (11001, 8192), (6001, 9001)]
MOST = 128 << 20


def bytes_of(rows, dim, dtype, rdtype, out):
    size = lambda t: torch.empty(0, dtype=t).element_size()  # noqa: E731
    return rows * dim * (size(dtype) + size(out) + (2 * size(rdtype) if rdtype else 0))


def rows_of(rows, dim, dtype, seed, scale, pad):
    """Rows that lie `pad` elements apart from each other, from an odd address on."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.empty(rows, dim + pad, dtype=dtype, device="cuda")
    x[:, pad // 2:pad // 2 + dim] = torch.randn(rows, dim, generator=g, device="cuda") * scale + 0.25
    return x[:, pad // 2:pad // 2 + dim]


def parts(rows, each):
    step = max(1, int(MOST * 0.9 / each * rows) // 2 * 2 + 1)  # odd: rows that go in pairs lie otherwise
    return [(i, min(rows, i + step)) for i in range(0, rows, step)]


@pytest.mark.parametrize("dtype,rdtype,out", [(BF, BF, BF), (BF, F32, BF), (HF, HF, F32), (F32, F32, F32)])
@pytest.mark.parametrize("rows,dim", SIZES)
@pytest.mark.parametrize("kind,pad", [("layer", 0), ("rms", 3), (None, 2)])
def test_add_norm_of_many_bytes(ops, rows, dim, dtype, rdtype, out, kind, pad):  # noqa: F811
    say("add_norm large", rows, dim, dtype, rdtype, out, kind, pad)
    each = bytes_of(rows, dim, dtype, rdtype, out)
    assert each > MOST
    x, r = rows_of(rows, dim, dtype, 1, 2.0, pad), rows_of(rows, dim, rdtype, 2, 3.0, pad)
    w = rows_of(1, dim, F32, 3, 0.2, 0)[0] + 1 if kind else None
    y, total = ops.add_norm(x, r, weight=w, kind=kind, out_dtype=out)
    for a, e in parts(rows, each):
        py, pt = ops.add_norm(x[a:e], r[a:e], weight=w, kind=kind, out_dtype=out)
        assert torch.equal(y[a:e], py) and torch.equal(total[a:e], pt), (a, e)
    some = torch.tensor([0, 1, 2, rows // 3, rows // 2, rows - 3, rows - 2, rows - 1], device="cuda")
    t = sum_want(x[some], r[some])
    inside(total[some], t, (U[rdtype] + 2.0 ** -24) * 1.01 * t.abs() + floor_of(rdtype), "total")
    want, err = normed(t, w, None, kind)
    inside(y[some], want, err + U[out] * (want.abs() + err) * 1.01 + floor_of(out), "norm")
    # in place: the same bits, and nothing beside the rows
    r2 = r.clone()
    y2, total2 = ops.add_norm(x, r2, weight=w, kind=kind, total=r2, out=x if out == dtype else None, out_dtype=out)
    assert total2 is r2 and torch.equal(total2, total) and torch.equal(y2, y)


@pytest.mark.parametrize("dtype,rdtype", [(BF, F32), (HF, HF), (F32, None), (BF, None)])
@pytest.mark.parametrize("rows,dim", SIZES)
@pytest.mark.parametrize("kind,pad", [("rms", 0), (None, 3)])
def test_norm_q8_of_many_bytes(ops, rows, dim, dtype, rdtype, kind, pad):  # noqa: F811
    say("norm_q8 large", rows, dim, dtype, rdtype, kind, pad)
    if rdtype is None and dtype != F32:
        rows = rows * 2 + 1
    each = bytes_of(rows, dim, dtype, rdtype, torch.int8)
    assert each > MOST
    x = rows_of(rows, dim, dtype, 1, 2.0, pad)
    r = None if rdtype is None else rows_of(rows, dim, rdtype, 2, 3.0, pad)
    x[rows - 1, dim - 1], x[rows // 2] = float("inf"), 0
    if r is not None:
        r[rows // 2] = 0
    q, s, total = ops.norm_q8(x, residual=r, kind=kind)
    for a, e in parts(rows, each):
        pq, ps, pt = ops.norm_q8(x[a:e], residual=None if r is None else r[a:e], kind=kind)
        assert torch.equal(q[a:e], pq) and torch.equal(s[a:e].view(torch.int32), ps.view(torch.int32)), (a, e)
        assert r is None or torch.equal(total[a:e], pt), (a, e)
    assert torch.isnan(s[rows - 1]) and (q[rows - 1] == 0).all()
    assert s[rows // 2] == 0 and (q[rows // 2] == 0).all()
    some = torch.tensor([0, 1, 2, rows // 3, rows - 4, rows - 3, rows - 2], device="cuda")
    t = sum_want(x[some], None if r is None else r[some])
    want, err = normed(t, None, None, kind)
    if kind is None and r is None:
        err = torch.zeros_like(want)
    codes_fit(q[some], s[some], want, err, f"norm_q8 {kind}")
