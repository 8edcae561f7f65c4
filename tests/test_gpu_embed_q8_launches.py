"""The operators in 8 bits and attention with a window at sizes that take more than one
launch (a launch of 2^32 threads runs the low 32 bits of their number)."""

import pytest
import torch

from tests.helpers import say
from tests.test_gpu_embed import BF, F32, HF, cu_of, dev_cu, ops, rand  # noqa: F401

pytestmark = pytest.mark.gpu
I8 = torch.int8


def room_for(gigabytes):
    if torch.cuda.mem_get_info()[0] < gigabytes << 30:
        pytest.skip("not enough device memory free")


def test_linear_q8_of_many_columns(ops):  # noqa: F811
    """Few rows: 2^25 columns a launch."""
    m, n = 2, 2 ** 25 + 40
    say("linear_q8, 2^25 + 40 columns")
    room_for(4)
    w = (torch.arange(n, device="cuda") % 127).to(I8)[:, None]
    x, sx = torch.tensor([[1], [-2]], dtype=I8, device="cuda"), torch.tensor([1.0, 0.5], device="cuda")
    sw, b = 2.0 ** (torch.arange(n, device="cuda") % 3), (torch.arange(n, device="cuda") % 5).to(HF)
    r = torch.ones(m, n, dtype=F32, device="cuda")
    y = ops.linear_q8(x, sx, w, sw, bias=b, residual=r)
    assert torch.equal(y, x.float() * w[:, 0].float() * sx[:, None] * sw + b.float() + 1)  # exact in 32 bits
    del w, sw, b, r, y
    torch.cuda.empty_cache()


def test_linear_q8_of_many_rows(ops):  # noqa: F811
    """2^21 tiles a launch, of 64 rows here."""
    m, n, k = 2 ** 27 + 300, 3, 16
    say("linear_q8, 2^27 + 300 rows")
    room_for(16)
    x = torch.empty(m, k, dtype=I8, device="cuda")
    sx = torch.empty(m, device="cuda")
    for a in range(0, m, 2 ** 26):
        at = torch.arange(a, min(m, a + 2 ** 26), device="cuda")
        x[a:a + 2 ** 26] = (at % 127).to(I8)[:, None]
        sx[a:a + 2 ** 26] = 2.0 ** (at % 3 - 4)
    w, sw = torch.tensor([[1] * k, [-3] * k, [0] * k], dtype=I8, device="cuda"), torch.tensor([1.0, 0.5, 2.0], device="cuda")
    y = ops.linear_q8(x, sx, w, sw, out_dtype=F32)
    for a in range(0, m, 2 ** 26):
        want = x[a:a + 2 ** 26, :1].float() * sx[a:a + 2 ** 26, None] * torch.tensor([16.0, -24.0, 0.0], device="cuda")  # exact in 32 bits
        assert torch.equal(y[a:a + 2 ** 26], want), a
    del x, sx, y, want
    torch.cuda.empty_cache()


@pytest.mark.parametrize("rows,dim", [(2 ** 24 + 101, 8), (2 ** 22 + 51, 520), (2 ** 21 + 1, 8200)])
def test_add_norm_and_norm_q8_of_more_rows_than_a_launch(ops, rows, dim):  # noqa: F811
    """Rows of one, two and sixteen waves."""
    say("add_norm, rows", rows, dim)
    room_for(3 * 2 * rows * dim // 2 ** 30 + 16)
    edge = rows - 40
    x, r = torch.full((rows, dim), 3.0, dtype=BF, device="cuda"), torch.full((rows, dim), -1.0, dtype=BF, device="cuda")
    r[edge:] = 13
    q, s, total = ops.norm_q8(x, residual=r, kind=None)
    same = lambda t, head, tail: all((t[a:min(edge, a + 2 ** 18)] == head).all() for a in range(0, edge, 2 ** 18)) and (t[edge:] == tail).all()  # noqa: E731
    assert same(total, 2, 16) and same(q, 127, 127)
    two, sixteen = torch.tensor([2.0, 16.0]) / 127
    assert same(s, two.item(), sixteen.item())
    del q, s, total
    _, total = ops.add_norm(x, r, kind="rms", total=r, out=x)  # 2 / sqrt(4 + 1e-5) is 1 in bfloat16
    assert total is r and same(r, 2, 16) and same(x, 1, 1)
    del x, r, total
    torch.cuda.empty_cache()


@pytest.mark.parametrize("d,window,sinks,max_q,batch", [(64, (64, 64), 0, 300, 2 ** 22 + 1000), (32, (64, 0), 4, 300, 2 ** 22 + 1000),
                                                        (64, (150, 20), 3, 700, 2 ** 22 + 1000), (9, (100, 0), 0, 300, 2 ** 22 + 1000),
                                                        (64, (50, 0), 4, 1, 2 ** 25 + 1000)])
@pytest.mark.parametrize("causal", [False, True])
def test_windows_of_more_sequences_than_a_launch(ops, d, window, sinks, max_q, batch, causal):  # noqa: F811
    """Nearly all of them empty; the others as without those, bit by bit (windows that
    are not split, however few sequences there are)."""
    say("windows of sequences", d, window, sinks, max_q, batch, causal)
    room_for(4)
    lens = [300, 1, 129, 700, 33] if max_q > 1 else [1, 1, 4, 2, 1]
    places = [0, 5, batch // 2, batch - 2, batch - 1]
    nk = [n + (0 if max_q > 1 else 90) for n in lens]
    cq, ck = cu_of(lens), cu_of(nk)
    cus = []
    for n in (lens, nk):
        each = torch.zeros(batch + 1, dtype=torch.int32, device="cuda")
        each[torch.tensor(places, device="cuda") + 1] = torch.tensor(n, dtype=torch.int32, device="cuda")
        cus.append(torch.cumsum(each, 0, dtype=torch.int32))
    q, k, v = rand((cq[-1], 2, d), 1, BF, 1.5).cuda(), rand((ck[-1], 1, d), 2, BF).cuda(), rand((ck[-1], 1, d), 3, BF).cuda()
    want = ops.attention(q, k, v, dev_cu(cq), dev_cu(ck), max_q=max_q, max_k=max(nk), causal=causal, window=window, sinks=sinks)
    got = ops.attention(q, k, v, *cus, max_q=max_q, max_k=max(nk), causal=causal, window=window, sinks=sinks)
    assert torch.isfinite(want).all() and (want.float().abs().amax((1, 2)) > 0).all()
    assert torch.equal(got, want)
