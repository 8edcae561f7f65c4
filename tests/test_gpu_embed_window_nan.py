"""Attention with a window where a query, a key or a value is not finite: who is
touched, and what it costs."""

import pytest
import torch

from tests.helpers import say
from tests.test_gpu_embed import BF, HF, dev_cu, inside, ops, rand  # noqa: F401
from tests.test_gpu_embed_window import seen_of, window_want

pytestmark = pytest.mark.gpu

# windows of each kernel, whole and in parts
CALLS = [(1500, 4, 2, 64, BF, (64, 64), 0), (1500, 4, 2, 64, BF, (100, 0), 4), (1500, 2, 1, 128, HF, (200, 0), 3), (1500, 4, 2, 64, BF, (700, 0), 3),
         (1500, 4, 4, 32, HF, (400, 30), 0), (9000, 8, 2, 128, BF, (600, 0), 4), (1500, 2, 2, 72, BF, (300, 20), 2), (700, 1, 1, 200, BF, (300, 0), 0)]


def placed(t, offset):
    """t with its rows `offset` elements into wider ones."""
    wide = torch.zeros(*t.shape[:-1], t.shape[-1] + offset, dtype=t.dtype, device="cuda")
    wide[..., offset:] = t.cuda()
    return wide[..., offset:]


def rows_seeing(n, causal, window, sinks, key):
    return seen_of(n, n, causal, *window, sinks)[:, key]


@pytest.mark.parametrize("n,hq,hk,d,dtype,window,sinks", CALLS)
@pytest.mark.parametrize("offset", [0, 1])
def test_queries_and_keys_of_nan_stay_where_they_are(ops, n, hq, hk, d, dtype, window, sinks, offset):  # noqa: F811
    """A NaN query makes its own row NaN, a NaN key the rows that see it, with every
    element; an infinite value among them reaches who sees it.  All others are as they
    would be."""
    say("window nan", n, hq, hk, d, dtype, window, sinks, offset)
    causal, group, at, odd = window[1] == 0, hq // hk, n // 2, n // 3
    q, k, v = (rand((n, h, d), i + 1, dtype).cuda() for i, h in enumerate((hq, hk, hk)))
    want, bound = window_want(q, k, v, [0, n], [0, n], causal, *window, sinks)
    sees, sees_odd = rows_seeing(n, causal, window, sinks, at), rows_seeing(n, causal, window, sinks, odd)
    for what in ("key", "query", "key and value", "token"):
        q2, k2, v2 = q.clone(), k.clone(), v.clone()
        nan = torch.zeros(n, hq, d, dtype=torch.bool)
        inf = torch.zeros(n, hq, d, dtype=torch.bool)
        if what != "query":
            k2[at, hk - 1, 0] = float("nan")
            nan[sees, (hk - 1) * group:] = True
        if what in ("query", "token"):
            q2[at, 0] = float("nan")
            nan[at, 0] = True
        if what == "token":
            v2[at, hk - 1] = float("nan")
        if what == "key and value":
            v2[odd, hk - 1, d - 1] = float("inf")
            inf[sees_odd, (hk - 1) * group:, d - 1] = True
        got = ops.attention(*(placed(t, offset) for t in (q2, k2, v2)), dev_cu([0, n]), max_q=n, causal=causal, window=window, sinks=sinks).cpu().double()
        assert torch.isnan(got[nan]).all(), what
        assert (got[inf & ~nan] == float("inf")).all(), what
        fine = ~nan & ~inf
        inside(got[fine], want[fine], bound[fine], what)


def time_of(f):
    f()
    torch.cuda.synchronize()
    best = float("inf")
    for _ in range(3):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        f()
        b.record()
        torch.cuda.synchronize()
        best = min(best, a.elapsed_time(b))
    return best


@pytest.mark.parametrize("hq,hk,d,window,sinks", [(8, 2, 128, (4095, 0), 4), (8, 8, 64, (64, 64), 0), (4, 4, 64, (1000, 0), 0)])
def test_queries_and_keys_of_nan_cost_nothing(ops, hq, hk, d, window, sinks):  # noqa: F811
    """The rows that a NaN query or key touches are not done again one by one, which
    takes 70 to 600 times as long as the call; ten times is far from either."""
    say("window nan cost", hq, hk, d, window, sinks)
    n = 8192
    q, k, v = (rand((n, h, d), i + 1, BF).cuda() for i, h in enumerate((hq, hk, hk)))
    q2, k2 = q.clone(), k.clone()
    q2[3000], k2[3000] = float("nan"), float("nan")
    cu = dev_cu([0, n])
    run = lambda q, k: ops.attention(q, k, v, cu, max_q=n, causal=window[1] == 0, window=window, sinks=sinks)  # noqa: E731
    good = time_of(lambda: run(q, k))
    for what, t in (("query", time_of(lambda: run(q2, k))), ("key", time_of(lambda: run(q, k2)))):
        assert t < 10 * good, f"{what}: {t * 1e3:.0f} us, without NaN {good * 1e3:.0f}"
