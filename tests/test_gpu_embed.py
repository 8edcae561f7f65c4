"""The embedding operators (EmbedOps) against plain implementations in 64 bits.

Bounds: u is half a unit in the last place of a type relative to its value
(2^-24 float32, 2^-11 float16, 2^-8 bfloat16).  Each test says how its bound
follows from the arithmetic; matrix instructions may round each of k additions
once in either direction, so a sum of k products is within k 2^-23 sum |x w|.
"""

import math

import numpy as np
import pytest
import torch

from tests.helpers import need_gpu, say

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def ops():
    need_gpu()
    from browservec_amd import DeviceContext, EmbedOps

    ctx = DeviceContext(0)
    e = EmbedOps(ctx)
    yield e
    e.destroy()
    ctx.destroy()


def rand(shape, seed, dtype, scale=1.0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale + shift).to(dtype)


def inside(got, want, bound, what):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, f"{what}: {got.shape} {want.shape}"
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), f"{what}: infinities differ"
    over = ((got - want).abs() - bound)[fine]
    if over.numel():
        assert over.max() <= 0, f"{what}: {int((over > 0).sum())} of {over.numel()} values outside, worst by {over.max():.3g}"


# ------------------------------------------------------------------ linear --
ACTS = {
    "none": lambda z: z,
    "relu": lambda z: z.clamp(min=0),
    "gelu": lambda z: z * torch.special.ndtr(z),
    "gelu_tanh": lambda z: 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))),
    "silu": lambda z: z * torch.sigmoid(z),
}


def linear_want(x, w, b, r, act, out_dtype):
    x, w = x.cpu().double(), w.cpu().double()
    z = x @ w.t()
    mag = x.abs() @ w.abs().t()
    if b is not None:
        z, mag = z + b.cpu().double(), mag + b.cpu().double().abs()
    y = ACTS[act](z)
    # the activations' slopes stay below 1.13; their own arithmetic is within
    # 2^-20 of max(1, |z|)
    bound = 1.13 * (x.shape[1] + 2) * 2.0 ** -23 * mag + 2.0 ** -20 * z.abs().clamp(min=1) * (act not in ("none", "relu"))
    if r is not None:
        y = y + r.cpu().double()
        bound = bound + 2.0 ** -23 * y.abs()
    return y, bound + U[out_dtype] * (y.abs() + bound) + (2.0 ** -25 if out_dtype == HF else 0.0)


@pytest.mark.parametrize("dtype,out", [(BF, BF), (HF, HF), (BF, F32), (HF, F32)])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 384, 384), (3, 100, 72), (16, 512, 64), (17, 130, 1001), (64, 64, 8),
                                   (65, 257, 136), (127, 129, 31), (256, 256, 256), (300, 770, 1000), (1, 5, 4096),
                                   (33, 1536, 384), (513, 1024, 128), (7, 2048, 2051)])
def test_linear(ops, m, n, k, dtype, out):
    say("linear", m, n, k, dtype, out)
    for i, (act, bias, res) in enumerate([("none", False, False), ("gelu", True, False), ("silu", True, True),
                                          ("relu", False, True), ("gelu_tanh", True, True)]):
        x, w = rand((m, k), i, dtype).cuda(), rand((n, k), i + 10, dtype, k ** -0.5).cuda()
        b = rand((n,), i + 20, dtype).cuda() if bias else None
        r = rand((m, n), i + 30, out).cuda() if res else None
        y = ops.linear(x, w, bias=b, residual=r, activation=act, out_dtype=out)
        assert y.dtype == out
        inside(y, *linear_want(x, w, b, r, act, out), f"linear {m}x{n}x{k} {act}")


@pytest.mark.parametrize("m,n,k", [(700, 1300, 520), (2037, 768, 768), (4100, 256, 192), (1025, 4096, 72), (40, 4100, 2050)])
def test_linear_many_tiles(ops, m, n, k):
    say("linear many tiles", m, n, k)
    x, w, b = rand((m, k), 1, BF).cuda(), rand((n, k), 2, BF, k ** -0.5).cuda(), rand((n,), 3, BF).cuda()
    r = rand((m, n), 4, BF).cuda()
    inside(ops.linear(x, w, bias=b, residual=r, activation="gelu"), *linear_want(x, w, b, r, "gelu", BF), "linear")


@pytest.mark.parametrize("m,n,k", [(2100, 1500, 264), (10000, 1000, 136), (6000, 1500, 264), (8200, 4100, 520), (5000, 700, 1003)])
def test_linear_large_tiles(ops, m, n, k):
    """Every shape of tile, ragged at all three ends; 64-bit products on the GPU."""
    say("linear large tiles", m, n, k)
    x, w, b = rand((m, k), 1, HF).cuda(), rand((n, k), 2, HF, k ** -0.5).cuda(), rand((n,), 3, HF).cuda()
    r = rand((m, n), 4, HF).cuda()
    y = ops.linear(x, w, bias=b, residual=r, activation="silu")
    xd, wd = x.double(), w.double()
    z = (xd @ wd.t().contiguous() + b.double()).cpu()
    mag = (xd.abs() @ wd.abs().t().contiguous() + b.double().abs()).cpu()
    want = ACTS["silu"](z) + r.cpu().double()
    bound = 1.13 * (k + 2) * 2.0 ** -23 * mag + 2.0 ** -20 * z.abs().clamp(min=1) + 2.0 ** -23 * want.abs()
    inside(y, want, bound + U[HF] * (want.abs() + bound) + 2.0 ** -25, "large tiles")


@pytest.mark.parametrize("m", [5, 300])
@pytest.mark.parametrize("offset,extra", [(1, 3), (3, 8), (8, 16), (0, 1)])
def test_linear_strides_and_alignment(ops, m, offset, extra):
    """Rows that start anywhere and lie apart; the result's gaps stay as they were."""
    say("linear strides", m, offset, extra)
    n, k = 200, 136
    xb, wb = rand((m, k + extra + offset), 1, HF).cuda(), rand((n, k + extra + offset), 2, HF, 0.1).cuda()
    x, w = xb[:, offset:offset + k], wb[:, offset:offset + k]
    rb = rand((m, n + extra + offset), 3, HF).cuda()
    yb = torch.full((m, n + extra + offset), 7.0, dtype=HF, device="cuda")
    y, r = yb[:, offset:offset + n], rb[:, offset:offset + n]
    b = rand((n + 1,), 4, HF).cuda()[1:]
    got = ops.linear(x, w, bias=b, residual=r, out=y)
    assert got is y
    inside(y, *linear_want(x, w, b, r, "none", HF), "linear strided")
    assert torch.all(yb[:, :offset] == 7) and torch.all(yb[:, offset + n:] == 7)


def test_linear_in_place_residual_and_empty(ops):
    say("linear in place, empty")
    x, w = rand((37, 64), 1, BF).cuda(), rand((96, 64), 2, BF, 0.1).cuda()
    h = rand((37, 96), 3, F32).cuda()
    want = linear_want(x, w, None, h, "none", F32)
    got = ops.linear(x, w, residual=h, out=h)
    inside(got, *want, "residual in place")
    assert ops.linear(x[:0], w).shape == (0, 96)
    assert ops.linear(x, w[:0]).shape == (37, 0)
    b = rand((96,), 5, BF).cuda()
    y = ops.linear(x[:, :0], w[:, :0], bias=b)  # a sum of nothing
    assert torch.equal(y, b.expand(37, 96))


@pytest.mark.parametrize("m", [2, 300])
def test_linear_infinities_and_nan(ops, m):
    """A row or weight that is not finite stays in its own row or column."""
    say("linear nan", m)
    x, w = rand((m, 100), 1, BF), rand((150, 100), 2, BF)
    x[1, 99] = float("nan")
    x[0, 3] = float("inf")
    w[149, 0] = float("-inf")
    y = ops.linear(x.cuda(), w.cuda(), activation="relu").cpu()
    want = torch.relu(x.double() @ w.double().t())
    assert torch.equal(torch.isnan(y), torch.isnan(want))
    assert torch.equal(torch.isinf(y), torch.isinf(want))


# ------------------------------------------------------------------ rotary --
def rotary_want(x, table, pos, interleaved):
    rot = table.shape[1] * 2
    y = x.cpu().double().clone()
    c, s = (table.cpu().double()[pos.cpu().long()][:, None, :, i] for i in (0, 1))
    a, b = (y[..., 0:rot:2], y[..., 1:rot:2]) if interleaved else (y[..., :rot // 2], y[..., rot // 2:rot])
    u, v = a * c - b * s, b * c + a * s
    mag = a.abs() + b.abs()
    bound = torch.zeros_like(y)
    if interleaved:
        y[..., 0:rot:2], y[..., 1:rot:2] = u, v
        bound[..., 0:rot:2] = bound[..., 1:rot:2] = mag
    else:
        y[..., :rot // 2], y[..., rot // 2:rot] = u, v
        bound[..., :rot // 2] = bound[..., rot // 2:rot] = mag
    # two products and a sum in 32 bits, one rounding to the type; elements that
    # do not turn are copied
    return y, bound * 2.0 ** -22 * 1.5 + (bound > 0) * (U[x.dtype] * y.abs() * 1.01 + (2.0 ** -25 if x.dtype == HF else 0))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("tokens,hq,hk,d,rot", [(1, 1, 1, 2, 2), (17, 12, 12, 32, 16), (33, 8, 2, 64, 64), (5, 3, 1, 80, 50),
                                                (9, 40, 8, 128, 96), (130, 6, 0, 96, 96), (3, 2, 2, 7, 6), (2, 300, 20, 256, 256),
                                                (4, 2, 1, 64, 0)])
def test_rotary(ops, tokens, hq, hk, d, rot, dtype, interleaved):
    from browservec_amd import rotary_table

    say("rotary", tokens, hq, hk, d, rot, dtype, interleaved)
    table = torch.from_numpy(rotary_table(501, rot, scaling="linear", factor=4.0)).cuda()
    g = torch.Generator().manual_seed(3)
    pos = torch.randint(0, 501, (tokens,), generator=g, dtype=torch.int32).cuda()
    qkv = rand((tokens, (hq + 2 * hk) * d + 3), 1, dtype).cuda()  # rows of any alignment
    q = qkv[:, :hq * d].unflatten(1, (hq, d))
    k = qkv[:, hq * d:(hq + hk) * d].unflatten(1, (hk, d)) if hk else None
    oq, ok = ops.rotary(q, k, table, positions=pos, interleaved=interleaved)
    inside(oq, *rotary_want(q, table, pos, interleaved), "rotary q")
    if hk:
        inside(ok, *rotary_want(k, table, pos, interleaved), "rotary k")
    before = qkv.clone()
    r = ops.rotary(q, k, table, positions=pos, interleaved=interleaved, out_q=q, out_k=k)
    assert r[0] is q and r[1] is k
    assert torch.equal(q, oq) and (k is None or torch.equal(k, ok))  # in place: the same bits
    assert torch.equal(qkv[:, (hq + hk) * d:], before[:, (hq + hk) * d:])


def test_rotary_positions(ops):
    """Positions default to the token's place; one outside the table gives NaN there only."""
    from browservec_amd import rotary_table

    say("rotary positions")
    table = torch.from_numpy(rotary_table(6, 8)).cuda()
    q = rand((6, 2, 12), 1, F32).cuda()
    got, none = ops.rotary(q, None, table)
    assert none is None
    inside(got, *rotary_want(q, table, torch.arange(6), False), "default positions")
    pos = torch.tensor([0, 5, 6, -1, 2, 2 ** 31 - 1], dtype=torch.int32).cuda()
    got = ops.rotary(q, None, table, positions=pos)[0].cpu()
    for t, ok in enumerate([True, True, False, False, True, False]):
        assert torch.isnan(got[t, :, :8]).all() == (not ok) and torch.equal(got[t, :, 8:], q[t, :, 8:].cpu())


# --------------------------------------------------------------- attention --
def attention_want(q, k, v, cu_q, cu_k, causal, scale=None):
    """The result in 64 bits and its bound: scores within (d + 2) 2^-23 sum |q k|
    scale, exponentials within 2^-17 of their value, weights rounded to the type
    once (float16: or by 2^-25), sums of n terms, one rounding at the end."""
    q, k, v = q.cpu(), k.cpu(), v.cpu()
    u = U[q.dtype]
    out, bound = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    group = q.shape[1] // k.shape[1]
    scale = scale or q.shape[2] ** -0.5
    for a, e, ka, ke in zip(cu_q, cu_q[1:], cu_k, cu_k[1:]):
        if e <= a:
            continue
        n = ke - ka
        seen = torch.ones(e - a, n, dtype=torch.bool)
        if causal:
            seen = torch.arange(n)[None] <= torch.arange(e - a)[:, None] + n - (e - a)
        for h in range(q.shape[1]):
            qq, kk, vv = q[a:e, h].double(), k[ka:ke, h // group].double(), v[ka:ke, h // group].double()
            for i in range(e - a):
                on = seen[i]
                if not on.any():
                    continue
                s = scale * (kk[on] @ qq[i])
                p = torch.exp(s - s.max())
                out[a + i, h] = p @ vv[on] / p.sum()
                delta = (q.shape[2] + 2) * 2.0 ** -23 * scale * (kk[on].abs() @ qq[i].abs()).max()
                spread = p @ vv[on].abs() / p.sum()
                bound[a + i, h] = spread * (u + 4 * delta + 2.0 ** -16 + 2 * int(on.sum()) * 2.0 ** -24) + u * out[a + i, h].abs() * 1.01
                if q.dtype == HF:
                    bound[a + i, h] += 2.0 ** -24 * (1 + vv[on].abs().sum(0) / p.sum())
    return out, bound


def cu_of(lens):
    return np.concatenate([[0], np.cumsum(lens)]).astype(np.int32).tolist()


def dev_cu(cu):
    return torch.tensor(cu, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("hq,hk,d,dtype", [(4, 4, 32, BF), (6, 2, 64, HF), (8, 1, 128, BF), (3, 3, 80, HF), (4, 2, 96, BF),
                                           (2, 1, 1, BF), (5, 5, 17, HF), (2, 2, 256, BF), (7, 1, 200, HF)])
@pytest.mark.parametrize("lens", [[1], [17], [0, 3, 0, 64, 65, 1, 0], [129, 2, 31], [200]])
def test_attention_packed(ops, lens, hq, hk, d, dtype, causal):
    say("attention", lens, hq, hk, d, dtype, causal)
    cu = cu_of(lens)
    q, k, v = rand((cu[-1], hq, d), 1, dtype, 1.5).cuda(), rand((cu[-1], hk, d), 2, dtype).cuda(), rand((cu[-1], hk, d), 3, dtype).cuda()
    o = ops.attention(q, k, v, dev_cu(cu), causal=causal)
    inside(o, *attention_want(q, k, v, cu, cu, causal), "attention")


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("hq,hk,d", [(4, 1, 64), (16, 16, 32), (6, 2, 128)])
@pytest.mark.parametrize("nq,nk", [([1], [700]), ([1, 1, 1], [1, 0, 333]), ([4, 2], [65, 1000]), ([5, 3, 130], [2, 3, 64]),
                                   ([64, 0, 1], [1500, 20, 64]), ([1] * 40, list(range(1, 81, 2)))])
def test_attention_queries_over_kept_keys(ops, nq, nk, hq, hk, d, causal):
    """More keys than queries, fewer, and none: the last query sees the last
    key, and queries before the first key see nothing."""
    say("attention kept", nq, nk, hq, hk, d, causal)
    cq, ck = cu_of(nq), cu_of(nk)
    q, k, v = rand((cq[-1], hq, d), 1, BF, 1.5).cuda(), rand((ck[-1], hk, d), 2, BF).cuda(), rand((ck[-1], hk, d), 3, BF).cuda()
    want = attention_want(q, k, v, cq, ck, causal)
    for hints in (dict(), dict(max_q=max(nq), max_k=max(nk)), dict(max_q=1, max_k=1), dict(max_q=1, max_k=100000)):
        o = ops.attention(q, k, v, dev_cu(cq), dev_cu(ck), causal=causal, **hints)
        inside(o, *want, f"attention kept {hints}")


@pytest.mark.parametrize("nq,nk", [(70, 70), (1, 300), (90, 200), (40, 9)])
def test_attention_ignores_what_it_does_not_see(ops, nq, nk):
    """Keys and values outside a query's sequence, or past its place, may hold
    anything: NaN, infinities, the type's lowest value."""
    say("attention unseen", nq, nk)
    hq, hk, d = 4, 2, 64
    q, k, v = rand((nq + 2, hq, d), 1, BF), rand((nk + 6, hk, d), 2, BF), rand((nk + 6, hk, d), 3, BF)
    cq, ck = [1, nq + 1], [3, nk + 3]
    low = torch.finfo(BF).min
    for t in (k, v):
        t[:3], t[nk + 3:] = float("nan"), float("inf")
        t[2] = low
    bad = max(3, nk + 3 - nq // 2)  # a place that only the later queries see
    for value in (float("nan"), float("inf"), float("-inf"), low):
        k2, v2 = k.clone(), v.clone()
        v2[bad, :, 5] = value
        if bad + 1 < nk + 3:
            k2[bad + 1, :, 0] = value
        first = max(0, bad - 3 - (nk - nq))  # the first query that sees either
        o = torch.full((nq + 2, hq, d), 9.0, dtype=BF, device="cuda")
        ops.attention(q.cuda(), k2.cuda(), v2.cuda(), dev_cu(cq), dev_cu(ck), causal=True, out=o)
        o = o.cpu()
        want, bound = attention_want(q[1:nq + 1], k2[3:nk + 3], v2[3:nk + 3], [0, nq], [0, nk], True)
        inside(o[1:1 + first], want[:first], bound[:first], f"unseen {value}")
        assert torch.all(o[0] == 9) and torch.all(o[nq + 1] == 9)  # queries of no sequence


def attention_want_gpu(q, k, v, lens, causal):
    """attention_want with its products on the GPU, for long sequences."""
    u, out, bound = U[q.dtype], [], []
    group, scale, a = q.shape[1] // k.shape[1], q.shape[2] ** -0.5, 0
    for n in lens:
        o, b = (torch.zeros(n, q.shape[1], q.shape[2], dtype=torch.float64) for _ in range(2))
        for h in range(q.shape[1] if n else 0):
            qq, kk, vv = (t[a:a + n, i].double() for t, i in ((q, h), (k, h // group), (v, h // group)))
            s = scale * (qq @ kk.t().contiguous())
            size = scale * (qq.abs() @ kk.abs().t().contiguous())
            if causal:
                unseen = torch.ones(n, n, dtype=torch.bool, device=q.device).triu(1)
                s, size = s.masked_fill(unseen, float("-inf")), size.masked_fill(unseen, 0)
            p = torch.exp(s - s.amax(1, keepdim=True))
            total = p.sum(1, keepdim=True)
            count = torch.arange(1, n + 1, device=q.device)[:, None] if causal else n
            delta = (q.shape[2] + 2) * 2.0 ** -23 * size.amax(1, keepdim=True)
            x = p @ vv / total
            e = p @ vv.abs() / total * (u + 4 * delta + 2.0 ** -16 + 2 * count * 2.0 ** -24) + u * x.abs() * 1.01
            if q.dtype == HF:
                seen_v = torch.cumsum(vv.abs(), 0) if causal else vv.abs().sum(0, keepdim=True)
                e += 2.0 ** -24 * (1 + seen_v / total)
            o[:, h], b[:, h] = x.cpu(), e.cpu()
        out.append(o)
        bound.append(b)
        a += n
    return torch.cat(out), torch.cat(bound)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("hq,hk,d,dtype", [(16, 4, 128, BF), (8, 8, 80, HF), (12, 3, 96, BF), (16, 4, 256, HF), (24, 8, 64, BF)])
def test_attention_long_packed(ops, hq, hk, d, dtype, causal):
    """Enough rows that a call fills the card: the tiles that only then run."""
    lens = [3000, 1, 0, 2100, 77, 6000 if hq == hk else 130]
    say("attention long", lens, hq, hk, d, dtype, causal)
    t = sum(lens)
    q, k, v = rand((t, hq, d), 1, dtype, 1.5).cuda(), rand((t, hk, d), 2, dtype).cuda(), rand((t, hk, d), 3, dtype).cuda()
    o = ops.attention(q, k, v, dev_cu(cu_of(lens)), causal=causal)
    inside(o, *attention_want_gpu(q, k, v, lens, causal), "attention long")
    if causal:  # a value near the end that is not finite: nothing before it changes, everything after does
        v[2990, :, d // 2] = float("nan")
        again = ops.attention(q, k, v, dev_cu(cu_of(lens)), causal=True)
        same = torch.ones(t, dtype=torch.bool)
        same[2990:3000] = False
        # (rows done one by one round otherwise: within twice the bound of each other)
        want, bound = attention_want_gpu(q[:2990], k[:2990], v[:2990], [2990], True)
        inside(again[:2990], want, bound, "before the NaN")
        assert torch.equal(again[3000:], o[3000:])
        assert torch.isnan(again[2990:3000, :, d // 2]).all() and not torch.isnan(again[2990:3000, :, :d // 2]).any()


def test_many_short_sequences(ops):
    """Thousands of sequences of one token or none: attention gives the value, the mean is the row."""
    say("many short sequences")
    n, hq, hk, d = 9000, 4, 2, 64
    lens = [1 if i % 7 else 0 for i in range(n)]
    t, cu = sum(lens), dev_cu(cu_of(lens))
    q, k, v = rand((t, hq, d), 1, BF).cuda(), rand((t, hk, d), 2, BF).cuda(), rand((t, hk, d), 3, BF).cuda()
    for hint in (0, 1):
        assert torch.equal(ops.attention(q, k, v, cu, max_q=hint, max_k=hint), v.repeat_interleave(2, 1))
    x = rand((t, 40), 4, F32).cuda()
    got = ops.pool(x, cu, unit=False)
    live = torch.tensor(lens, dtype=torch.bool)
    assert torch.equal(got.cpu()[live], x.cpu()) and torch.all(got.cpu()[~live] == 0)
    for mode in ("first", "last"):
        assert torch.equal(ops.pool(x, cu, mode=mode, unit=False), got)


def test_attention_large_scores(ops):
    """Scores far from 0, rising and falling along the keys: the running maximum
    has to follow, and nothing overflows."""
    say("attention large scores")
    n, d = 500, 64
    q = torch.ones(n, 2, d).to(HF)
    k = (torch.arange(n, dtype=torch.float32)[:, None, None] * 2 - 300).expand(n, 2, d).clone()
    k[:, 1] = k[:, 1].flip(0)
    k, v = k.to(HF), rand((n, 2, d), 1, HF)
    want = attention_want(q, k, v, [0, n], [0, n], False, scale=0.5)
    o = ops.attention(q.cuda(), k.cuda(), v.cuda(), dev_cu([0, n]), causal=False, scale=0.5)
    inside(o, *want, "large scores")


def test_attention_strides(ops):
    """Views of one fused row, heads outside tokens, rows of any alignment."""
    say("attention strides")
    t, hq, hk, d = 150, 4, 2, 40
    cu = cu_of([100, 50])
    qkv = rand((t, (hq + 2 * hk) * d + 1), 1, BF).cuda()
    q = qkv[:, 1:1 + hq * d].unflatten(1, (hq, d))
    k = qkv[:, 1 + hq * d:1 + (hq + hk) * d].unflatten(1, (hk, d))
    v = rand((hk, t, d), 2, BF).cuda().transpose(0, 1)
    ob = torch.zeros(hq, t + 1, d + 3, dtype=BF, device="cuda")
    o = ob[:, 1:, 3:].transpose(0, 1)
    assert ops.attention(q, k, v, dev_cu(cu), causal=True, out=o) is o
    inside(o, *attention_want(q, k, v, cu, cu, True), "strided")
    assert torch.all(ob[:, 0] == 0) and torch.all(ob[:, :, :3] == 0)


def test_attention_offsets_past_32_bits(ops):
    """Keys further than 2^31 elements into their buffer."""
    say("attention far offsets")
    hk, d, far = 1, 128, 2 ** 31 // 128 + 1000
    kv = torch.empty(far + 300, hk, d, dtype=HF, device="cuda")
    k, v = rand((300, hk, d), 1, HF), rand((300, hk, d), 2, HF)
    kv[far:] = k.cuda()
    vv = torch.empty_like(kv)
    vv[far:] = v.cuda()
    for n in (1, 200):
        q = rand((n, 2, d), 3, HF)
        want = attention_want(q, k, v, [0, n], [0, 300], True)
        o = ops.attention(q.cuda(), kv, vv, dev_cu([0, n]), dev_cu([far, far + 300]), causal=True)
        inside(o, *want, "far offsets")


def test_attention_clips_offsets(ops):
    """Offsets past the tokens there are end at them."""
    say("attention clipped offsets")
    q, k, v = rand((50, 2, 64), 1, BF).cuda(), rand((50, 1, 64), 2, BF).cuda(), rand((50, 1, 64), 3, BF).cuda()
    o = ops.attention(q, k, v, dev_cu([0, 30, 500]), dev_cu([-5, 30, 10 ** 9]), causal=True)
    inside(o, *attention_want(q, k, v, [0, 30, 50], [0, 30, 50], True), "clipped")


# ------------------------------------------------------------------- norms --
def norm_want(x, w, b, kind, eps=1e-5):
    """Sums of dim values by threads and then by halves: within 64 2^-24 of the
    values' size, once for the mean and once for the squares."""
    x = x.cpu().double()
    size = x.abs().amax(-1, keepdim=True)
    y, err = x, torch.zeros_like(x)
    if kind == "layer":
        y = y - y.mean(-1, keepdim=True)
        err = 64 * 2.0 ** -24 * size + 0 * y
    if kind:
        r = torch.rsqrt(y.square().mean(-1, keepdim=True) + eps)
        y = y * r
        err = (err + 64 * 2.0 ** -24 * y.abs() / r) * r + y.abs() * err * r * 2
    if w is not None:
        y, err = y * w.cpu().double(), err * w.cpu().double().abs() + 2.0 ** -23 * (y * w.cpu().double()).abs()
    if b is not None:
        y = y + b.cpu().double()
        err = err + 2.0 ** -23 * y.abs()
    return y, err


@pytest.mark.parametrize("dtype,out", [(BF, BF), (HF, HF), (F32, F32), (F32, BF), (HF, F32)])
@pytest.mark.parametrize("rows,dim", [(1, 1), (3, 7), (17, 384), (5, 1000), (9, 1024), (6, 2047), (5, 4096), (3, 4100), (2, 16384),
                                      (2, 9001)])
@pytest.mark.parametrize("kind", ["layer", "rms", None])
def test_norm(ops, rows, dim, dtype, out, kind):
    say("norm", rows, dim, dtype, out, kind)
    x = rand((rows, dim + 3), 1, dtype, 2.0, 0.5).cuda()[:, 1:dim + 1]
    for wt in (None, dtype, F32):
        w = None if wt is None else rand((dim,), 2, wt, 0.2, 1.0).cuda()
        b = None if wt is None or kind == "rms" else rand((dim,), 3, wt).cuda()
        y = ops.norm(x, weight=w, bias=b, kind=kind, out_dtype=out)
        want, err = norm_want(x, w, b, kind)
        inside(y, want, err + U[out] * want.abs() * 1.01 + (2.0 ** -25 if out == HF else 1e-37), f"norm {kind}")
    z = x.contiguous()
    y = ops.norm(z, kind=kind, eps=1e-5)
    assert torch.equal(ops.norm(z, kind=kind, out=z), y)  # in place: the same bits


def test_norm_constant_and_zero_rows(ops):
    say("norm constant rows")
    x = torch.full((2, 768), 3.0, dtype=F32, device="cuda")
    x[1] = 0
    assert torch.all(ops.norm(x, kind="layer") == 0)
    y = ops.norm(x, kind="rms", eps=0.0).cpu()
    assert torch.allclose(y[0], torch.ones(768), rtol=1e-6) and torch.isnan(y[1]).all()  # 0 / sqrt(0)


# ----------------------------------------------------------------- pooling --
@pytest.mark.parametrize("mode", ["mean", "first", "last"])
@pytest.mark.parametrize("kind", [None, "layer", "rms"])
@pytest.mark.parametrize("dim,dtype", [(384, BF), (1, HF), (1000, F32), (1024, HF), (2500, BF), (5000, BF), (16000, F32)])
@pytest.mark.parametrize("lens", [[1], [3, 0, 64, 65, 1, 0], [300, 1, 129]])
def test_pool(ops, lens, dim, dtype, kind, mode):
    say("pool", lens, dim, dtype, kind, mode)
    cu = cu_of(lens)
    x = rand((cu[-1] + 2, dim), 1, dtype, 1.0, 0.3).cuda()
    x[cu[-1]:] = float("nan")  # rows of no sequence
    w = rand((dim,), 2, dtype, 0.2, 1.0).cuda() if kind else None
    rows, err = norm_want(x, w, None, kind)
    for unit in (False, True):
        want, bound = torch.zeros(len(lens), dim, dtype=torch.float64), torch.zeros(len(lens), dim, dtype=torch.float64)
        for s, (a, e) in enumerate(zip(cu, cu[1:])):
            if e == a:
                continue
            pick = {"mean": slice(a, e), "first": slice(a, a + 1), "last": slice(e - 1, e)}[mode]
            y = rows[pick].mean(0)
            # at most 16 + 2 rows and then the chunks are added in turn
            er = err[pick].mean(0) + (64 + (e - a) // 64) * 2.0 ** -24 * rows[pick].abs().mean(0)
            if unit and y.norm() > 0:  # a zero vector stays
                norm = y.norm()
                er = er / norm + y.abs() / norm * (er.norm() / norm + 64 * 2.0 ** -24)
                y = y / norm
            want[s], bound[s] = y, er + 1e-37
        got = ops.pool(x, dev_cu(cu), mode=mode, kind=kind, weight=w, unit=unit)
        assert got.dtype == F32
        inside(got, want, bound, f"pool {mode} {kind} unit {unit}")


@pytest.mark.parametrize("dim,dtype,kind", [(384, BF, "rms"), (1000, HF, None), (2500, BF, "layer"), (3901, F32, None), (5000, HF, "rms"), (9001, BF, "layer")])
def test_pool_many_sequences(ops, dim, dtype, kind):
    """More sequences than compute units, of none, one or several chunks."""
    say("pool many", dim, dtype, kind)
    lens = [(0, 1, 16, 17, 33, 5, 64, 2)[i % 8] for i in range(299)] + [140]
    cu = cu_of(lens)
    x = rand((cu[-1], dim), 1, dtype, 1.0, 0.3)
    rows, err = norm_want(x, None, None, kind)
    want, bound = torch.zeros(len(lens), dim, dtype=torch.float64), torch.zeros(len(lens), dim, dtype=torch.float64)
    for s, (a, e) in enumerate(zip(cu, cu[1:])):
        if e > a:  # a row's elements are added one by one at most
            want[s] = rows[a:e].mean(0)
            bound[s] = err[a:e].mean(0) + (e - a + 2) * 2.0 ** -24 * rows[a:e].abs().mean(0) + 1e-37
    got = ops.pool(x.cuda(), dev_cu(cu), kind=kind, unit=False)
    inside(got, want, bound, "pool many")
    assert torch.equal(got, ops.pool(x.cuda(), dev_cu(cu), kind=kind, unit=False))


def test_pool_zero_vector_and_far_rows(ops):
    say("pool zero vector")
    x = torch.zeros(5, 64, dtype=BF, device="cuda")
    assert torch.all(ops.pool(x, dev_cu([0, 5])) == 0)
    big = torch.empty(2 ** 31 // 16384 + 10, 16384, dtype=HF, device="cuda")  # past 2^31 elements
    big[-3:] = rand((3, 16384), 1, HF).cuda()
    n = big.shape[0]
    got = ops.pool(big, dev_cu([n - 3, n]), unit=False)
    inside(got, big[-3:].cpu().double().mean(0, keepdim=True), 2.0 ** -22 * torch.ones(1, 16384), "far rows")


# ------------------------------------------------- streams, graphs, repeats --
def calls(ops):
    """One call of each operator on inputs of its own, as a function of nothing."""
    from browservec_amd import rotary_table

    cu = dev_cu(cu_of([70, 1, 200]))
    qkv = rand((271, 8 * 64), 1, BF).cuda()
    q, k, v = qkv[:, :256].unflatten(1, (4, 64)), qkv[:, 256:384].unflatten(1, (2, 64)), qkv[:, 384:].unflatten(1, (2, 64))
    table, w, b = torch.from_numpy(rotary_table(300, 64)).cuda(), rand((300, 512), 2, BF, 0.05).cuda(), rand((300,), 3, BF).cuda()
    ck = dev_cu([0, 271])
    return [lambda: ops.linear(qkv, w, bias=b, activation="gelu"), lambda: ops.linear(qkv[:3], w),
            lambda: ops.rotary(q, k, table)[0], lambda: ops.attention(q, k, v, cu),
            lambda: ops.attention(q[:1], k, v, dev_one, ck, max_q=1, max_k=271),
            lambda: ops.norm(qkv), lambda: ops.pool(qkv, cu, kind="rms")]


dev_one = None


@pytest.fixture(autouse=True)
def _one():
    global dev_one
    if torch.cuda.is_available() and dev_one is None:
        dev_one = dev_cu([0, 1])


def test_same_bits_again_and_on_another_stream(ops):
    say("repeats and streams")
    fns = calls(ops)
    torch.cuda.synchronize()
    first = [f() for f in fns]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [f() for f in fns]
    again = [f() for f in fns]
    torch.cuda.synchronize()
    for a, b, c in zip(first, other, again):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_graph_replays(ops):
    """Captured calls give the eager results on every replay, with eager work
    and waits between."""
    say("graph replays")
    fns = calls(ops)
    eager = [f() for f in fns]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for f in fns:
            f()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        out = [f() for f in fns]
    for _ in range(4):
        for t in out:
            t.zero_()
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(eager, out):
            assert torch.equal(a, b)
        for a, b in zip(eager, [f() for f in fns]):
            assert torch.equal(a, b)


# ---------------------------------------------------------------- refusals --
def test_refusals(ops):
    from browservec_amd import _lib as L
    from browservec_amd import DeviceContext, EmbedOps, rotary_table

    say("refusals")
    x, w = rand((4, 16), 1, BF).cuda(), rand((8, 16), 2, BF).cuda()
    cu = dev_cu([0, 4])
    q = rand((4, 2, 8), 3, BF).cuda()
    table = torch.from_numpy(rotary_table(10, 8)).cuda()
    base = rand((8, 32), 4, BF).cuda()
    for fn in (
        lambda: ops.linear(x, w[:, :8]),
        lambda: ops.linear(x, w.to(HF)),
        lambda: ops.linear(x.float(), w.float()),
        lambda: ops.linear(x, w, bias=x[0]),
        lambda: ops.linear(x, w, residual=x),
        lambda: ops.linear(x, w, activation="tanh"),
        lambda: ops.linear(x.cpu(), w),
        lambda: ops.linear(x, w.cpu()),
        lambda: ops.linear(x, w, out_dtype=HF),
        lambda: ops.linear(base[:, :16], base[:, :16], out=base[:, 8:16]),
        lambda: ops.rotary(q, None, table[:, :3].contiguous().repeat(1, 2, 1)),  # 12 of 8 elements
        lambda: ops.rotary(q, None, table.double()),
        lambda: ops.rotary(q, None, table, positions=cu),
        lambda: ops.rotary(q, q[:3], table),
        lambda: ops.attention(q, q[:, :0], q[:, :0], cu),
        lambda: ops.attention(rand((4, 3, 8), 1, BF).cuda(), q, q, cu),
        lambda: ops.attention(q.float(), q.float(), q.float(), cu),
        lambda: ops.attention(q, q.to(HF), q, cu),
        lambda: ops.attention(q, q, q, cu.long()),
        lambda: ops.attention(q, q, q, cu, dev_cu([0, 2, 4])),
        lambda: ops.attention(q, q, q, cu, scale=float("nan")),
        lambda: ops.attention(q, q, q, cu, out=q),
        lambda: ops.attention(*(rand((4, 1, 257), i, BF).cuda() for i in range(3)), cu),
        lambda: ops.norm(x, kind="batch"),
        lambda: ops.norm(x, eps=-1.0),
        lambda: ops.norm(x, weight=w[0, :8]),
        lambda: ops.norm(rand((2, 16385), 1, BF).cuda()),
        lambda: ops.pool(x, cu, mode="max"),
        lambda: ops.pool(x, cu.float()),
        lambda: ops.pool(x, cu, out=x),
    ):
        with pytest.raises(L.BVError) as e:
            fn()
        assert e.value.code in (L.BV_E_INVALID, L.BV_E_UNSUPPORTED) and str(e.value)
    # side by side in one buffer is no overlap
    y = ops.linear(base[:, :16], w, out=base[:, 16:24])
    inside(y, *linear_want(base[:, :16], w, None, None, "none", BF), "side by side")
    ctx = DeviceContext(0)
    lost = EmbedOps(ctx)
    ctx.debug_inject("lost")
    with pytest.raises(L.BVError) as e:
        lost.linear(x, w)
    assert e.value.code == L.BV_E_DEVICE_LOST
    lost.destroy()
    ctx.destroy()


def test_c_refusals(ops):
    """What the Python layer cannot hand over: null pointers, short strides, other struct sizes."""
    import ctypes

    from browservec_amd import _lib as L

    say("refusals of the C entry points")
    lib = L.load()
    buf = torch.zeros(4096, dtype=BF, device="cuda")
    p = buf.data_ptr()

    def linear(**kw):
        a = L.LinearArgs(ctypes.sizeof(L.LinearArgs))
        a.dtype = a.out_dtype = 2
        a.m, a.n, a.k, a.x, a.w, a.y = 4, 8, 16, p, p + 1024, p + 4096
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.bv_embed_linear(ops.handle, ctypes.addressof(a))

    assert linear() == L.BV_OK
    for kw in (dict(size=8), dict(x=None), dict(w=None), dict(y=None), dict(x_stride=15), dict(y_stride=7), dict(dtype=3),
               dict(out_dtype=1), dict(activation=9), dict(x=p + 1), dict(y=p), dict(m=2 ** 62), dict(residual=p + 4098),
               dict(bias=p + 4096)):
        assert linear(**kw) in (L.BV_E_INVALID, L.BV_E_UNSUPPORTED), kw
        assert lib.bv_last_error()
    assert lib.bv_embed_linear(None, None) == L.BV_E_INVALID
    assert lib.bv_embed_linear(ops.handle, None) == L.BV_E_INVALID
    ops.sync()
