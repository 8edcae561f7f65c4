"""The embedding operators in 8 bits (EmbedOps.linear_q8, norm_q8) and the norm
with its addition (add_norm) against plain implementations in 64 bits."""

import ctypes

import pytest
import torch

from tests.helpers import say
from tests.test_gpu_embed import ACTS, BF, F32, HF, U, inside, norm_want, ops, rand  # noqa: F401

pytestmark = pytest.mark.gpu
I8 = torch.int8


def codes(shape, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-128, 128, shape, generator=g, dtype=torch.int32).to(I8)


def scales(n, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.rand(n, generator=g) * 0.02 + 1e-4


def floor_of(dtype):
    """Half of a type's smallest number, where results may fall below its normal ones."""
    return 2.0 ** -25 if dtype == HF else 1e-37


# --------------------------------------------------------------- linear_q8 --
def linear_q8_want(x, sx, w, sw, b, r, act, out):
    """The sum is exact; it is rounded to 32 bits, multiplied by two scales and
    added to the bias: four roundings of 2^-24 of the product's size, the last of
    the sum's.  The activations' slopes stay below 1.13; their own arithmetic is
    within 2^-20 of max(1, |z|)."""
    dev = x.device
    z = (x.double() @ w.double().t().contiguous()) * sx.double()[:, None] * sw.double()  # whole numbers below 2^53
    mag = z.abs()
    if b is not None:
        z = z + b.double()
        mag = mag + b.double().abs()
    y = ACTS[act](z)
    bound = 1.13 * 4 * 2.0 ** -24 * 1.01 * mag + 2.0 ** -20 * z.abs().clamp(min=1) * (act not in ("none", "relu"))
    if r is not None:
        y = y + r.to(dev).double()
        bound = bound + 2.0 ** -23 * y.abs()
    return y.cpu(), (bound + U[out] * (y.abs() + bound)).cpu() + floor_of(out)


@pytest.mark.parametrize("out", [BF, HF, F32])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 384, 384), (3, 100, 72), (16, 512, 64), (17, 130, 1001), (32, 40, 63), (33, 64, 8),
                                   (65, 257, 136), (127, 129, 31), (256, 256, 256), (300, 770, 1000), (1, 5, 4096), (64, 64, 2064),
                                   (33, 1536, 384), (513, 1024, 128), (7, 2048, 2051), (100, 200, 4097)])
def test_linear_q8(ops, m, n, k, out):  # noqa: F811
    say("linear_q8", m, n, k, out)
    for i, (act, bias, res) in enumerate([("none", None, False), ("gelu", F32, False), ("silu", BF, True), ("relu", None, True),
                                          ("gelu_tanh", HF, True)]):
        x, w = codes((m, k), i).cuda(), codes((n, k), i + 10).cuda()
        sx, sw = scales(m, i + 20).cuda(), scales(n, i + 30).cuda()
        b = rand((n,), i + 40, bias).cuda() if bias else None
        r = rand((m, n), i + 50, out).cuda() if res else None
        y = ops.linear_q8(x, sx, w, sw, bias=b, residual=r, activation=act, out_dtype=out)
        assert y.dtype == out
        inside(y, *linear_q8_want(x, sx, w, sw, b, r, act, out), f"linear_q8 {m}x{n}x{k} {act}")


@pytest.mark.parametrize("out", [BF, F32])
@pytest.mark.parametrize("m,n,k", [(700, 1300, 520), (2037, 768, 768), (4100, 256, 192), (1025, 4096, 72), (40, 4100, 2050), (2100, 1500, 264),
                                   (10000, 1000, 144), (6000, 1500, 272), (8200, 4100, 520), (5000, 700, 1003), (9000, 4000, 1040)])
def test_linear_q8_many_tiles(ops, m, n, k, out):  # noqa: F811
    """Every shape of tile, ragged at all three ends."""
    say("linear_q8 many tiles", m, n, k, out)
    x, w, sx, sw = codes((m, k), 1).cuda(), codes((n, k), 2).cuda(), scales(m, 3).cuda(), scales(n, 4).cuda()
    b, r = rand((n,), 5, F32).cuda(), rand((m, n), 6, out).cuda()
    y = ops.linear_q8(x, sx, w, sw, bias=b, residual=r, activation="silu", out_dtype=out)
    inside(y, *linear_q8_want(x, sx, w, sw, b, r, "silu", out), "linear_q8")


@pytest.mark.parametrize("out", [BF, F32])
@pytest.mark.parametrize("m,n,k", [(16400, 1000, 1003), (4112, 4096, 1003), (20011, 1024, 4096)])
def test_linear_q8_rows_behind_whole_rounds(ops, m, n, k, out):  # noqa: F811
    """Sizes whose last rows go in other tiles than the rest; the result lies in wider rows."""
    say("linear_q8 rows behind", m, n, k, out)
    x, w, sx, sw = codes((m, k), 1).cuda(), codes((n, k), 2).cuda(), scales(m, 3).cuda(), scales(n, 4).cuda()
    b, r = rand((n,), 5, F32).cuda(), rand((m, n + 8), 6, out).cuda()[:, :n]
    y = torch.full((m + 1, n + 8), 7.0, dtype=out, device="cuda")
    ops.linear_q8(x, sx, w, sw, bias=b, residual=r, activation="gelu", out_dtype=out, out=y[:m, :n])
    inside(y[:m, :n], *linear_q8_want(x, sx, w, sw, b, r, "gelu", out), "linear_q8")
    assert (y[m:] == 7).all() and (y[:, n:] == 7).all()


@pytest.mark.parametrize("m", [3, 40, 600])
def test_linear_q8_of_the_largest_sums(ops, m):  # noqa: F811
    """The longest k of products of -128 and -128: sums of 2^31 - 2^14."""
    say("linear_q8 largest sums", m)
    n, k = 70, 131071
    x = torch.full((m, k), -128, dtype=I8, device="cuda")
    w = torch.full((n, k), -128, dtype=I8, device="cuda")
    w[1] = 127
    one = torch.ones(max(m, n), device="cuda")
    y = ops.linear_q8(x, one[:m], w, one[:n], out_dtype=F32).cpu().double()
    want = torch.full((m, n), 2.0 ** 14 * k, dtype=torch.float64)
    want[:, 1] = -128 * 127 * k
    assert ((y - want).abs() <= 2.0 ** -24 * want.abs()).all()


@pytest.mark.parametrize("m", [5, 300])
@pytest.mark.parametrize("offset,extra", [(1, 3), (3, 8), (16, 16), (0, 1)])
def test_linear_q8_strides_and_alignment(ops, m, offset, extra):  # noqa: F811
    """Rows that start anywhere and lie apart; the result's gaps stay as they were."""
    say("linear_q8 strides", m, offset, extra)
    n, k = 200, 144
    x, w = codes((m, k + extra + offset), 1).cuda()[:, offset:offset + k], codes((n, k + extra + offset), 2).cuda()[:, offset:offset + k]
    sx, sw = scales(m + 1, 3).cuda()[1:], scales(2 * n, 4).cuda()[::2]
    r = rand((m, n + extra + offset), 3, HF).cuda()[:, offset:offset + n]
    yb = torch.full((m, n + extra + offset), 7.0, dtype=HF, device="cuda")
    y, b = yb[:, offset:offset + n], rand((n + 1,), 4, HF).cuda()[1:]
    assert ops.linear_q8(x, sx, w, sw, bias=b, residual=r, out=y) is y
    inside(y, *linear_q8_want(x, sx, w, sw, b, r, "none", HF), "linear_q8 strided")
    assert torch.all(yb[:, :offset] == 7) and torch.all(yb[:, offset + n:] == 7)


def test_linear_q8_in_place_shapes_and_nothing(ops):  # noqa: F811
    say("linear_q8 in place, empty")
    x, w, sx, sw = codes((37, 64), 1).cuda(), codes((96, 64), 2).cuda(), scales(37, 3).cuda(), scales(96, 4).cuda()
    h = rand((37, 96), 3, F32).cuda()
    want = linear_q8_want(x, sx, w, sw, None, h, "none", F32)
    got = ops.linear_q8(x, sx, w, sw, residual=h, out=h)
    assert got is h
    inside(got, *want, "residual in place")
    assert ops.linear_q8(x, sx, w, sw).dtype == BF and ops.linear_q8(x, sx, w, sw, residual=h).dtype == F32
    assert ops.linear_q8(x[:0], sx[:0], w, sw).shape == (0, 96)
    assert ops.linear_q8(x, sx, w[:0], sw[:0]).shape == (37, 0)
    b = rand((96,), 5, F32).cuda()
    assert torch.equal(ops.linear_q8(x[:, :0], sx, w[:, :0], sw, bias=b, out_dtype=F32), b.expand(37, 96))  # a sum of nothing
    one = ops.linear_q8(x, sx, w, sw)
    for shape in ((1, 37), (37, 1)):
        assert torch.equal(ops.linear_q8(x.view(*shape, 64), sx.view(shape), w, sw), one.view(*shape, 96))
    assert torch.equal(ops.linear_q8(x[3], sx[3], w, sw), ops.linear_q8(x[3:4], sx[3:4], w, sw)[0])


@pytest.mark.parametrize("m", [2, 300])
def test_linear_q8_of_a_scale_of_nan(ops, m):  # noqa: F811
    """A row that was not finite makes its own row or column NaN, no other."""
    say("linear_q8 nan", m)
    x, w, sx, sw = codes((m, 100), 1), codes((150, 100), 2), scales(m, 3), scales(150, 4)
    sx[1], sw[149], x[1] = float("nan"), float("nan"), 0
    y = ops.linear_q8(x.cuda(), sx.cuda(), w.cuda(), sw.cuda()).cpu()
    nan = torch.zeros(m, 150, dtype=torch.bool)
    nan[1], nan[:, 149] = True, True
    assert torch.equal(torch.isnan(y), nan)


def test_linear_q8_of_rows_past_32_bits(ops):  # noqa: F811
    """Rows that lie 2^24 codes apart, of which the last is past 2^31 bytes; results
    past 2^31 elements."""
    say("linear_q8 far rows")
    far = torch.zeros(140, 2 ** 24, dtype=I8, device="cuda")
    x, w, sx, sw = far[:, 5:105], codes((90, 100), 1).cuda(), scales(140, 2).cuda(), scales(90, 3).cuda()
    x.copy_(codes((140, 100), 4))
    inside(ops.linear_q8(x, sx, w, sw), *linear_q8_want(x, sx, w, sw, None, None, "none", BF), "far rows")
    wide = torch.zeros(70, 2 ** 25, dtype=BF, device="cuda")
    y = wide[:, 7:97]
    x = x[:70].contiguous()
    ops.linear_q8(x, sx[:70], w, sw, out=y)
    inside(y, *linear_q8_want(x, sx[:70], w, sw, None, None, "none", BF), "far results")


# ------------------------------------------------------- add_norm, norm_q8 --
SIZES = [(1, 1), (3, 7), (17, 384), (5, 1000), (9, 1024), (6, 2047), (5, 4096), (3, 4100), (2, 16384), (2, 9001), (1, 8192)]


def sum_want(x, r):
    """t in 64 bits; in 32 it is within 2^-24 of its size."""
    t = x.cpu().double()
    return t if r is None else t + r.cpu().double()


def normed(t, w, b, kind):
    """The norm and its bound; the sum's own rounding passes through it as a change
    of 2^-24 of each element (times 1 / rms and the weight), and of the mean and the
    rms, by at most as much of the largest."""
    want, err = norm_want(t, w, b, kind)
    lift = torch.ones_like(t) * 3 * 2.0 ** -24 * t.abs().amax(-1, keepdim=True)
    if kind:
        c = t - t.mean(-1, keepdim=True) if kind == "layer" else t
        lift = lift / torch.sqrt(c.square().mean(-1, keepdim=True) + 1e-5) * (1 + c.abs().amax(-1, keepdim=True) / torch.sqrt(c.square().mean(-1, keepdim=True) + 1e-5))
    if w is not None:
        lift = lift * w.cpu().double().abs()
    return want, err + lift


@pytest.mark.parametrize("dtype,rdtype,out", [(BF, BF, BF), (HF, HF, HF), (F32, F32, F32), (BF, F32, BF), (HF, F32, F32), (F32, F32, HF), (BF, BF, HF)])
@pytest.mark.parametrize("rows,dim", SIZES)
@pytest.mark.parametrize("kind", ["layer", "rms", None])
def test_add_norm(ops, rows, dim, dtype, rdtype, out, kind):  # noqa: F811
    say("add_norm", rows, dim, dtype, rdtype, out, kind)
    x = rand((rows, dim + 3), 1, dtype, 2.0, 0.5).cuda()[:, 1:dim + 1]
    r = rand((rows, dim + 5), 2, rdtype, 3.0).cuda()[:, 3:dim + 3]
    t = sum_want(x, r)
    for wt in (None, dtype, F32):
        w = None if wt is None else rand((dim,), 3, wt, 0.2, 1.0).cuda()
        b = None if wt is None or kind == "rms" else rand((dim,), 4, wt).cuda()
        y, total = ops.add_norm(x, r, weight=w, bias=b, kind=kind, out_dtype=out)
        assert y.dtype == out and total.dtype == rdtype
        inside(total, t, (U[rdtype] + 2.0 ** -24) * 1.01 * t.abs() + floor_of(rdtype), "total")
        want, err = normed(t, w, b, kind)
        inside(y, want, err + U[out] * (want.abs() + err) * 1.01 + floor_of(out), f"add_norm {kind}")
    # in place: the same bits
    y, total = ops.add_norm(x, r, kind=kind)
    for which in ("residual", "x", "both"):
        x2, r2 = x.clone(memory_format=torch.contiguous_format), r.clone(memory_format=torch.contiguous_format)
        if which != "residual" and dtype != rdtype:
            continue
        into = r2 if which != "x" else x2
        y2, total2 = ops.add_norm(x2, r2, kind=kind, total=into, out=x2 if which == "both" else None)
        assert total2 is into and torch.equal(total2, total) and torch.equal(y2, y)
    strided = torch.empty(rows, dim + 3, dtype=rdtype, device="cuda")[:, 1:dim + 1]
    assert torch.equal(ops.add_norm(x, r, kind=kind, total=strided)[1], total) and torch.equal(strided, total)


def codes_fit(q, s, want, err, what):
    """q s is the row, off by half a step (127 2^-22 of one more: two roundings of f
    127 / top and one of the scale) and what y itself is off by; the largest
    magnitude has code 127."""
    q, s = q.cpu().double(), s.cpu().double()
    top = want.abs().amax(-1)
    off = err.amax(-1)
    # a scale below 2^-126 is off by up to 2^-150
    assert ((s - top / 127).abs() <= off / 127 * 1.01 + 2.0 ** -23 * top / 127 + 2.0 ** -149).all(), what
    step = s[..., None]
    over = (q * step - want).abs() - (step * (0.5 + 2.0 ** -14) + err + 127 * 2.0 ** -149)
    assert over.max() <= 0, f"{what}: {over.max()}"
    assert (q.abs().amax(-1) == 127)[top > 127 * off].all() and q.abs().max() <= 127, what


@pytest.mark.parametrize("dtype,rdtype", [(BF, None), (HF, None), (F32, None), (BF, BF), (HF, HF), (BF, F32), (HF, F32), (F32, F32)])
@pytest.mark.parametrize("rows,dim", SIZES)
@pytest.mark.parametrize("kind", ["layer", "rms", None])
def test_norm_q8(ops, rows, dim, dtype, rdtype, kind):  # noqa: F811
    say("norm_q8", rows, dim, dtype, rdtype, kind)
    x = rand((rows, dim + 3), 1, dtype, 2.0, 0.5).cuda()[:, 1:dim + 1]
    r = None if rdtype is None else rand((rows, dim + 5), 2, rdtype, 3.0).cuda()[:, 3:dim + 3]
    t = sum_want(x, r)
    for wt in (None, F32):
        w = None if wt is None else rand((dim,), 3, wt, 0.2, 1.0).cuda()
        b = None if wt is None or kind == "rms" else rand((dim,), 4, wt).cuda()
        q, s, total = ops.norm_q8(x, residual=r, weight=w, bias=b, kind=kind)
        assert q.dtype == I8 and q.shape == x.shape and s.dtype == F32 and s.shape == (rows,)
        want, err = normed(t, w, b, kind)
        if kind is None and w is None and r is None:
            err = torch.zeros_like(want)  # the rows as they are
        codes_fit(q, s, want, err, f"norm_q8 {kind}")
        if r is None:
            assert total is None
        else:
            inside(total, t, (U[rdtype] + 2.0 ** -24) * 1.01 * t.abs() + floor_of(rdtype), "total")
    gap = torch.full((rows, dim + 4), 77, dtype=I8, device="cuda")
    into, sc = gap[:, 2:dim + 2], torch.empty(rows, device="cuda")
    a, c, _ = ops.norm_q8(x, residual=r, weight=w, bias=b, kind=kind, out=into, scales=sc)
    assert a is into and c is sc and torch.equal(into, q) and torch.equal(sc, s)
    assert (gap[:, :2] == 77).all() and (gap[:, dim + 2:] == 77).all()


@pytest.mark.parametrize("dim", [5, 384, 2000, 9000])
def test_norm_q8_rows_of_all_sizes(ops, dim):  # noqa: F811
    """Zeros, infinities, NaN, the largest and the smallest numbers; each row by itself."""
    say("norm_q8 rows", dim)
    x = rand((9, dim), 1, F32)
    x[0] = 0
    x[1, dim - 1] = float("nan")
    x[2, 0] = float("-inf")
    x[3] *= 1e-40 / x[3].abs().max()
    x[4] *= 3.4e38 / x[4].abs().max()
    x[5] *= 2.0 ** -100 / x[5].abs().max()
    x[6] = -0.0
    x[7] = 0
    x[7, dim // 2] = 1e-45
    q, s, _ = ops.norm_q8(x.cuda(), kind=None)
    bad, zero = [1, 2], [0, 6]
    assert torch.isnan(s[bad]).all() and (q[bad] == 0).all()
    assert (s[zero] == 0).all() and (q[zero] == 0).all()
    fine = [3, 4, 5, 8]
    codes_fit(q[fine], s[fine], x[fine].double(), torch.zeros(4, dim, dtype=torch.float64), "rows")
    assert q[7, dim // 2] == 127 and int((q[7] != 0).sum()) == 1
    # and through a product: NaN where the row was not finite, nothing elsewhere
    w, sw, _ = ops.norm_q8(rand((40, dim), 2, BF).cuda(), kind=None)
    y = ops.linear_q8(q, s, w, sw, out_dtype=F32)
    assert torch.isnan(y[bad]).all() and (y[zero] == 0).all() and torch.isfinite(y[[0, 3, 5, 6, 7, 8]]).all()


def test_norm_q8_ties_and_exact_codes(ops):  # noqa: F811
    """Rows whose largest magnitude is 127: codes are the values, halves go to even."""
    say("norm_q8 ties")
    x = (torch.arange(512) % 255 - 127).float()
    x[0] = 127
    rows = torch.stack([x, x.clamp(-126, 126) + 0.5 * (torch.arange(512) % 2)])
    rows[1, 0] = 127
    q, s, _ = ops.norm_q8(rows.cuda(), kind=None)
    assert (s == 1).all()
    assert torch.equal(q.cpu().float(), rows.round())
    for dtype in (BF, HF):
        assert torch.equal(ops.norm_q8(rows[:1].to(dtype).cuda(), kind=None)[0].cpu().float(), rows[:1])


def test_add_norm_of_many_rows_and_nothing(ops):  # noqa: F811
    say("add_norm many rows")
    n, dim = 20001, 100
    x, r = rand((n, dim), 1, BF).cuda(), rand((n, dim), 2, F32).cuda()
    y, t = ops.add_norm(x, r, kind="rms", out_dtype=F32)
    want, err = normed(sum_want(x, r), None, None, "rms")
    inside(y, want, err + 2.0 ** -23 * want.abs(), "many rows")
    assert torch.equal(t, x.float() + r)
    y, t = ops.add_norm(x[:0], r[:0])
    assert y.shape == t.shape == (0, dim)
    q, s, t = ops.norm_q8(x[:0])
    assert q.shape == (0, dim) and s.shape == (0,) and t is None
    for shape in ((3, 4, 100), (1, 12, 100), (100,)):
        xs, rs = x[:12].reshape(-1)[:torch.Size(shape).numel()].view(shape), r[:12].reshape(-1)[:torch.Size(shape).numel()].view(shape)
        q, s, t = ops.norm_q8(xs, residual=rs)
        flat = ops.norm_q8(xs.reshape(-1, 100), residual=rs.reshape(-1, 100))
        assert q.shape == t.shape == shape and s.shape == shape[:-1]
        assert all(torch.equal(a.reshape(-1), c.reshape(-1)) for a, c in zip((q, s, t), flat))


# ------------------------------------------------- streams, graphs, repeats --
def test_streams_and_graphs(ops):  # noqa: F811
    """The layer's calls one after the other, eager, on another stream and in a
    captured graph, whose replays follow eager work and waits."""
    say("q8 streams and graphs")
    x, r = rand((333, 500), 1, BF).cuda(), rand((333, 500), 2, F32).cuda()
    w, sw, _ = ops.norm_q8(rand((501, 500), 3, BF, 0.05).cuda(), kind=None)  # packed rows
    b = rand((501,), 4, F32).cuda()

    def layer():
        q, s, t = ops.norm_q8(x, residual=r, kind="rms")
        y = ops.linear_q8(q, s, w, sw, bias=b, activation="gelu")
        few = ops.linear_q8(q[:9], s[:9], w, sw, bias=b, activation="gelu")
        return [q, s, t, y, few, *ops.add_norm(y, y, kind="layer")]
    want = layer()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = layer()
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(want, other))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        out = layer()
    for _ in range(4):
        for t in out:
            t.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(want, out))
        assert all(torch.equal(a, c) for a, c in zip(want, layer()))


# ---------------------------------------------------------------- refusals --
def test_refusals(ops):  # noqa: F811
    from browservec_amd import _lib as L

    say("q8 refusals")
    x, w, sx, sw = codes((4, 16), 1).cuda(), codes((8, 16), 2).cuda(), scales(4, 3).cuda(), scales(8, 4).cuda()
    h, f = rand((4, 16), 5, BF).cuda(), rand((4, 16), 6, F32).cuda()
    buf = rand((8, 32), 7, F32).cuda()
    for fn in (
        lambda: ops.linear_q8(x, sx, w[:, :8], sw),
        lambda: ops.linear_q8(x.float(), sx, w, sw),
        lambda: ops.linear_q8(x, sx, w.to(torch.uint8), sw),
        lambda: ops.linear_q8(x, sx[:3], w, sw),
        lambda: ops.linear_q8(x, sx.double(), w, sw),
        lambda: ops.linear_q8(x, sx, w, sw[:7]),
        lambda: ops.linear_q8(x, sx, w, sw.to(HF)),
        lambda: ops.linear_q8(x, sx, w, sw, bias=sx),
        lambda: ops.linear_q8(x, sx, w, sw, bias=sw.double()),
        lambda: ops.linear_q8(x, sx, w, sw, residual=h),
        lambda: ops.linear_q8(x, sx, w, sw, residual=f[:, :8].double()),
        lambda: ops.linear_q8(x, sx, w, sw, residual=f[:, :8], out_dtype=BF),
        lambda: ops.linear_q8(x, sx, w, sw, out_dtype=I8),
        lambda: ops.linear_q8(x, sx, w, sw, activation="tanh"),
        lambda: ops.linear_q8(x, sx, w.cpu(), sw),
        lambda: ops.linear_q8(x, sx.cpu(), w, sw),
        lambda: ops.linear_q8(x[:, :1].expand(4, 131072), sx, w[:, :1].expand(8, 131072), sw),
        lambda: ops.linear_q8(x, sx, w, sw, out=torch.empty(1, 8, device="cuda").expand(4, 8)),
        lambda: ops.linear_q8(x, buf[0, :4], w, sw, out=buf[:4, :8]),
        lambda: ops.add_norm(h, h.to(HF)),
        lambda: ops.add_norm(f, h),
        lambda: ops.add_norm(h, h[:3]),
        lambda: ops.add_norm(h, None),
        lambda: ops.add_norm(h, h, kind="batch"),
        lambda: ops.add_norm(h, h, eps=-1.0),
        lambda: ops.add_norm(h, h, weight=sx),
        lambda: ops.add_norm(h, h, out_dtype=I8),
        lambda: ops.add_norm(h, f, total=h),
        lambda: ops.add_norm(h, f, total=f[:3]),
        lambda: ops.add_norm(f, f.clone(), total=f, out=f),
        lambda: ops.add_norm(f[:, :8], f[:, 8:], total=f[:, 4:12]),
        lambda: ops.add_norm(f[:, :8], f[:, 8:], out=f[:, 6:14]),
        lambda: ops.add_norm(h.cpu(), h),
        lambda: ops.add_norm(*(rand((2, 16385), 1, BF).cuda(),) * 2),
        lambda: ops.norm_q8(h, out=h),
        lambda: ops.norm_q8(h, scales=sx[:3]),
        lambda: ops.norm_q8(h, scales=buf[:4, 0]),
        lambda: ops.norm_q8(h, total=h),
        lambda: ops.norm_q8(x),
        lambda: ops.norm_q8(f[:, :8], residual=f[:, 8:], scales=f[0, :4]),
        lambda: ops.norm_q8(f[:, :8], residual=f[:, 8:], total=f[:, 8:], scales=f[1, 8:12]),
        lambda: ops.norm_q8(torch.tensor(1.0, device="cuda")),
        lambda: ops.norm_q8(f[:, :0]),
    ):
        with pytest.raises(L.BVError) as e:
            fn()
        assert e.value.code in (L.BV_E_INVALID, L.BV_E_UNSUPPORTED) and str(e.value)


def test_c_refusals(ops):  # noqa: F811
    from browservec_amd import _lib as L

    say("q8 refusals of the C entry points")
    lib = L.load()
    buf = torch.zeros(16384, dtype=torch.uint8, device="cuda")
    p = buf.data_ptr()

    def call(cls, fn, base, kw):
        a = cls(ctypes.sizeof(cls))
        for k, v in {**base, **kw}.items():
            setattr(a, k, v)
        return fn(ops.handle, ctypes.addressof(a))

    base = dict(out_dtype=2, activation=0, m=4, n=8, k=16, x=p, w=p + 1024, x_scales=p + 2048, w_scales=p + 2560, y=p + 4096)
    assert call(L.LinearQ8Args, lib.bv_embed_linear_q8, base, {}) == L.BV_OK
    for kw in (dict(size=8), dict(x=None), dict(w=None), dict(x_scales=None), dict(w_scales=None), dict(y=None), dict(x_stride=15),
               dict(y_stride=7), dict(out_dtype=3), dict(bias=p + 8192, bias_dtype=3), dict(activation=9), dict(x_scales=p + 2049),
               dict(y=p), dict(y=p + 2048), dict(y=p + 2590), dict(m=2 ** 62), dict(residual=p + 4098), dict(bias=p + 4096), dict(k=131072)):
        assert call(L.LinearQ8Args, lib.bv_embed_linear_q8, base, kw) in (L.BV_E_INVALID, L.BV_E_UNSUPPORTED), kw
        assert lib.bv_last_error()
    base = dict(dtype=2, residual_dtype=2, out_dtype=3, norm=2, dim=16, eps=1e-5, tokens=4, x=p, residual=p + 1024, total=p + 2048,
                y=p + 4096, scales=p + 8192)
    assert call(L.AddNormArgs, lib.bv_embed_add_norm, base, {}) == L.BV_OK
    for kw in (dict(size=8), dict(x=None), dict(residual=None), dict(y=None), dict(scales=None), dict(x_stride=15), dict(total_stride=8),
               dict(residual_dtype=1), dict(residual_dtype=3), dict(dtype=3), dict(out_dtype=4), dict(norm=3), dict(dim=0), dict(dim=16385),
               dict(weight=p + 512, weight_dtype=3), dict(total=p + 1026), dict(y=p + 2048), dict(scales=p + 4100), dict(scales=p + 8193),
               dict(scales=p + 4), dict(weight=p + 4096, weight_dtype=2), dict(tokens=2 ** 62), dict(eps=float("nan"))):
        assert call(L.AddNormArgs, lib.bv_embed_add_norm, base, kw) in (L.BV_E_INVALID, L.BV_E_UNSUPPORTED), kw
        assert lib.bv_last_error()
    ops.sync()
