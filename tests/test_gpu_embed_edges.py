"""Edges of the embedding operators' sizes, layouts and arguments, against plain
implementations in 64 bits where there are values to compare."""

import ctypes

import pytest
import torch

from tests.helpers import say
from tests.test_gpu_embed import BF, F32, HF, U, attention_want, cu_of, dev_cu, inside, linear_want, norm_want, ops, rand  # noqa: F401

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


# ------------------------------------------------------------------ outputs --
def test_outputs_that_overlap_themselves_are_refused(ops):  # noqa: F811
    """An expanded output holds fewer elements than its shape says."""
    from browservec_amd import _lib as L
    from browservec_amd import rotary_table

    say("outputs that overlap themselves")
    x, w = rand((6, 16), 1, BF).cuda(), rand((16, 16), 2, BF).cuda()
    q, cu, table = rand((6, 2, 8), 3, BF).cuda(), dev_cu([0, 6]), torch.from_numpy(rotary_table(6, 8)).cuda()
    row, head = torch.zeros(1, 16, dtype=BF, device="cuda"), torch.zeros(1, 1, 8, dtype=BF, device="cuda")
    one = torch.zeros(1, 16, dtype=F32, device="cuda")
    for fn in (
        lambda: ops.linear(x, w, out=row.expand(6, 16)),
        lambda: ops.linear(x, w, residual=row.expand(6, 16), out=row.expand(6, 16)),
        lambda: ops.linear(x.unflatten(0, (2, 3)), w, out=row.expand(2, 3, 16)),
        lambda: ops.norm(x, out=row.expand(6, 16)),
        lambda: ops.pool(x, dev_cu([0, 2, 6]), out=one.expand(2, 16)),
        lambda: ops.attention(q, q, q, cu, out=head.expand(6, 2, 8)),
        lambda: ops.attention(q[:1], q, q, dev_cu([0, 1]), cu, out=head.expand(1, 2, 8)),
        lambda: ops.rotary(q, None, table, out_q=head.expand(6, 2, 8)),
        lambda: ops.rotary(q, q.clone(), table, out_k=torch.zeros(6, 1, 8, dtype=BF, device="cuda").expand(6, 2, 8)),
    ):
        with pytest.raises(L.BVError) as e:
            fn()
        assert e.value.code == L.BV_E_INVALID
    assert not row.any() and not head.any() and not one.any()
    e = row.expand(6, 16)  # in place, of the input itself
    with pytest.raises(L.BVError):
        ops.norm(e, out=e)
    # inputs may be expanded: they are copied
    inside(ops.linear(x[:1].expand(6, 16), w), *linear_want(x[:1].expand(6, 16), w, None, None, "none", BF), "expanded input")


# --------------------------------------------------------- attention, sizes --
def attention_args(**kw):
    """One query head over one key head of 8 elements, packed, pointers that the checks accept."""
    from browservec_amd import _lib as L

    buf = torch.zeros(4096, dtype=BF, device="cuda")
    p = buf.data_ptr()
    a = L.AttentionArgs(ctypes.sizeof(L.AttentionArgs), 2, 1, 1, 8, 1, 1)
    a.tokens_q, a.tokens_k, a.q, a.k, a.v, a.o, a.cu_q, a.cu_k = 1, 1, p, p + 64, p + 128, p + 192, p + 256, p + 320
    for k, v in kw.items():
        setattr(a, k, v)
    return a, buf


@pytest.mark.parametrize("tokens_k", [2 ** 31 - 1024, 2 ** 31 - 128, 2 ** 31 - 1, 2 ** 31, 2 ** 40])
def test_attention_of_too_many_keys_is_refused(ops, tokens_k):  # noqa: F811
    """A tile's end has to fit 32 bits as well."""
    from browservec_amd import _lib as L

    say("attention, too many keys", tokens_k)
    a, buf = attention_args(tokens_k=tokens_k)
    assert L.load().bv_embed_attention(ops.handle, ctypes.addressof(a)) in (L.BV_E_INVALID, L.BV_E_UNSUPPORTED)
    assert b"attention" in L.load().bv_last_error()
    ops.sync()


@pytest.mark.parametrize("d", [1, 8])
def test_attention_of_the_most_keys(ops, d):  # noqa: F811
    """One sequence of as many keys as a call takes: the last one counts most,
    and the rest not nothing."""
    n = 2 ** 31 - 1025
    say("attention, the most keys", d)
    if torch.cuda.mem_get_info()[0] < 2 * n * d * 2 + 2 ** 32:
        pytest.skip("not enough device memory free")
    q = torch.ones(1, 1, d, dtype=BF, device="cuda")
    k, v = torch.zeros(n, 1, d, dtype=BF, device="cuda"), torch.ones(n, 1, d, dtype=BF, device="cuda")
    k[-1, 0, 0] = 22.0  # its weight against 2^31 others of 1: e^22 = 3.6e9
    v[-1] = -1.0
    o = ops.attention(q, k, v, dev_cu([0, 1]), dev_cu([0, n]), scale=1.0)
    top = torch.exp(torch.tensor(22.0, dtype=torch.float64))
    want = ((n - 1 - top) / (n - 1 + top)).expand(1, 1, d)
    # weights are exact but for the last one's exponential, within 2^-17 of its
    # value, and sums of 2^31 terms by 128 parts of 2^24, each exact in 32 bits up to 2^24
    inside(o, want, U[BF] * want.abs() * 1.01 + 2 * 2.0 ** -16, "the most keys")
    del q, k, v, o
    torch.cuda.empty_cache()


# ------------------------------------------------------------ linear, sizes --
def test_linear_of_rows_past_32_bits(ops):  # noqa: F811
    """The elements after the last whole step lie past 2^31 in their row."""
    k = 2 ** 31 + 5
    say("linear, rows of 2^31 + 5")
    if torch.cuda.mem_get_info()[0] < 5 * 2 ** 32:
        pytest.skip("not enough device memory free")
    x, w = torch.zeros(1, k, dtype=BF, device="cuda"), torch.zeros(1, k, dtype=BF, device="cuda")
    for at, a, b in ((0, 3, 5), (2 ** 31 - 1, 2, 7), (2 ** 31, 4, 11), (k - 1, 8, 13)):
        x[0, at], w[0, at] = a, b
    y = ops.linear(x, w, out_dtype=F32)
    assert y.item() == 3 * 5 + 2 * 7 + 4 * 11 + 8 * 13  # exact in 32 bits
    del x, w
    torch.cuda.empty_cache()


@pytest.mark.parametrize("m,n,k", [(40, 3, 2 ** 26), (33, 17, 2 ** 22 + 3)])
def test_linear_of_long_rows(ops, m, n, k):  # noqa: F811
    """Tens of rows so long that some lie 2^32 bytes and more after the first,
    as one tile would address them."""
    say("linear, long rows", m, n, k)
    if torch.cuda.mem_get_info()[0] < 2 * (m + n) * k + 2 ** 32:
        pytest.skip("not enough device memory free")
    x, w = torch.zeros(m, k, dtype=BF, device="cuda"), torch.zeros(n, k, dtype=BF, device="cuda")
    a, b = torch.arange(1, m + 1).to(BF).cuda(), torch.arange(1, n + 1).to(BF).cuda()
    for at in (0, 1000, k - 1):
        x[:, at], w[:, at] = a, b
    r = rand((m, n), 3, BF).round().cuda()
    y = ops.linear(x, w, residual=r, out=torch.empty(m, n + 5, dtype=BF, device="cuda")[:, 2:n + 2])
    want = 3 * a.double()[:, None] * b.double() + r.double()  # exact in 32 bits, rounded once
    assert torch.equal(y, want.to(BF))
    del x, w
    torch.cuda.empty_cache()


def test_linear_of_many_columns(ops):  # noqa: F811
    """More columns than one launch's 2^32 threads reach."""
    m, n = 2, 2 ** 27 + 40
    say("linear, 2^27 + 40 columns")
    w = (torch.arange(n, device="cuda") % 127).to(BF)[:, None]
    x, b = torch.tensor([[1.0], [-2.0]], dtype=BF, device="cuda"), (torch.arange(n, device="cuda") % 3).to(BF)
    r = torch.ones(m, n, dtype=BF, device="cuda")
    y = ops.linear(x, w, bias=b, residual=r)
    assert torch.equal(y, (x.float() * w[:, 0].float() + b.float() + 1).to(BF))  # exact in 32 bits
    del w, b, r, y
    torch.cuda.empty_cache()


# ------------------------------------------------------------- rows, sizes --
def test_norm_of_more_rows_than_a_launch(ops):  # noqa: F811
    """Rows of 16 waves, one a workgroup: 2^22 workgroups are 2^32 threads."""
    rows, dim = 2 ** 22 + 100, 4104
    say("norm of 2^22 + 100 rows")
    if torch.cuda.mem_get_info()[0] < 2 * rows * dim + 2 ** 32:
        pytest.skip("not enough device memory free")
    x = torch.full((rows, dim), 3.0, dtype=BF, device="cuda")
    ops.norm(x, kind="rms", out=x)  # 3 / sqrt(9 + 1e-5) is 1 in bfloat16
    assert all((x[a:a + 2 ** 17] == 1).all() for a in range(0, rows, 2 ** 17))
    del x
    torch.cuda.empty_cache()


@pytest.mark.parametrize("mode", ["mean", "last"])
def test_pool_of_more_sequences_than_a_launch(mode):
    """The same of sequences, nearly all of them empty: the first and the last are not."""
    from browservec_amd import DeviceContext, EmbedOps
    from tests.helpers import need_gpu

    need_gpu()
    n, dim = 2 ** 22 + 100, 4104
    say("pool of 2^22 + 100 sequences", mode)
    if torch.cuda.mem_get_info()[0] < 8 * n * dim + 2 ** 32:  # the result and as many partial sums
        pytest.skip("not enough device memory free")
    ctx = DeviceContext(0)
    e = EmbedOps(ctx)
    x = torch.cat([torch.full((2, dim), 2.0), torch.full((3, dim), -5.0)]).to(BF).cuda()
    cu = torch.full((n + 1,), 2, dtype=torch.int32, device="cuda")
    cu[0], cu[-1] = 0, 5
    y = torch.full((n, dim), 7.0, device="cuda")
    e.pool(x, cu, mode=mode, unit=False, out=y)
    assert (y[0] == 2).all() and (y[-1] == -5).all()
    assert all((y[a:min(n - 1, a + 2 ** 17)] == 0).all() for a in range(1, n - 1, 2 ** 17))
    del x, y, cu
    torch.cuda.empty_cache()
    e.destroy()
    ctx.destroy()


# ------------------------------------------------------------------- graphs --
def test_graphs_run_beside_each_other(ops):  # noqa: F811
    """Two graphs of calls that need workspaces, captured on one stream, replayed
    on two streams at once, with eager calls on a third: none uses another's
    workspace."""
    say("graphs beside each other")

    def calls(seed):
        x, w = rand((700, 1003), seed, BF).cuda(), rand((500, 1003), seed + 1, BF, 0.05).cuda()  # packed rows
        rows = rand((6000, 520), seed + 2, HF).cuda()  # partial sums
        q, k, v = (rand((n, h, 64), seed + i, BF).cuda() for i, (n, h) in enumerate([(3, 8), (9000, 2), (9000, 2)], 3))  # split keys
        cu, cq, ck = dev_cu([0, 2500, 6000]), dev_cu([0, 1, 3]), dev_cu([0, 4000, 9000])
        return [lambda: ops.linear(x, w), lambda: ops.pool(rows, cu, kind="layer"),
                lambda: ops.attention(q, k, v, cq, ck, max_q=2, max_k=5000)]

    sets = [calls(10), calls(50), calls(90)]
    want = [[f() for f in fns] for fns in sets]
    torch.cuda.synchronize()
    capture, streams = torch.cuda.Stream(), [torch.cuda.Stream() for _ in range(2)]
    graphs, outs = [], []
    for fns in sets[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=capture):
            outs.append([[f() for f in fns] for _ in range(4)])
        graphs.append(g)
    for _ in range(5):
        for o in (t for out in outs for row in out for t in row):
            o.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(capture):
            eager = [[f() for f in sets[2]] for _ in range(4)]
        torch.cuda.synchronize()
        for out, w in zip(outs + [eager], want):
            for row in out:
                assert all(torch.equal(a, b) for a, b in zip(row, w))


def test_a_capture_on_a_stream_without_calls_before(ops):  # noqa: F811
    """Workspaces that a capture is the first to need."""
    say("capture without calls before")
    rows, cu = rand((5000, 264), 1, BF).cuda(), dev_cu([0, 5000])
    want = ops.pool(rows, cu)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.Stream()):
        out = ops.pool(rows, cu)
    for _ in range(3):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert torch.equal(ops.pool(rows, cu), want)


# -------------------------------------------------------- attention, values --
@pytest.mark.parametrize("nq,nk,low", [(200, 200, 100), (200, 200, 64), (8, 200, 190), (8, 3000, 2900), (40, 3000, 2900), (150, 150, 10)])
def test_attention_of_keys_that_score_minus_infinity(ops, nq, nk, low):  # noqa: F811
    """Keys at the front that weigh nothing, a value at the end that only the last
    query sees and that is not finite: the other queries' results are those of the
    finite keys."""
    say("attention, scores of -inf", nq, nk, low)
    hq, hk, d = 4, 2, 64
    q, k, v = rand((nq, hq, d), 1, BF), rand((nk, hk, d), 2, BF), rand((nk, hk, d), 3, BF)
    q[:, :, 0] = q[:, :, 0].abs() + 0.5
    k[:low, :, 0] = float("-inf")
    v[-1, :, 5] = float("nan")
    first = max(0, low - (nk - nq))  # the first query that sees a finite key
    for hints in (dict(), dict(max_q=nq, max_k=nk)):
        o = ops.attention(q.cuda(), k.cuda(), v.cuda(), dev_cu([0, nq]), dev_cu([0, nk]), **hints).cpu()
        assert torch.isnan(o[:first]).all()  # 0 / 0
        want, bound = attention_want(q[first:], k[low:], v[low:], [0, nq - first], [0, nk - low], True)
        inside(o[first:-1], want[:-1], bound[:-1], f"scores of -inf {hints}")
        assert torch.isnan(o[-1, :, 5]).all() and torch.isfinite(o[-1, :, :5]).all()


# ------------------------------------------------------------------ rotary --
FUSED = {  # a fused product's queries, keys and values as [tokens, heads, d] views
    "tokens, 3, heads, d": lambda t, h, d: [x for x in rand((t, 3, h, d), 1, BF).cuda().unbind(1)],
    "tokens, heads, 3 d": lambda t, h, d: rand((t, h, 3 * d), 1, BF).cuda().split(d, 2),
    "tokens, heads, 3 d + 1": lambda t, h, d: rand((t, h, 3 * d + 1), 1, BF).cuda()[:, :, 1:].split(d, 2),
    "heads, tokens, 3 d": lambda t, h, d: [x.transpose(0, 1) for x in rand((h, t, 3 * d), 1, BF).cuda().split(d, 2)],
    "heads, 3, tokens, d": lambda t, h, d: [x.transpose(0, 1) for x in rand((h, 3, t, d), 1, BF).cuda().unbind(1)],
    "tokens, 3 heads d + 5": lambda t, h, d: [x.unflatten(1, (h, d)) for x in rand((t, 3 * h * d + 5), 1, BF).cuda()[:, :3 * h * d].split(h * d, 1)],
}


@pytest.mark.parametrize("layout", FUSED)
@pytest.mark.parametrize("tokens,heads", [(37, 4), (1, 4), (37, 1), (1, 1)])
def test_rotary_of_fused_layouts_in_place(ops, layout, tokens, heads):  # noqa: F811
    from browservec_amd import rotary_table

    say("rotary in place", layout, tokens, heads)
    table = torch.from_numpy(rotary_table(64, 16)).cuda()
    q, k, v = FUSED[layout](tokens, heads, 32)
    want = ops.rotary(q, k, table)
    before = v.clone()
    got = ops.rotary(q, k, table, out_q=q, out_k=k)
    assert got[0] is q and torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(v, before)


def test_rotary_outputs_that_overlap_are_refused(ops):  # noqa: F811
    """Heads of queries and keys are turned in no order: neither output may be
    the other's input or output."""
    from browservec_amd import _lib as L
    from browservec_amd import rotary_table

    say("rotary outputs that overlap")
    table = torch.from_numpy(rotary_table(64, 16)).cuda()
    q, k, _ = FUSED["tokens, 3, heads, d"](9, 4, 32)
    fused = rand((9, 5, 32), 2, BF).cuda()
    own = torch.empty(9, 4, 32, dtype=BF, device="cuda")
    before = [t.clone() for t in (q, k, fused)]
    for kw in (dict(out_q=k), dict(out_k=q), dict(out_q=k, out_k=q), dict(out_q=own, out_k=own), dict(out_q=q, out_k=q)):
        with pytest.raises(L.BVError) as e:
            ops.rotary(q, k, table, **kw)
        assert e.value.code == L.BV_E_INVALID and "overlaps" in str(e.value)
    for kw in (dict(out_q=fused[:, :4]), dict(out_q=fused[:, 1:]), dict(out_k=fused[:, :4])):  # one head in common
        with pytest.raises(L.BVError):
            ops.rotary(fused[:, 1:] if "out_k" in kw else q, fused[:, :4] if "out_q" in kw else k, table, **kw)
    assert all(torch.equal(a, b) for a, b in zip((q, k, fused), before))


# --------------------------------------------------------- attention, scale --
def test_attention_scale_of_zero_is_refused(ops):  # noqa: F811
    """Weights would all be equal; the library's 0 means the default."""
    from browservec_amd import _lib as L

    say("attention, scale 0")
    q, cu = rand((4, 2, 8), 1, BF).cuda(), dev_cu([0, 4])
    for scale in (0, 0.0, -0.0, 1e-60):
        with pytest.raises(L.BVError) as e:
            ops.attention(q, q, q, cu, scale=scale)
        assert e.value.code == L.BV_E_INVALID and "scale" in str(e.value)
    # as small as 32 bits hold: all weights equal
    o = ops.attention(q, q, q, cu, causal=False, scale=1e-38)
    want = q.cpu().double().mean(0, keepdim=True).expand(4, 2, 8)
    inside(o, want, U[BF] * want.abs() * 1.01 + 2.0 ** -16, "equal weights")
    assert torch.equal(ops.attention(q, q, q, cu, scale=None), ops.attention(q, q, q, cu, scale=8 ** -0.5))


# ------------------------------------------------------------------- counts --
def test_dimensions_past_32_bits_are_refused(ops):  # noqa: F811
    """Their low 32 bits would fit, and give part of a result.  (Expanded
    tensors: nothing of the size is allocated.)"""
    from browservec_amd import _lib as L

    say("dimensions past 32 bits")
    many = 2 ** 32 + 8
    one, cu = torch.zeros(1, 1, dtype=BF, device="cuda"), dev_cu([0, 1])
    heads = torch.zeros(1, 1, 1, dtype=BF, device="cuda")
    table = torch.zeros(4, 0, 2, device="cuda")
    for fn in (
        lambda: ops.linear(one, one.expand(many, 1)),
        lambda: ops.linear(one.expand(1, many), one.expand(1, many)),
        lambda: ops.rotary(heads.expand(1, many, 1), None, table),
        lambda: ops.rotary(heads, heads.expand(1, many, 1), table),
        lambda: ops.rotary(heads.expand(1, 1, many), None, table),
        lambda: ops.rotary(heads, None, torch.zeros(many, 0, 2, device="cuda")),
        lambda: ops.attention(heads.expand(1, many, 1), heads, heads, cu, out=heads.expand(1, many, 1)),
        lambda: ops.attention(heads, heads.expand(1, many, 1), heads.expand(1, many, 1), cu),
        lambda: ops.attention(*(heads.expand(1, 1, many),) * 3, cu, out=heads.expand(1, 1, many)),
        lambda: ops.norm(one.expand(1, many), out=one.expand(1, many)),
        lambda: ops.pool(one.expand(1, many), cu, out=torch.zeros(1, 1, device="cuda").expand(1, many)),
    ):
        with pytest.raises(L.BVError) as e:
            fn()
        assert e.value.code == L.BV_E_UNSUPPORTED and "32 bits" in str(e.value)


# ----------------------------------------------------- attention, workspace --
def bidirectional_want(q, k, v, cu_q, cu_k):
    """attention_want without a mask, its products on the GPU."""
    u, group, scale = U[q.dtype], q.shape[1] // k.shape[1], q.shape[2] ** -0.5
    out, bound = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    for a, e, ka, ke in zip(cu_q, cu_q[1:], cu_k, cu_k[1:]):
        if e == a or ke == ka:
            continue
        for h in range(q.shape[1]):
            qq, kk, vv = q[a:e, h].double(), k[ka:ke, h // group].double(), v[ka:ke, h // group].double()
            s = scale * (qq @ kk.t().contiguous())
            p = torch.exp(s - s.amax(1, keepdim=True))
            total = p.sum(1, keepdim=True)
            delta = (q.shape[2] + 2) * 2.0 ** -23 * scale * (qq.abs() @ kk.abs().t().contiguous()).amax(1, keepdim=True)
            x = p @ vv / total
            b = p @ vv.abs() / total * (u + 4 * delta + 2.0 ** -16 + 2 * (ke - ka) * 2.0 ** -24) + u * x.abs() * 1.01
            if q.dtype == HF:
                b += 2.0 ** -24 * (1 + vv.abs().sum(0, keepdim=True) / total)
            out[a:e, h], bound[a:e, h] = x.cpu(), b.cpu()
    return out, bound


def test_attention_without_lengths_takes_little_memory():
    """Parts of the keys are made for one sequence that might have all of them,
    but not without end: 64 sequences of 600 keys, their lengths not said."""
    from browservec_amd import DeviceContext, EmbedOps
    from tests.helpers import need_gpu

    need_gpu()
    say("attention, workspace")
    ctx = DeviceContext(0)
    e = EmbedOps(ctx)
    hq, hk, d = 32, 1, 256
    cq, ck = cu_of([12] * 64), cu_of([600] * 64)
    q, k, v = rand((cq[-1], hq, d), 1, BF, 1.5).cuda(), rand((ck[-1], hk, d), 2, BF).cuda(), rand((ck[-1], hk, d), 3, BF).cuda()
    o, dq, dk = torch.empty_like(q), dev_cu(cq), dev_cu(ck)
    torch.cuda.synchronize()
    free = torch.cuda.mem_get_info()[0]
    e.attention(q, k, v, dq, dk, causal=False, out=o)
    torch.cuda.synchronize()
    taken = free - torch.cuda.mem_get_info()[0]
    inside(o, *bidirectional_want(q, k, v, cq, ck), "without lengths")
    e.destroy()
    ctx.destroy()
    assert taken < 2 ** 28 + 2 ** 25, taken


# ------------------------------------------------------------------- shapes --
def test_shapes_of_other_than_two_dimensions(ops):  # noqa: F811
    """Rows in any number of dimensions; outputs of theirs that are no rows at
    one stride are refused, not left to torch."""
    from browservec_amd import _lib as L

    say("shapes")
    x, w = rand((4, 5, 16), 1, BF).cuda(), rand((8, 16), 2, BF).cuda()
    flat = ops.linear(x.flatten(0, 1), w)
    y = torch.zeros(4, 5, 12, dtype=BF, device="cuda")
    assert torch.equal(ops.linear(x, w, out=y[:, :, 2:10]).flatten(0, 1), flat)
    assert torch.equal(ops.linear(x.transpose(0, 1), w).transpose(0, 1).flatten(0, 1), flat)
    assert torch.equal(ops.linear(x[1, 2], w), flat[7])
    n = ops.norm(x)
    assert torch.equal(n, ops.norm(x.flatten(0, 1)).view(4, 5, 16)) and torch.equal(ops.norm(x[1, 2]), n[1, 2])
    t = x.transpose(0, 1)
    scalar = torch.zeros((), dtype=BF, device="cuda")
    for fn in (lambda: ops.linear(x, w, out=torch.zeros(5, 4, 8, dtype=BF, device="cuda").transpose(0, 1)),
               lambda: ops.linear(x, w, out=torch.zeros(4, 6, 8, dtype=BF, device="cuda")[:, :5]),
               lambda: ops.norm(t, out=t), lambda: ops.norm(scalar), lambda: ops.linear(scalar, w)):
        with pytest.raises(L.BVError) as e:
            fn()
        assert e.value.code == L.BV_E_INVALID


def test_sums_and_results_of_nothing(ops):  # noqa: F811
    say("sums and results of nothing")
    x, w, b = rand((2, 3, 16), 1, BF).cuda(), rand((8, 16), 2, BF).cuda(), rand((8,), 3, BF).cuda()
    assert torch.equal(ops.linear(x[:, :, :0], w[:, :0], bias=b), b.expand(2, 3, 8))
    assert ops.linear(x, w[:0]).shape == (2, 3, 0) and ops.linear(x[:, :0], w).shape == (2, 0, 8)
    assert torch.equal(ops.linear(x[0, 0, :0], w[:, :0], bias=b), b)
    assert ops.norm(x[:, :0]).shape == (2, 0, 16)


@pytest.mark.parametrize("tokens,heads,strides", [(1, 1, (1, 1, 1)), (1, 1, (3, 5, 1)), (1, 3, (2, 24, 1)), (6, 1, (24, 1, 1))])
def test_strides_of_a_single_token_or_head(ops, tokens, heads, strides):  # noqa: F811
    """They mean nothing, and a contiguous tensor may have any."""
    from browservec_amd import rotary_table

    say("strides of one", tokens, heads, strides)
    d = 24
    flat = [rand((200,), i, HF).cuda() for i in range(4)]
    odd = [t.as_strided((tokens, heads, d), strides) for t in flat]
    q, k, v = (t.clone(memory_format=torch.contiguous_format) for t in odd[:3])
    cu = dev_cu([0, tokens])
    want = ops.attention(q, k, v, cu)
    assert torch.equal(ops.attention(*odd[:3], cu, out=odd[3]), want)
    table = torch.from_numpy(rotary_table(8, 16)).cuda()
    want = ops.rotary(q, k, table)
    got = ops.rotary(*odd[:2], table, out_q=odd[0], out_k=odd[1])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


# ------------------------------------------- paths of larger calls, both signs --
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("m,n,k", [(4096, 768, 768), (4100, 1030, 203), (6000, 1500, 264), (9000, 1400, 203), (8200, 4100, 520)])
def test_linear_32_bit_results_of_large_tiles(ops, m, n, k, dtype):  # noqa: F811
    """32-bit results and residuals out of tiles of 128 x 128 and 256 x 256."""
    say("linear, 32-bit results", m, n, k, dtype)
    x, w, b = rand((m, k), 1, dtype).cuda(), rand((n, k), 2, dtype, k ** -0.5).cuda(), rand((n,), 3, dtype).cuda()
    r = rand((m, n), 4, F32).cuda()
    y = ops.linear(x, w, bias=b, residual=r, activation="gelu_tanh", out_dtype=F32)
    xd, wd, bd = x.double(), w.double(), b.double()
    z = xd @ wd.t().contiguous() + bd
    mag = xd.abs() @ wd.abs().t().contiguous() + bd.abs()
    c = 2 * (2 / torch.pi) ** 0.5
    want = z * torch.sigmoid(c * (z + 0.044715 * z ** 3)) + r.double()
    bound = 1.13 * (k + 2) * 2.0 ** -23 * mag + 2.0 ** -20 * z.abs().clamp(min=1) + 2.0 ** -23 * want.abs()
    inside(y, want.cpu(), (bound + U[F32] * (want.abs() + bound)).cpu(), "32-bit results")


@pytest.mark.parametrize("scale", [-0.3, -1e-3])
@pytest.mark.parametrize("d,dtype", [(64, BF), (80, HF), (17, BF), (128, HF), (200, BF)])
@pytest.mark.parametrize("nq,nk", [([70, 0, 130], [70, 5, 200]), ([1, 3], [900, 40])])
def test_attention_of_negative_scale(ops, nq, nk, d, dtype, scale):  # noqa: F811
    """Queries change sign before the products; also in rows done one by one,
    where a value that some do not see is not finite."""
    say("attention, negative scale", nq, nk, d, dtype, scale)
    cq, ck = cu_of(nq), cu_of(nk)
    q, k, v = rand((cq[-1], 4, d), 1, dtype, 1.5), rand((ck[-1], 2, d), 2, dtype), rand((ck[-1], 2, d), 3, dtype)
    want, bound = attention_want(q, k, v, cq, ck, True, scale=scale)
    want_p, bound_p = attention_want(-q, k, v, cq, ck, True, scale=-scale)
    assert torch.equal(want, want_p)  # the bound's sizes are those of the scores
    args = [t.cuda() for t in (q, k, v)]
    o = ops.attention(*args, dev_cu(cq), dev_cu(ck), scale=scale)
    inside(o, want, bound_p, "negative scale")
    assert torch.equal(o, ops.attention(-args[0], *args[1:], dev_cu(cq), dev_cu(ck), scale=-scale))
    args[2][-1] = float("inf")
    o = ops.attention(*args, dev_cu(cq), dev_cu(ck), scale=scale).cpu()
    inside(o[:-1], want[:-1], bound_p[:-1], "negative scale, rows one by one")


@pytest.mark.parametrize("hq,hk,d,dtype", [(12, 12, 96, BF), (8, 8, 128, HF), (16, 4, 128, BF), (12, 4, 112, HF)])
def test_attention_of_hundreds_of_short_texts(ops, hq, hk, d, dtype):  # noqa: F811
    """Bidirectional, as an encoder's: more texts than compute units, of lengths
    that end inside tiles, enough rows for the kernel of eight waves; a value that
    is not finite stays in its text."""
    lens = [(1, 17, 64, 65, 128, 200, 0, 333, 100, 256)[i % 10] for i in range(430)]
    say("attention, short texts", hq, hk, d, dtype)
    cu = cu_of(lens)
    t = cu[-1]
    q, k, v = rand((t, hq, d), 1, dtype, 1.5).cuda(), rand((t, hk, d), 2, dtype).cuda(), rand((t, hk, d), 3, dtype).cuda()
    o = ops.attention(q, k, v, dev_cu(cu), causal=False)
    want, bound = bidirectional_want(q, k, v, cu, cu)
    inside(o, want, bound, "short texts")
    assert torch.equal(o, ops.attention(q, k, v, dev_cu(cu), causal=False, max_q=max(lens), max_k=max(lens)))
    s = 207  # 333 tokens
    assert lens[s] == 333
    v[cu[s] + 300, :, d // 2] = float("nan")
    again = ops.attention(q, k, v, dev_cu(cu), causal=False)
    same = torch.ones(t, dtype=torch.bool, device="cuda")
    same[cu[s]:cu[s + 1]] = False
    assert torch.equal(again[same], o[same])
    mine = again[cu[s]:cu[s + 1]]
    assert torch.isnan(mine[:, :, d // 2]).all() and torch.isfinite(mine[:, :, :d // 2]).all()
