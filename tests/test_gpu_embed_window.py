"""Attention with a window of keys and first keys (EmbedOps.attention, window and
sinks) against its formula in 64 bits."""

import pytest
import torch

from tests.helpers import say
from tests.test_gpu_embed import BF, HF, U, cu_of, dev_cu, inside, ops, rand  # noqa: F401

pytestmark = pytest.mark.gpu
ALL = 2 ** 40


def seen_of(nq, nk, causal, left, right, sinks, device="cpu"):
    """[nq, nk]: which keys each query sees."""
    p = torch.arange(nq, device=device)[:, None] + nk - nq
    j = torch.arange(nk, device=device)[None]
    seen = ((j >= p - (ALL if left is None else left)) & (j <= p + (ALL if right is None else right))) | (j < sinks)
    return seen & (j <= p) if causal else seen


def window_want(q, k, v, cu_q, cu_k, causal, left, right, sinks, scale=None):
    """The result in 64 bits and its bound (as attention_want's: scores within (d +
    2) 2^-23 sum |q k| scale, exponentials within 2^-17, weights rounded to the type
    once, or by 2^-25 in float16, sums of n terms, one rounding at the end)."""
    u, group, scale = U[q.dtype], q.shape[1] // k.shape[1], scale or q.shape[2] ** -0.5
    out, bound = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    for a, e, ka, ke in zip(cu_q, cu_q[1:], cu_k, cu_k[1:]):
        if e <= a or ke <= ka:
            continue
        seen = seen_of(e - a, ke - ka, causal, left, right, sinks, q.device)
        none, n = ~seen.any(1, keepdim=True), seen.sum(1, keepdim=True)
        for h in range(q.shape[1]):
            qq, kk, vv = q[a:e, h].double(), k[ka:ke, h // group].double(), v[ka:ke, h // group].double()
            s = (scale * (qq @ kk.t().contiguous())).masked_fill(~seen, float("-inf"))
            size = (abs(scale) * (qq.abs() @ kk.abs().t().contiguous())).masked_fill(~seen, 0).amax(1, keepdim=True)
            p = torch.exp(s - s.amax(1, keepdim=True)).masked_fill(none, 0)
            total = p.sum(1, keepdim=True).masked_fill(none, 1)
            x = p @ vv / total
            delta = (q.shape[2] + 2) * 2.0 ** -23 * size
            b = p @ vv.abs() / total * (u + 4 * delta + 2.0 ** -16 + 2 * n * 2.0 ** -24) + u * x.abs() * 1.01
            if q.dtype == HF:
                b += 2.0 ** -24 * (1 + seen.double() @ vv.abs() / total) * ~none
            out[a:e, h], bound[a:e, h] = x.cpu(), b.cpu()
    return out, bound


WINDOWS = [(0, 0, 0), (3, 5, 0), (64, 64, 0), (31, 33, 70), (100, 0, 4), (7, None, 3), (None, 2, 0), (0, 200, 1), (None, None, 5),
           (2 ** 31, 2 ** 35, 2 ** 33), (1, 1, 2 ** 31)]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("hq,hk,d,dtype", [(4, 4, 32, BF), (6, 2, 64, HF), (8, 1, 128, BF), (3, 3, 80, HF), (4, 2, 96, BF),
                                           (2, 1, 1, BF), (5, 5, 17, HF), (2, 2, 256, BF)])
@pytest.mark.parametrize("lens", [[1], [17], [0, 3, 0, 64, 65, 1, 0], [129, 2, 31], [400]])
def test_window_packed(ops, lens, hq, hk, d, dtype, causal):  # noqa: F811
    say("window", lens, hq, hk, d, dtype, causal)
    cu = cu_of(lens)
    q, k, v = rand((cu[-1], hq, d), 1, dtype, 1.5).cuda(), rand((cu[-1], hk, d), 2, dtype).cuda(), rand((cu[-1], hk, d), 3, dtype).cuda()
    for left, right, sinks in WINDOWS:
        o = ops.attention(q, k, v, dev_cu(cu), causal=causal, window=(left, right), sinks=sinks)
        inside(o, *window_want(q, k, v, cu, cu, causal, left, right, sinks), f"window {left} {right} {sinks}")


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("hq,hk,d", [(4, 1, 64), (16, 16, 32), (6, 2, 128)])
@pytest.mark.parametrize("nq,nk", [([1], [700]), ([1, 1, 1], [1, 0, 333]), ([4, 2], [65, 1000]), ([5, 3, 130], [2, 3, 64]),
                                   ([64, 0, 1], [1500, 20, 64]), ([1] * 40, list(range(1, 81, 2))), ([300], [40])])
def test_window_over_kept_keys(ops, nq, nk, hq, hk, d, causal):  # noqa: F811
    """New tokens over kept keys; more queries than keys, whose first ones may see
    nothing."""
    say("window kept", nq, nk, hq, hk, d, causal)
    cq, ck = cu_of(nq), cu_of(nk)
    q, k, v = rand((cq[-1], hq, d), 1, BF, 1.5).cuda(), rand((ck[-1], hk, d), 2, BF).cuda(), rand((ck[-1], hk, d), 3, BF).cuda()
    for left, right, sinks in [(0, 0, 0), (100, 3, 4), (500, 0, 70), (40, 40, 0), (None, 0, 1), (3, None, 0)]:
        want = window_want(q, k, v, cq, ck, causal, left, right, sinks)
        for hints in (dict(), dict(max_q=max(nq), max_k=max(nk)), dict(max_q=1, max_k=1), dict(max_q=1, max_k=100000)):
            o = ops.attention(q, k, v, dev_cu(cq), dev_cu(ck), causal=causal, window=(left, right), sinks=sinks, **hints)
            inside(o, *want, f"window kept {left} {right} {sinks} {hints}")


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("hq,hk,d,dtype,lens,window,sinks", [
    (16, 4, 128, BF, [5000, 1, 3300], (1000, 200), 4), (8, 8, 96, HF, [9000], (64, 64), 0), (16, 16, 80, HF, [2049, 3000], (300, 300), 130),
    (12, 12, 64, BF, [4097, 511], (64, 64), 0), (16, 2, 128, BF, [8200], (4095, 0), 4), (8, 8, 256, HF, [2500], (513, 100), 1)])
def test_window_long(ops, hq, hk, d, dtype, lens, window, sinks, causal):  # noqa: F811
    say("window long", hq, hk, d, dtype, lens, window, sinks, causal)
    cu = cu_of(lens)
    q, k, v = rand((cu[-1], hq, d), 1, dtype, 1.5).cuda(), rand((cu[-1], hk, d), 2, dtype).cuda(), rand((cu[-1], hk, d), 3, dtype).cuda()
    o = ops.attention(q, k, v, dev_cu(cu), causal=causal, window=window, sinks=sinks)
    inside(o, *window_want(q, k, v, cu, cu, causal, *window, sinks), "window long")


@pytest.mark.parametrize("hq,hk,d,dtype", [(16, 4, 64, BF), (8, 2, 128, HF), (12, 12, 32, BF)])
def test_window_next_tokens(ops, hq, hk, d, dtype):  # noqa: F811
    """Many sequences' next tokens, keys split and joined."""
    say("window next tokens", hq, hk, d, dtype)
    nk = [20000, 1, 5000, 300, 4100, 17]
    cq, ck = cu_of([1, 1, 2, 1, 4, 1]), cu_of(nk)
    q, k, v = rand((cq[-1], hq, d), 1, dtype, 1.5).cuda(), rand((ck[-1], hk, d), 2, dtype).cuda(), rand((ck[-1], hk, d), 3, dtype).cuda()
    for left, sinks in [(4095, 4), (4095, 0), (511, 600), (0, 3), (16000, 1)]:
        o = ops.attention(q, k, v, dev_cu(cq), dev_cu(ck), max_q=4, max_k=20000, window=(left, 0), sinks=sinks)
        inside(o, *window_want(q, k, v, cq, ck, True, left, 0, sinks), f"next tokens {left} {sinks}")


def test_a_window_without_ends_gives_the_same_bits(ops):  # noqa: F811
    say("window without ends")
    cu = dev_cu([0, 200, 201, 330])
    q, k, v = (rand((330, 4, 64), i, BF).cuda() for i in range(3))
    for causal in (False, True):
        want = ops.attention(q, k, v, cu, causal=causal)
        for window, sinks in (((None, None), 0), ((330, 330), 7), ((None, 2 ** 31), 0)):
            assert torch.equal(ops.attention(q, k, v, cu, causal=causal, window=window, sinks=sinks), want)


@pytest.mark.parametrize("nq,nk,left,right,sinks", [(200, 200, 20, 0, 3), (300, 300, 40, 30, 0), (1, 900, 100, 0, 4), (3, 500, 64, 0, 0),
                                                     (90, 400, 10, 5, 2)])
@pytest.mark.parametrize("d", [64, 128])
def test_window_ignores_what_it_does_not_see(ops, nq, nk, left, right, sinks, d):  # noqa: F811
    """Keys and values that a query does not see may hold anything."""
    say("window unseen", nq, nk, left, right, sinks, d)
    hq, hk = 4, 2
    causal = right == 0
    q, k, v = rand((nq + 2, hq, d), 1, BF), rand((nk + 6, hk, d), 2, BF), rand((nk + 6, hk, d), 3, BF)
    cq, ck = [1, nq + 1], [3, nk + 3]
    for t in (k, v):
        t[:3], t[nk + 3:] = float("nan"), float("inf")
    seen = seen_of(nq, nk, causal, left, right, sinks)
    for bad in sorted({sinks, nk // 2, nk - 1, max(0, nk - nq - left - 1)}):
        for value in (float("nan"), float("inf"), torch.finfo(BF).min):
            k2, v2 = k.clone(), v.clone()
            v2[3 + bad, :, 5] = value
            k2[3 + bad, :, 0] = value
            o = torch.full((nq + 2, hq, d), 9.0, dtype=BF, device="cuda")
            ops.attention(q.cuda(), k2.cuda(), v2.cuda(), dev_cu(cq), dev_cu(ck), causal=causal, window=(left, right), sinks=sinks, out=o)
            o = o.cpu()
            want, bound = window_want(q[1:nq + 1].cuda(), k[3:nk + 3].cuda(), v[3:nk + 3].cuda(), [0, nq], [0, nk], causal, left, right, sinks)
            blind = ~seen[:, bad]
            inside(o[1:nq + 1][blind], want[blind], bound[blind], f"unseen {bad} {value}")
            if value != value:
                assert torch.isnan(o[1:nq + 1][~blind]).all()
            assert torch.all(o[0] == 9) and torch.all(o[nq + 1] == 9)


def test_window_strides_alignment_and_scale(ops):  # noqa: F811
    """Heads anywhere in a fused row, keys at odd addresses, heads ahead of tokens,
    a negative scale."""
    say("window strides")
    n, hq, hk = 300, 4, 2
    for d in (64, 72, 128):
        for offset in (0, 1):
            qkv = rand((n, (hq + 2 * hk) * d + 3), 1, HF).cuda()[:, offset:]
            q, k, v = (qkv[:, a * d:e * d].unflatten(1, (e - a, d)) for a, e in ((0, hq), (hq, hq + hk), (hq + hk, hq + 2 * hk)))
            for scale in (None, -0.1):
                o = ops.attention(q, k, v, dev_cu([0, n]), causal=False, window=(30, 50), sinks=2, scale=scale)
                inside(o, *window_want(q, k, v, [0, n], [0, n], False, 30, 50, 2, scale), f"strides {d} {offset}")
        q, k, v = (rand((h, n, d), i, HF).cuda().transpose(0, 1) for i, h in enumerate((hq, hk, hk)))
        out = torch.empty(hq, n, d, dtype=HF, device="cuda").transpose(0, 1)
        o = ops.attention(q, k, v, dev_cu([0, n]), window=(30, 0), sinks=2, out=out)
        assert o is out
        inside(o, *window_want(q, k, v, [0, n], [0, n], True, 30, 0, 2), "heads ahead of tokens")


def test_window_offsets_past_32_bits(ops):  # noqa: F811
    """Keys past 2^31 elements."""
    say("window far keys")
    nk, hk, d = 2 ** 31 // 1024 + 5000, 4, 256
    k = torch.zeros(nk, hk, d, dtype=BF, device="cuda")
    v = torch.zeros(nk, hk, d, dtype=BF, device="cuda")
    tail = 3000
    k[-tail:], v[-tail:] = rand((tail, hk, d), 1, BF).cuda(), rand((tail, hk, d), 2, BF).cuda()
    k[:2], v[:2] = rand((2, hk, d), 3, BF).cuda(), rand((2, hk, d), 4, BF).cuda()
    for nq in (1, 200):
        q = rand((nq, hk, d), 5, BF).cuda()
        o = ops.attention(q, k, v, dev_cu([0, nq]), dev_cu([0, nk]), max_q=nq, max_k=nk, window=(2000, 0), sinks=2)
        # the same places relative to each other: the last 2900 keys, after the two first ones
        near_k, near_v = torch.cat([k[:2], k[-2900:]]), torch.cat([v[:2], v[-2900:]])
        inside(o, *window_want(q, near_k, near_v, [0, nq], [0, 2902], True, 2000, 0, 2), f"far keys {nq}")


def test_window_streams_and_graphs(ops):  # noqa: F811
    say("window graphs")
    cu, cq, ck = dev_cu([0, 70, 71, 1500]), dev_cu([0, 1, 3]), dev_cu([0, 4000, 9000])
    q, k, v = (rand((1500, 4, 64), i, BF).cuda() for i in range(3))
    q2, k2, v2 = (rand((n, h, 64), i, BF).cuda() for i, (n, h) in enumerate([(3, 8), (9000, 2), (9000, 2)]))
    fns = [lambda: ops.attention(q, k, v, cu, causal=False, window=(64, 64)), lambda: ops.attention(q, k, v, cu, window=(200, 0), sinks=3),
           lambda: ops.attention(q2, k2, v2, cq, ck, max_q=2, max_k=5000, window=(3000, 0), sinks=4)]
    want = [f() for f in fns]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        assert all(torch.equal(f(), w) for f, w in zip(fns, want))
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        out = [f() for f in fns]
    for _ in range(4):
        for t in out:
            t.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        assert all(torch.equal(f(), b) for f, b in zip(fns, want))


def test_window_refusals_and_the_struct_before_it(ops):  # noqa: F811
    import ctypes

    from browservec_amd import _lib as L

    say("window refusals")
    q, cu = rand((8, 2, 64), 1, BF).cuda(), dev_cu([0, 8])
    for kw in (dict(window=(-1, 0)), dict(window=(0, -2)), dict(window=(0, 0), sinks=-1), dict(window=5), dict(window=(1, 2, 3))):
        with pytest.raises(L.BVError) as e:
            ops.attention(q, q, q, cu, **kw)
        assert e.value.code == L.BV_E_INVALID and str(e.value)
    lib, o = L.load(), torch.zeros_like(q)
    a = L.AttentionArgs(168, 2, 2, 2, 64, 1, 1)
    a.tokens_q = a.tokens_k = 8
    a.q = a.k = a.v = q.data_ptr()
    a.o, a.cu_q, a.cu_k = o.data_ptr(), cu.data_ptr(), cu.data_ptr()
    a.window = 1  # past the end of the struct as it was: not read
    torch.cuda.synchronize()
    assert lib.bv_embed_attention(ops.handle, ctypes.addressof(a)) == L.BV_OK
    ops.sync()
    assert torch.equal(o, ops.attention(q, q, q, cu))
    for size in (0, 160, 172, 176, 192):
        a.size = size
        assert lib.bv_embed_attention(ops.handle, ctypes.addressof(a)) == L.BV_E_INVALID


@pytest.mark.parametrize("hq,hk,d,dtype", [(2, 2, 64, BF), (6, 2, 64, HF), (8, 2, 96, BF), (7, 1, 128, HF), (3, 3, 128, BF), (4, 1, 32, BF),
                                           (2, 2, 72, HF)])
def test_short_windows(ops, hq, hk, d, dtype):  # noqa: F811
    """Windows about the lengths at which a wave takes one tile of keys more or another
    way: 160 and 288 keys of 32 rows; first keys up to 32 and one more."""
    say("short windows", hq, hk, d, dtype)
    cu = cu_of([700, 33, 128, 129, 1, 260])
    q, k, v = rand((cu[-1], hq, d), 1, dtype, 1.5).cuda(), rand((cu[-1], hk, d), 2, dtype).cuda(), rand((cu[-1], hk, d), 3, dtype).cuda()
    for causal, left, right, sinks in [(False, 64, 64, 0), (False, 64, 65, 1), (False, 140, 0, 32), (False, 0, 150, 33), (True, 128, 0, 4),
                                       (True, 129, 5, 32), (False, 128, 128, 0), (False, 128, 129, 4), (True, 256, 0, 32), (True, 257, 0, 1),
                                       (False, 270, 10, 31), (False, 300, 1, 0), (False, 5, 0, 20)]:
        o = ops.attention(q, k, v, dev_cu(cu), causal=causal, window=(left, right), sinks=sinks)
        inside(o, *window_want(q, k, v, cu, cu, causal, left, right, sinks), f"short window {causal} {left} {right} {sinks}")


@pytest.mark.parametrize("nq,nk", [(1500, 1500), (900, 2000), (2000, 700)])
@pytest.mark.parametrize("left,right,sinks", [(64, 64, 0), (100, 0, 4), (600, 0, 3)])
def test_window_of_a_long_prompt_ignores_what_it_does_not_see(ops, nq, nk, left, right, sinks):  # noqa: F811
    """One sequence and one head, whose keys would be split were the window longer; a
    value that is not finite, which some rows see."""
    say("window long unseen", nq, nk, left, right, sinks)
    q, k, v = rand((nq, 1, 64), 1, BF).cuda(), rand((nk, 1, 64), 2, BF).cuda(), rand((nk, 1, 64), 3, BF).cuda()
    seen = seen_of(nq, nk, right == 0, left, right, sinks)
    want, bound = window_want(q, k, v, [0, nq], [0, nk], right == 0, left, right, sinks)
    for bad in (0, nk // 2, nk - 1):
        v2 = v.clone()
        v2[bad, 0, 7] = float("nan")
        o = ops.attention(q, k, v2, dev_cu([0, nq]), dev_cu([0, nk]), max_q=nq, max_k=nk, causal=right == 0, window=(left, right),
                          sinks=sinks).cpu()
        blind = ~seen[:, bad]
        inside(o[blind], want[blind], bound[blind], f"unseen {bad}")
        assert torch.isnan(o[~blind][:, 0, 7]).all() and torch.isfinite(o[~blind][:, 0, :7]).all()


def test_window_of_many_texts(ops):  # noqa: F811
    """More texts than a wave has lanes, of all lengths, and none at all between."""
    say("window many texts")
    g = torch.Generator().manual_seed(5)
    lens = torch.randint(0, 300, (333,), generator=g).tolist()
    cu = cu_of(lens)
    for hq, hk, d in ((2, 1, 64), (3, 3, 32)):
        q, k, v = rand((cu[-1], hq, d), 1, BF, 1.5).cuda(), rand((cu[-1], hk, d), 2, BF).cuda(), rand((cu[-1], hk, d), 3, BF).cuda()
        for causal, left, right, sinks in ((False, 16, 30, 0), (True, 50, 0, 2)):
            o = ops.attention(q, k, v, dev_cu(cu), causal=causal, window=(left, right), sinks=sinks, max_q=300)
            inside(o, *window_want(q, k, v, cu, cu, causal, left, right, sinks), "many texts")


def test_short_window_of_far_keys_and_odd_rows(ops):  # noqa: F811
    """Keys past 2^31 elements; queries and results at odd addresses; no keys at all."""
    say("short window, far keys")
    nk, hk, d, tail = 2 ** 31 // 1024 + 700, 4, 256, 300
    big = torch.zeros(nk, hk, d, dtype=BF, device="cuda")
    big[-tail:] = rand((tail, hk, d), 1, BF).cuda()
    k, v = big[:, :, :128], big[:, :, 128:]
    q = rand((200, hk, 129), 5, BF).cuda()[:, :, 1:]
    out = torch.full((200, hk, 131), 7.0, dtype=BF, device="cuda")
    o = ops.attention(q, k, v, dev_cu([0, 200]), dev_cu([0, nk]), max_q=200, window=(40, 0), out=out[:, :, 1:129])
    near = [t[-250:].contiguous() for t in (k, v)]
    inside(o, *window_want(q, *near, [0, 200], [0, 250], True, 40, 0, 0), "far keys")
    assert torch.all(out[:, :, 0] == 7) and torch.all(out[:, :, 129:] == 7)
    o = ops.attention(q[:, :, :64], k[:0, :, :64], v[:0, :, :64], dev_cu([0, 200]), dev_cu([0, 0]), causal=False, window=(40, 40), sinks=3)
    assert torch.all(o == 0)


@pytest.mark.parametrize("hq,hk,d", [(4, 1, 128), (2, 2, 128), (8, 2, 64), (4, 1, 96), (6, 2, 32), (2, 1, 104)])
def test_short_windows_and_their_first_keys(ops, hq, hk, d):  # noqa: F811
    """First keys of every number beside windows of few and many keys, queries before
    the first key, whose window is empty, among them."""
    say("first keys", hq, hk, d)
    nq, nk = [333, 200, 1, 70, 150], [333, 90, 1, 260, 1]
    cq, ck = cu_of(nq), cu_of(nk)
    q, k, v = rand((cq[-1], hq, d), 1, BF, 1.5).cuda(), rand((ck[-1], hk, d), 2, BF).cuda(), rand((ck[-1], hk, d), 3, BF).cuda()
    for left, right, sinks in [(0, 0, 1), (5, 3, 4), (150, 0, 4), (120, 0, 5), (200, 0, 8), (250, 0, 9), (100, 100, 16), (60, 70, 17),
                               (31, 31, 31), (200, 50, 32), (250, 0, 3), (0, 0, 32)]:
        for causal in (False, True):
            o = ops.attention(q, k, v, dev_cu(cq), dev_cu(ck), causal=causal, window=(left, right), sinks=sinks)
            inside(o, *window_want(q, k, v, cq, ck, causal, left, right, sinks), f"first keys {left} {right} {sinks} {causal}")


def test_a_windows_values_that_are_not_finite_reach_whoever_sees_them(ops):  # noqa: F811
    """An infinite and a NaN value within some rows' windows: those rows are as the
    formula has them, the others as with finite values."""
    n, d = 1500, 64
    for hq, hk, left, sinks in ((4, 2, 40, 0), (4, 2, 700, 3), (2, 2, 300, 0)):
        say("not finite", hq, hk, left, sinks)
        q, k, v = rand((n, hq, d), 1, BF).cuda(), rand((n, hk, d), 2, BF).cuda(), rand((n, hk, d), 3, BF).cuda()
        bad = v.clone()
        bad[500, 0, 3], bad[901, hk - 1, 60] = float("inf"), float("nan")
        run = lambda v: ops.attention(q, k, v, dev_cu([0, n]), window=(left, 0), sinks=sinks).cpu()  # noqa: E731
        good, got = run(v), run(bad)
        want, bound = window_want(q, k, v, [0, n], [0, n], True, left, 0, sinks)
        sees = seen_of(n, n, True, left, 0, sinks)
        hit = torch.zeros(n, hq, d, dtype=torch.bool)
        group = hq // hk
        for key, head, at, value in ((500, 0, 3, float("inf")), (901, hk - 1, 60, float("nan"))):
            rows = sees[:, key]
            for h in range(head * group, (head + 1) * group):
                hit[rows, h, at] = True
                x = got[rows, h, at].float()
                assert (x == value).all() if value == value else x.isnan().all()
        assert torch.isfinite(got[~hit].float()).all() and torch.isfinite(good.float()).all()
        assert ((got.double() - want).abs() <= bound)[~hit].all()
