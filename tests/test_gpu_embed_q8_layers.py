"""Layers of the operators in 8 bits and of windows, run together as an encoder
runs them: the example's, and a prompt against its tokens one by one."""

import os
import sys

import numpy as np
import pytest
import torch

from tests.helpers import need_gpu, say
from tests.test_gpu_embed import BF, F32, HF, U, cu_of, dev_cu, inside, ops, rand  # noqa: F401
from tests.test_gpu_embed_q8 import ACTS
from tests.test_gpu_embed_window import seen_of, window_want

pytestmark = pytest.mark.gpu
sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


def plain(enc, sequences, window):
    """The example's encoder of one sequence at a time in 64 bits, its weights as they
    are before they become codes."""
    out = []
    rms = lambda x, w: x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-5) * w.cpu().double()  # noqa: E731
    table = enc.table.cpu().double()
    for s in sequences:
        x = enc.embeddings.cpu().double()[s]
        cos, sin = table[:len(s), None, :, 0], table[:len(s), None, :, 1]

        def turn(t):
            a, b = t.chunk(2, -1)
            return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        seen = seen_of(len(s), len(s), False, window, window, 0)
        for layer in enc.layers:
            w = {k: v.cpu().double() for k, v in layer.items()}
            qkv = (rms(x, w["norm1"]) @ w["qkv"].t()).unflatten(1, (-1, enc.d))
            q, k, v = turn(qkv[:, :enc.heads]), turn(qkv[:, enc.heads:enc.heads + enc.key_heads]), qkv[:, enc.heads + enc.key_heads:]
            g = enc.heads // enc.key_heads
            p = torch.einsum("qhd,khd->hqk", q, k.repeat_interleave(g, 1)) * enc.d ** -0.5
            p = torch.softmax(p.masked_fill(~seen, float("-inf")), -1)
            x = x + torch.einsum("hqk,khd->qhd", p, v.repeat_interleave(g, 1)).flatten(1) @ w["out"].t()
            u = rms(x, w["norm2"]) @ w["up"].t() + w["up_bias"]
            x = x + ACTS["gelu"](u) @ w["down"].t()
        y = rms(x, enc.last).mean(0)
        out.append(y / y.norm())
    return torch.stack(out)


@pytest.mark.parametrize("q8,window", [(True, 20), (True, None), (False, 20)])
def test_encoder_and_index(q8, window):
    need_gpu()
    import embed_and_search as ex
    from browservec_amd import DeviceContext, EmbedOps, FlatIndex

    say("encoder example", q8, window)
    ctx = DeviceContext(0)
    e = EmbedOps(ctx)
    index = FlatIndex(ctx, 384, "cosine")
    enc = ex.Encoder(e, q8=q8, window=window)
    torch.cuda.synchronize()
    r = np.random.default_rng(3)
    passages = [r.integers(0, 1000, n).tolist() for n in [1, 2, 17, 64, 65, 130, 200, 33, 5]]
    with torch.cuda.stream(torch.cuda.ExternalStream(index.stream_ptr())):
        vectors = enc(passages)
        index.append_device(vectors.data_ptr(), len(passages))
        rows, scores = ex.search(index, enc(passages), 2)
        index.sync()
        vectors, rows, scores = vectors.cpu(), rows.cpu(), scores.cpu()
    want = plain(enc, passages, window)
    # 16 bits: as in the example's own test, well under 12 2^-8.  8 bits: a row's codes
    # are off by a step over sqrt(12) each on average, a step being its largest magnitude
    # over 127; of 384 to 1536 normal values that is some 3.5 times their size: 0.8%.
    # A product's two operands then make 0.8% sqrt(2) of its size; the eight products
    # of two layers, were their errors to add up in one direction, 9%.
    off = (vectors.double() - want).norm(dim=1)
    assert off.max() < 12 * 2.0 ** -8 + q8 * 8 * 2 ** 0.5 * 3.5 / 127 / 12 ** 0.5, off
    assert (vectors.double().norm(dim=1) - 1).abs().max() < 1e-6
    assert rows[:, 0].tolist() == list(range(len(passages)))  # every passage finds itself
    torch.cuda.synchronize()
    index.destroy()
    e.destroy()
    ctx.destroy()


@pytest.mark.parametrize("hq,hk,d,dtype", [(4, 4, 64, BF), (8, 2, 128, HF)])
@pytest.mark.parametrize("left,sinks", [(63, 0), (63, 4), (200, 40), (0, 1)])
def test_a_prompt_and_its_tokens_one_by_one(ops, hq, hk, d, dtype, left, sinks):  # noqa: F811
    """A prompt's attention, and each of its tokens as a new one over the keys so far."""
    say("prompt and tokens", hq, hk, d, dtype, left, sinks)
    n = 333
    q, k, v = rand((n, hq, d), 1, dtype, 1.5).cuda(), rand((n, hk, d), 2, dtype).cuda(), rand((n, hk, d), 3, dtype).cuda()
    want = window_want(q, k, v, [0, n], [0, n], True, left, None, sinks)
    inside(ops.attention(q, k, v, dev_cu([0, n]), window=(left, 0), sinks=sinks), *want, "prompt")
    out = torch.empty_like(q)
    one = dev_cu([0, 1])
    for i in range(0, n, 7):
        ops.attention(q[i:i + 1], k[:i + 1], v[:i + 1], one, dev_cu([0, i + 1]), max_q=1, max_k=i + 1, window=(left, None), sinks=sinks,
                      out=out[i:i + 1])
    inside(out[::7], want[0][::7], want[1][::7], "tokens")


@pytest.mark.parametrize("tokens", [3, 300])
def test_codes_through_a_product(ops, tokens):  # noqa: F811
    """norm_q8's codes and scales through linear_q8, its result through add_norm:
    against 64 bits, from the codes that came out."""
    say("codes through a product", tokens)
    x, r = rand((tokens, 500), 1, BF).cuda(), rand((tokens, 500), 2, F32).cuda()
    w, sw, _ = ops.norm_q8(rand((500, 500), 3, BF, 0.05).cuda(), kind=None)
    q, s, t = ops.norm_q8(x, residual=r, kind="rms")
    y = ops.linear_q8(q, s, w, sw, out_dtype=BF)
    z, total = ops.add_norm(y, t, kind="layer", out_dtype=F32)
    exact = (q.double() @ w.double().t().contiguous()) * s.double()[:, None] * sw.double()  # whole numbers below 2^53
    # three roundings in 32 bits, together below 4 2^-24; one to bf16, of what they made:
    # |y - e| <= 4 2^-24 |e| + 2^-8 (1 + 4 2^-24) |e|
    inside(y, exact.cpu(), (exact.abs() * (4 * 2.0 ** -24 + U[BF] * (1 + 4 * 2.0 ** -24))).cpu() + 1e-37, "product")
    inside(total, (y.double() + t.double()).cpu(), (2.0 ** -24 * 1.01 * (y.double() + t.double()).abs()).cpu(), "sum")
    c = y.double() + t.double()
    want = ((c - c.mean(-1, keepdim=True)) / torch.sqrt(c.var(-1, unbiased=False, keepdim=True) + 1e-5)).cpu()
    # sums of 500 values by threads and halves: within 64 2^-24 of the values' size,
    # for the mean and for the squares, and the sum's own rounding
    inside(z, want, 200 * 2.0 ** -24 * (1 + want.abs()) * (1 + c.abs().amax(-1, keepdim=True).cpu()), "norm")
