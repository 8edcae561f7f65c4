"""The example's encoder against the same layers in 64 bits, and its vectors in
an index, on the index's stream."""

import os
import sys

import numpy as np
import pytest
import torch

from tests.helpers import need_gpu, say

pytestmark = pytest.mark.gpu
sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


def plain(enc, sequences):
    """The encoder of one sequence at a time, 64 bits throughout."""
    out = []
    rms = lambda x, w: x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-5) * w.cpu().double()  # noqa: E731
    table = enc.table.cpu().double()
    for s in sequences:
        x = enc.embeddings.cpu().double()[s]
        cos, sin = table[:len(s), None, :, 0], table[:len(s), None, :, 1]

        def turn(t):
            a, b = t.chunk(2, -1)
            return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        for layer in enc.layers:
            w = {k: v.cpu().double() for k, v in layer.items()}
            qkv = (rms(x, w["norm1"]) @ w["qkv"].t()).unflatten(1, (-1, enc.d))
            q, k, v = turn(qkv[:, :enc.heads]), turn(qkv[:, enc.heads:enc.heads + enc.key_heads]), qkv[:, enc.heads + enc.key_heads:]
            g = enc.heads // enc.key_heads
            p = torch.softmax(torch.einsum("qhd,khd->hqk", q, k.repeat_interleave(g, 1)) * enc.d ** -0.5, -1)
            x = x + torch.einsum("hqk,khd->qhd", p, v.repeat_interleave(g, 1)).flatten(1) @ w["out"].t()
            u = rms(x, w["norm2"]) @ w["up"].t() + w["up_bias"]
            x = x + (u * torch.special.ndtr(u)) @ w["down"].t()
        y = rms(x, enc.last).mean(0)
        out.append(y / y.norm())
    return torch.stack(out)


def test_encoder_and_index():
    need_gpu()
    import embed_and_search as ex
    from browservec_amd import DeviceContext, EmbedOps, FlatIndex

    say("encoder example")
    ctx = DeviceContext(0)
    ops = EmbedOps(ctx)
    index = FlatIndex(ctx, 384, "cosine")
    enc = ex.Encoder(ops)
    torch.cuda.synchronize()
    r = np.random.default_rng(3)
    passages = [r.integers(0, 1000, n).tolist() for n in [1, 2, 17, 64, 65, 130, 200, 33, 5]]
    with torch.cuda.stream(torch.cuda.ExternalStream(index.stream_ptr())):
        vectors = enc(passages)
        index.append_device(vectors.data_ptr(), len(passages))
        rows, scores = ex.search(index, enc(passages), 2)
        index.sync()
        vectors, rows, scores = vectors.cpu(), rows.cpu(), scores.cpu()
    want = plain(enc, passages)
    # Each layer rounds activations of size about 1 to bfloat16 (2^-9 on average
    # relative) some six times; independent roundings over 2 layers, averaged
    # over a sequence's rows: a unit vector is off by well under
    # 2 * 6 * 2^-8 in its 2-norm.
    off = (vectors.double() - want).norm(dim=1)
    assert off.max() < 12 * 2.0 ** -8, off
    assert (vectors.double().norm(dim=1) - 1).abs().max() < 1e-6
    assert rows[:, 0].tolist() == list(range(len(passages)))  # every passage finds itself
    assert (scores[:, 0] - 1).abs().max() < 1e-5
    torch.cuda.synchronize()
    index.destroy()
    ops.destroy()
    ctx.destroy()
