"""Text to answers on one GPU: packed token rows go through an encoder made of
the embedding operators, the vectors it pools go into an index without leaving
the device, and questions are embedded and searched the same way, all on the
index's stream.

    python examples/embed_and_search.py [--q8] [--window TOKENS]

--q8: the layers' products in 8 bits; --window: a token sees so many on both sides.
The weights are random and the tokens are numbers: a real program loads a
model's weights and its tokenizer's output in their place.
"""

from __future__ import annotations

import argparse
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from browservec_amd import DeviceContext, EmbedOps, FlatIndex, rotary_table  # noqa: E402


class Encoder:
    """A bidirectional encoder: embeddings, then layers of RMS norm, attention
    with rotary positions and grouped heads, and a wide layer, on a residual of
    32-bit floats; the last norm, the mean and unit length make the vector.  q8: the
    products of a layer take codes of 8 bits, of activations with a scale a token
    and of weights with a scale a row.  window: how many tokens a token sees on each
    side."""

    def __init__(self, ops: EmbedOps, vocab=1000, dim=384, layers=2, heads=6, key_heads=2, wide=1536, max_tokens=512,
                 dtype=torch.bfloat16, seed=0, q8=False, window=None):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.ops, self.heads, self.key_heads, self.d, self.dtype = ops, heads, key_heads, dim // heads, dtype
        self.q8, self.window = q8, None if window is None else (window, window)

        def w(n, k):
            return (torch.randn(n, k, generator=g, device="cuda") * k ** -0.5).to(dtype)

        self.embeddings = torch.randn(vocab, dim, generator=g, device="cuda")
        self.table = torch.from_numpy(rotary_table(max_tokens, self.d)).cuda()
        self.layers = [dict(norm1=torch.ones(dim, device="cuda"), qkv=w((heads + 2 * key_heads) * self.d, dim), out=w(dim, dim),
                            norm2=torch.ones(dim, device="cuda"), up=w(wide, dim), up_bias=torch.zeros(wide, device="cuda", dtype=dtype),
                            down=w(dim, wide)) for _ in range(layers)]
        self.last = torch.ones(dim, device="cuda")
        # the weights of the products, in the form that they take
        self.products = [{name: ops.norm_q8(layer[name], kind=None)[:2] if q8 else layer[name] for name in ("qkv", "out", "up", "down")}
                         for layer in self.layers]

    def norm(self, x, weight):
        """The RMS norm, or x as it is (weight None), as a product takes it."""
        kind = None if weight is None else "rms"
        if self.q8:
            return self.ops.norm_q8(x, weight=weight, kind=kind)[:2]
        return x if weight is None else self.ops.norm(x, weight=weight, kind=kind, out_dtype=self.dtype)

    def linear(self, x, weight, **kw):
        return self.ops.linear_q8(*x, *weight, **kw) if self.q8 else self.ops.linear(x, weight, **kw)

    def __call__(self, sequences: list[list[int]]) -> torch.Tensor:
        """Unit vectors [len(sequences), dim] of lists of token ids."""
        ops, lens = self.ops, [len(s) for s in sequences]
        cu = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")
        tokens = torch.tensor([t for s in sequences for t in s], device="cuda")
        positions = torch.tensor([i for n in lens for i in range(n)], dtype=torch.int32, device="cuda")
        x = self.embeddings[tokens]  # the residual, 32 bits
        hq, hk, d = self.heads, self.key_heads, self.d
        for layer, w in zip(self.layers, self.products):
            qkv = self.linear(self.norm(x, layer["norm1"]), w["qkv"], out_dtype=self.dtype)
            q, k, v = (t.unflatten(1, (-1, d)) for t in qkv.split([hq * d, hk * d, hk * d], 1))
            ops.rotary(q, k, self.table, positions=positions, out_q=q, out_k=k)
            o = ops.attention(q, k, v, cu, max_q=max(lens), causal=False, window=self.window)
            self.linear(self.norm(o.flatten(1), None), w["out"], residual=x, out=x, out_dtype=torch.float32)
            h = self.linear(self.norm(x, layer["norm2"]), w["up"], bias=layer["up_bias"], activation="gelu", out_dtype=self.dtype)
            self.linear(self.norm(h, None), w["down"], residual=x, out=x, out_dtype=torch.float32)
        return ops.pool(x, cu, kind="rms", weight=self.last)


def search(index, queries: torch.Tensor, k: int):
    """Rows and scores of the k nearest, on the current stream (the index's)."""
    n = queries.shape[0]
    rows = torch.empty(n, k, dtype=torch.int32, device="cuda")
    scores = torch.empty(n, k, dtype=torch.float32, device="cuda")
    found = torch.empty(n, dtype=torch.int32, device="cuda")
    index.search_device(queries.data_ptr(), n, 0, k, rows.data_ptr(), scores.data_ptr(), found.data_ptr())
    return rows, scores


def main() -> None:
    parser = argparse.ArgumentParser()
    parser.add_argument("--q8", action="store_true", help="the layers' products in 8 bits")
    parser.add_argument("--window", type=int, help="how many tokens a token sees on each side")
    args = parser.parse_args()
    ctx = DeviceContext(0)
    ops = EmbedOps(ctx)
    index = FlatIndex(ctx, 384, "cosine")
    encoder = Encoder(ops, q8=args.q8, window=args.window)
    torch.cuda.synchronize()  # the weights, made on torch's own stream
    r = np.random.default_rng(1)
    passages = [r.integers(0, 1000, r.integers(5, 200)).tolist() for _ in range(2000)]
    # one stream for everything: encoder, append and search follow one another
    with torch.cuda.stream(torch.cuda.ExternalStream(index.stream_ptr())):
        for i in range(0, len(passages), 500):
            vectors = encoder(passages[i:i + 500])
            index.append_device(vectors.data_ptr(), vectors.shape[0])
        questions = [passages[7][3:40], passages[1234], passages[42][:-2]]  # parts of passages
        rows, scores = search(index, encoder(questions), 3)
        index.sync()
        for q, (row, score) in enumerate(zip(rows.tolist(), scores.tolist())):
            print("question", q, "->", ", ".join(f"passage {a} ({b:.3f})" for a, b in zip(row, score)))
    torch.cuda.synchronize()
    index.destroy()
    ops.destroy()
    ctx.destroy()


if __name__ == "__main__":
    main()
