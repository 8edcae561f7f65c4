"""Performance cases of an embedding model's operators: what a program has them
do that turns text into the vectors an index holds, on the GPU that searches
them.

A case is a dict of plain values; ``op`` says which operator it calls:

  linear     y = act(x W^T + b) + r, the products of an encoder layer
  rotary     rotary positions of queries and keys, from a table of cosines and
             sines by position
  attention  softmax attention over packed sequences of different lengths with
             grouped heads; whole prompts, or a few new tokens over kept keys
  norm       layer or RMS norm of every token's row
  pool       each sequence's rows (normed or as they are) to one unit vector

``own`` false: the plain forms, elementary torch operations in 32 bits; true:
the calls of browservec_amd.EmbedOps.
"""

import functools
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}


def listed():
    return [
        # one question of a few words through a small model's wide layer: latency
        dict(name="linear_9x384_1536", op="linear", m=9, k=384, n=1536, dtype="bf16", out="bf16", act="gelu", bias=True,
             residual=False),
        # a handful of passages through an attention's output product, back onto
        # the residual; a token count that is no multiple of a tile
        dict(name="linear_2037x768_768", op="linear", m=2037, k=768, n=768, dtype="f16", out="f16", act="none", bias=True,
             residual=True),
        # a corpus being embedded: the wide layer of a 1024-wide model
        dict(name="linear_32768x1024_4096", op="linear", m=32768, k=1024, n=4096, dtype="bf16", out="bf16", act="gelu",
             bias=True, residual=False),
        # one question: queries and keys of a small model, half of each head turned
        dict(name="rotary_17_12x32", op="rotary", tokens=17, hq=12, hk=12, d=32, rot=16, rows=512, layout="interleaved",
             dtype="bf16"),
        # a corpus: the whole head turned, positions of long documents
        dict(name="rotary_65536_16x64", op="rotary", tokens=65536, hq=16, hk=4, d=64, rot=64, rows=32768, layout="half",
             dtype="bf16"),
        # one question through a small bidirectional model: latency
        dict(name="attention_1x17_12x32", op="attention", batch=1, lo=17, hi=17, new=0, hq=12, hk=12, d=32, causal=False,
             dtype="bf16"),
        # passages of very different lengths in one call
        dict(name="attention_96x512_12x64", op="attention", batch=96, lo=1, hi=512, new=0, hq=12, hk=4, d=64, causal=True,
             dtype="bf16"),
        # two whole documents, the longest a model of this kind takes
        dict(name="attention_2x16001_8x128", op="attention", batch=2, lo=9001, hi=16001, new=0, hq=8, hk=2, d=128,
             causal=True, dtype="f16"),
        # the next token of a few sequences whose keys are kept
        dict(name="attention_8x32768_step", op="attention", batch=8, lo=3000, hi=32768, new=1, hq=16, hk=4, d=64,
             causal=True, dtype="bf16"),
        # every token of a batch of passages
        dict(name="norm_30011x768", op="norm", tokens=30011, dim=768, kind="layer", dtype="bf16", out="bf16"),
        # one question's vector
        dict(name="pool_1x17_384", op="pool", batch=1, lo=17, hi=17, dim=384, mode="mean", kind="none", dtype="bf16"),
        # a corpus' vectors: the last norm, the mean, unit length
        dict(name="pool_3000x256_1024", op="pool", batch=3000, lo=1, hi=256, dim=1024, mode="mean", kind="rms",
             dtype="bf16"),
    ]


def _logint(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng):
    w = rng.choice([384, 768, 1000, 1024, 1536, 2048, 4096, rng.randint(64, 1024), rng.randint(64, 4096)])
    return w + 1 if w == 3072 else w


def draw(rng):
    op = rng.choice(["linear", "linear", "linear", "rotary", "attention", "attention", "attention", "norm", "pool", "pool"])
    half = rng.choice(["bf16", "f16"])
    if op == "linear":
        k, n = _width(rng), _width(rng)
        m = _logint(rng, 1, min(32768, 32768 * 1024 * 4096 // (k * n)))
        return dict(op=op, m=m, k=k, n=n, dtype=half, out=rng.choice([half, half, "f32"]),
                    act=rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"]), bias=rng.random() < 0.7,
                    residual=rng.random() < 0.4)
    if op == "rotary":
        hk = rng.choice([1, 2, 4, 8])
        d = rng.choice([32, 64, 80, 96, 128])
        hq = hk * rng.choice([1, 2, 3, 4])
        return dict(op=op, tokens=_logint(rng, 1, 65536 * 20 * 64 // ((hq + hk) * d)), hq=hq, hk=hk, d=d,
                    rot=rng.choice([d, d, d // 2]), rows=_logint(rng, 64, 32768), layout=rng.choice(["half", "interleaved"]),
                    dtype=rng.choice([half, half, "f32"]))
    if op == "attention":
        hk = rng.choice([1, 2, 4])
        hq = hk * rng.choice([1, 2, 3, 4])
        d = rng.choice([32, 64, 64, 80, 96, 128])
        if rng.random() < 0.35:
            batch = _logint(rng, 1, 64)
            hi = _logint(rng, 16, min(32768, 8 * 32768 * 4 * 64 // (batch * hk * d)))
            return dict(op=op, batch=batch, lo=rng.randint(1, hi), hi=hi, new=rng.choice([1, 1, 2, 4]), hq=hq, hk=hk, d=d,
                        causal=True, dtype=half)
        hi = _logint(rng, 1, 8192)
        batch = _logint(rng, 1, max(1, min(512, 8192 * 8192 * 2 // (hi * hi * (1 + hq // 9)))))
        return dict(op=op, batch=batch, lo=rng.randint(1, hi), hi=hi, new=0, hq=hq, hk=hk, d=d,
                    causal=rng.random() < 0.6, dtype=half)
    dim = _width(rng)
    if op == "norm":
        return dict(op=op, tokens=_logint(rng, 1, min(131072, 200_000_000 // dim)), dim=dim,
                    kind=rng.choice(["layer", "rms"]), dtype=rng.choice([half, half, "f32"]),
                    out=rng.choice([half, half, "f32"]))
    hi = _logint(rng, 1, 4096)
    return dict(op=op, batch=_logint(rng, 1, max(1, min(4096, 200_000_000 // (hi * dim)))), lo=rng.randint(1, hi), hi=hi,
                dim=dim, mode=rng.choice(["mean", "mean", "first", "last"]), kind=rng.choice(["none", "layer", "rms"]),
                dtype=rng.choice([half, half, "f32"]))


def _lengths(case):
    """The sequences' lengths, `lo` to `hi`, one of them `hi`: the case's, whatever the seed."""
    r = random.Random("%(batch)s %(lo)s %(hi)s" % case)
    lens = [r.randint(case["lo"], case["hi"]) for _ in range(case["batch"])]
    lens[r.randrange(len(lens))] = case["hi"]
    return lens


def _offsets(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu


# ------------------------------------------------------------------ inputs --
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def rand(*shape, scale=1.0, shift=0.0, dtype=dtype):
        return torch.randn(*shape, generator=g, device="cuda").mul_(scale).add_(shift).to(dtype)

    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        return dict(case=case, x=rand(m, k), w=rand(n, k, scale=k ** -0.5), b=rand(n, scale=0.1) if case["bias"] else None,
                    r=rand(m, n, dtype=DTYPES[case["out"]]) if case["residual"] else None)
    if case["op"] == "rotary":
        t, hq, hk, d, rot = (case[x] for x in ("tokens", "hq", "hk", "d", "rot"))
        # queries and keys as a layer's fused product leaves them: views of one
        # row per token; sequences of any start, so positions of any order
        qkv = rand(t, (hq + 2 * hk) * d)
        angle = torch.arange(case["rows"], device="cuda", dtype=torch.float64)[:, None] * \
            torch.pow(10000.0, -torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
        start = torch.randint(0, case["rows"], (1,), generator=g, device="cuda", dtype=torch.int32)
        return dict(case=case, q=qkv[:, :hq * d].view(t, hq, d), k=qkv[:, hq * d:(hq + hk) * d].view(t, hk, d),
                    table=torch.stack([angle.cos(), angle.sin()], dim=-1).float().contiguous(),
                    positions=(torch.arange(t, device="cuda", dtype=torch.int32) + start).remainder(case["rows"]).int())
    if case["op"] == "attention":
        lens = _lengths(case)
        new = [case["new"]] * len(lens) if case["new"] else lens
        hq, hk, d = case["hq"], case["hk"], case["d"]
        cu_q, cu_k = _offsets(new), _offsets(lens)
        as_cu = lambda c: torch.tensor(c, dtype=torch.int32, device="cuda")  # noqa: E731
        kv = rand(cu_k[-1], 2 * hk, d)
        return dict(case=case, q=rand(cu_q[-1], hq, d, scale=1.5), k=kv[:, :hk], v=kv[:, hk:], cu_q=as_cu(cu_q),
                    cu_k=as_cu(cu_k), max_q=max(new), max_k=max(lens))
    dim, weighted = case["dim"], case["op"] == "norm" or case["kind"] != "none"
    w = rand(dim, scale=0.1, shift=1.0) if weighted else None
    b = rand(dim, scale=0.1) if weighted and case["kind"] == "layer" else None
    if case["op"] == "norm":
        return dict(case=case, x=rand(case["tokens"], dim, scale=2.0, shift=0.3), w=w, b=b)
    cu = _offsets(_lengths(case))
    return dict(case=case, x=rand(cu[-1], dim, scale=2.0, shift=0.3), w=w, b=b,
                cu=torch.tensor(cu, dtype=torch.int32, device="cuda"))


# --------------------------------------------------------------------- run --
EPS = 1e-5


@functools.lru_cache(maxsize=1)
def _ops():
    from browservec_amd import DeviceContext, EmbedOps

    return EmbedOps(DeviceContext(0))


def run(state):
    case = state["case"]
    return (_own if own else _plain)[case["op"]](state, case)


def _own_linear(s, c):
    return _ops().linear(s["x"], s["w"], bias=s["b"], residual=s["r"], activation=c["act"], out_dtype=DTYPES[c["out"]])


def _own_rotary(s, c):
    return _ops().rotary(s["q"], s["k"], s["table"], positions=s["positions"], interleaved=c["layout"] == "interleaved")


def _own_attention(s, c):
    return _ops().attention(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], max_q=s["max_q"], max_k=s["max_k"],
                            causal=c["causal"])


def _own_norm(s, c):
    return _ops().norm(s["x"], weight=s["w"], bias=s["b"], kind=c["kind"], eps=EPS, out_dtype=DTYPES[c["out"]])


def _own_pool(s, c):
    return _ops().pool(s["x"], s["cu"], mode=c["mode"], kind=c["kind"], weight=s["w"], bias=s["b"], eps=EPS, unit=True)


_own = dict(linear=_own_linear, rotary=_own_rotary, attention=_own_attention, norm=_own_norm, pool=_own_pool)


def _act(y, kind):
    if kind == "relu":
        return torch.clamp(y, min=0)
    if kind == "gelu":
        return 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    if kind == "gelu_tanh":
        return 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
    if kind == "silu":
        return y / (1 + torch.exp(-y))
    return y


def _plain_linear(s, c):
    y = torch.matmul(s["x"].float(), s["w"].float().t())
    if s["b"] is not None:
        y = y + s["b"].float()
    y = _act(y, c["act"])
    if s["r"] is not None:
        y = y + s["r"].float()
    return y.to(DTYPES[c["out"]])


def _plain_turn(x, cos, sin, layout, rot):
    x32 = x.float()
    if layout == "half":
        a, b = x32[..., :rot // 2], x32[..., rot // 2:rot]
    else:
        a, b = x32[..., 0:rot:2], x32[..., 1:rot:2]
    u, v = a * cos - b * sin, b * cos + a * sin
    turned = torch.cat([u, v], -1) if layout == "half" else torch.stack([u, v], -1).flatten(-2)
    return torch.cat([turned, x32[..., rot:]], -1).to(x.dtype)


def _plain_rotary(s, c):
    at = s["table"][s["positions"].long()].unsqueeze(1)
    cos, sin = at[..., 0], at[..., 1]
    return _plain_turn(s["q"], cos, sin, c["layout"], c["rot"]), _plain_turn(s["k"], cos, sin, c["layout"], c["rot"])


def _plain_attention(s, c):
    q, k, v, cu_q, cu_k = s["q"], s["k"], s["v"], s["cu_q"].long(), s["cu_k"].long()
    hq, hk, d, lq, lk = c["hq"], c["hk"], c["d"], s["max_q"], s["max_k"]
    batch, group = cu_q.numel() - 1, c["hq"] // c["hk"]
    i, j = torch.arange(lq, device=q.device), torch.arange(lk, device=q.device)
    # sequences side by side, the shorter ones filled up
    at_q = (cu_q[:-1, None] + i).clamp(max=q.shape[0] - 1)
    at_k = (cu_k[:-1, None] + j).clamp(max=k.shape[0] - 1)
    nq, nk = cu_q[1:] - cu_q[:-1], cu_k[1:] - cu_k[:-1]
    qs = q.float()[at_q].view(batch, lq, hk, group, d).permute(0, 2, 3, 1, 4).reshape(batch * hk, group * lq, d)
    ks = k.float()[at_k].permute(0, 2, 3, 1).reshape(batch * hk, d, lk)
    vs = v.float()[at_k].permute(0, 2, 1, 3).reshape(batch * hk, lk, d)
    seen = (j < nk[:, None])[:, None, :].expand(batch, lq, lk)
    if c["causal"]:  # the last query sees the last key
        seen = seen & (j <= (i + (nk - nq)[:, None])[..., None])
    score = torch.matmul(qs, ks).mul_(d ** -0.5).view(batch, hk * group, lq, lk)
    score.masked_fill_(~seen[:, None], float("-inf"))
    top = score.amax(-1, keepdim=True).clamp(min=-1e30)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(batch * hk, group * lq, lk), vs).view(batch, hq, lq, d)
    o = torch.where(total > 0, o / total, torch.zeros_like(o)).permute(0, 2, 1, 3)
    t = torch.arange(q.shape[0], device=q.device)
    of = (t[:, None] >= cu_q[1:]).sum(1)
    return o[of, t - cu_q[of]].to(q.dtype)


def _normed(x, w, b, kind):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    if kind != "none":
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    if w is not None:
        x = x * w.float()
    return x if b is None else x + b.float()


def _plain_norm(s, c):
    return _normed(s["x"].float(), s["w"], s["b"], c["kind"]).to(DTYPES[c["out"]])


def _plain_pool(s, c):
    x, cu = s["x"], s["cu"].long()
    if c["mode"] == "mean":
        y = _normed(x.float(), s["w"], s["b"], c["kind"])
        of = (torch.arange(x.shape[0], device=x.device)[:, None] >= cu[1:]).sum(1)
        total = torch.zeros(cu.numel() - 1, x.shape[1], device=x.device).index_add_(0, of, y)
        y = total / (cu[1:] - cu[:-1]).clamp(min=1)[:, None]
    else:
        y = _normed(x[cu[:-1] if c["mode"] == "first" else cu[1:] - 1].float(), s["w"], s["b"], c["kind"])
    return y / y.square().sum(-1, keepdim=True).sqrt()


_plain = dict(linear=_plain_linear, rotary=_plain_rotary, attention=_plain_attention, norm=_plain_norm, pool=_plain_pool)


# -------------------------------------------------------------------- work --
def work(case):
    b = BYTES[case["dtype"]]
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        return dict(bytes=(m * k + n * k + n * case["bias"]) * b + m * n * (1 + case["residual"]) * BYTES[case["out"]],
                    flops=2 * m * n * k)
    if case["op"] == "rotary":
        heads = case["hq"] + case["hk"]
        return dict(bytes=case["tokens"] * (2 * heads * case["d"] * b + 4) + min(case["tokens"], case["rows"]) * case["rot"] * 4,
                    flops=case["tokens"] * heads * case["rot"] * 3)
    if case["op"] == "attention":
        lens, d = _lengths(case), case["d"]
        new = [case["new"]] * len(lens) if case["new"] else lens
        # query i of n sees keys up to its own place, the last query all l
        pairs = sum(q * n - q * (q - 1) // 2 if case["causal"] and q <= n else
                    n * (n + 1) // 2 if case["causal"] else q * n for q, n in zip(new, lens))
        return dict(bytes=(2 * sum(new) * case["hq"] + 2 * sum(lens) * case["hk"]) * d * b, flops=4 * pairs * d * case["hq"])
    if case["op"] == "norm":
        n = case["tokens"] * case["dim"]
        return dict(bytes=n * (b + BYTES[case["out"]]), flops=8 * n)
    rows = sum(_lengths(case)) if case["mode"] == "mean" else case["batch"]
    return dict(bytes=rows * case["dim"] * b + case["batch"] * case["dim"] * 4, flops=6 * rows * case["dim"])


# ------------------------------------------------------------------- exact --
def exact(case, seed):
    s = prepare(case, seed)
    f = lambda x: None if x is None else x.double()  # noqa: E731
    if case["op"] == "linear":
        if case["m"] * case["n"] * case["k"] > 2 ** 38:
            return None
        y = f(s["x"]) @ f(s["w"]).t().contiguous()
        if s["b"] is not None:
            y += f(s["b"])
        y = {"none": lambda z: z, "relu": lambda z: z.clamp(min=0), "gelu": lambda z: z * torch.special.ndtr(z),
             "gelu_tanh": lambda z: z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)),
             "silu": lambda z: z * torch.sigmoid(z)}[case["act"]](y)
        return y if s["r"] is None else y + f(s["r"])
    if case["op"] == "rotary":
        rot = case["rot"]
        at = s["table"].double()[s["positions"].long()]
        turn = torch.complex(at[..., 0], at[..., 1]).unsqueeze(1)

        def turned(x):
            y = f(x).clone()
            pair = (y[..., :rot // 2], y[..., rot // 2:rot]) if case["layout"] == "half" else (y[..., 0:rot:2], y[..., 1:rot:2])
            z = torch.complex(pair[0].contiguous(), pair[1].contiguous()) * turn
            pair[0].copy_(z.real)
            pair[1].copy_(z.imag)
            return y
        return turned(s["q"]), turned(s["k"])
    if case["op"] == "attention":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        group = case["hq"] // case["hk"]
        cu_q, cu_k = s["cu_q"].tolist(), s["cu_k"].tolist()
        for a, e, ka, ke in zip(cu_q, cu_q[1:], cu_k, cu_k[1:]):
            for h in range(case["hk"]):
                k, v = f(s["k"][ka:ke, h]), f(s["v"][ka:ke, h])
                for r in range(a, e, 2048):
                    q = f(s["q"][r:min(e, r + 2048), h * group:(h + 1) * group])
                    last = torch.arange(r, r + q.shape[0], device="cuda") - e + ke - ka
                    p = q.permute(1, 0, 2).reshape(-1, q.shape[2]) @ k.t().contiguous() / math.sqrt(case["d"])
                    p = p.view(group, q.shape[0], ke - ka)
                    if case["causal"]:
                        p = p.masked_fill(torch.arange(ke - ka, device="cuda") > last[:, None], -math.inf)
                    p = torch.nan_to_num(torch.softmax(p, -1), nan=0.0)
                    out[r:r + q.shape[0], h * group:(h + 1) * group] = torch.matmul(p, v).permute(1, 0, 2)
        return out
    x = f(s["x"])
    if case["kind"] == "layer":
        x = (x - x.mean(-1, keepdim=True)) / torch.sqrt(x.var(-1, unbiased=False, keepdim=True) + EPS)
    elif case["kind"] == "rms":
        x = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + EPS)
    x = x if s["w"] is None else x * f(s["w"])
    x = x if s["b"] is None else x + f(s["b"])
    if case["op"] == "norm":
        return x
    cu = s["cu"].tolist()
    pick = {"mean": lambda a, e: x[a:e].mean(0), "first": lambda a, e: x[a], "last": lambda a, e: x[e - 1]}[case["mode"]]
    y = torch.stack([pick(a, e) for a, e in zip(cu, cu[1:])])
    return y / torch.linalg.vector_norm(y, dim=-1, keepdim=True)
