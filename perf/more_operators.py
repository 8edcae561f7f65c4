"""Performance cases of an encoder's layers in 8 bits over long documents: what a
program has them do that embeds a corpus whose texts are too long, or too many,
for 16-bit layers and attention over whole texts.

A case is a dict of plain values; ``op`` says which operator it calls:

  linear_q8  y = act(sx sw (qx qw^T) + b) + r: codes of 8 bits, a scale for each
             token and each channel
  add_norm   the residual's addition and the norm of the sum in one pass
  norm_q8    the same (or the rows as they are) to codes of 8 bits and a scale a
             row: what linear_q8 takes
  local      softmax attention of packed sequences in which a query sees a window
             of keys about its place, and a few first keys

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
        dict(name="linear_q8_9x384_1536", op="linear_q8", m=9, k=384, n=1536, out="bf16", act="gelu", bias=True,
             residual=False),
        # a handful of passages through an attention's output product, back onto
        # the residual; a token count that is no multiple of a tile
        dict(name="linear_q8_2037x768_768", op="linear_q8", m=2037, k=768, n=768, out="f16", act="none", bias=True,
             residual=True),
        # a corpus: back from the wide layer onto a residual of 32 bits
        dict(name="linear_q8_20011x4096_1024", op="linear_q8", m=20011, k=4096, n=1024, out="f32", act="none", bias=False,
             residual=True),
        # a corpus: the wide layer of a 1024-wide model
        dict(name="linear_q8_32768x1024_4096", op="linear_q8", m=32768, k=1024, n=4096, out="bf16", act="gelu", bias=True,
             residual=False),
        # one question of a small model: latency
        dict(name="add_norm_17x384", op="add_norm", tokens=17, dim=384, kind="rms", dtype="bf16", rdtype="f32", out="bf16"),
        # a batch of passages, a model that norms after its additions
        dict(name="add_norm_30011x768", op="add_norm", tokens=30011, dim=768, kind="layer", dtype="bf16", rdtype="bf16",
             out="bf16"),
        # a batch of passages ahead of a product in 8 bits, onto a residual of 32 bits
        dict(name="norm_q8_30011x1024", op="norm_q8", tokens=30011, dim=1024, kind="rms", dtype="bf16", rdtype="f32"),
        # what the wide layer gives, as it is, ahead of the product back
        dict(name="norm_q8_20011x4096", op="norm_q8", tokens=20011, dim=4096, kind="none", dtype="bf16", rdtype=None),
        # passages of very different lengths, each token sees 64 on both sides
        dict(name="local_96x512_12x64", op="local", batch=96, lo=1, hi=512, new=0, hq=12, hk=12, d=64, causal=False,
             left=64, right=64, sinks=0, dtype="bf16"),
        # whole documents of the longest length, each token sees 64 on both sides
        dict(name="local_6x8192_12x64", op="local", batch=6, lo=4001, hi=8192, new=0, hq=12, hk=12, d=64, causal=False,
             left=64, right=64, sinks=0, dtype="bf16"),
        # a book through a causal model: the last 4096 tokens and the first four
        dict(name="local_1x32768_8x128", op="local", batch=1, lo=32768, hi=32768, new=0, hq=8, hk=2, d=128, causal=True,
             left=4095, right=0, sinks=4, dtype="f16"),
        # the next token of many sequences whose keys are kept
        dict(name="local_64x32768_step", op="local", batch=64, lo=3000, hi=32768, new=1, hq=16, hk=4, d=64, causal=True,
             left=4095, right=0, sinks=4, dtype="bf16"),
    ]


def _logint(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng):
    return rng.choice([384, 768, 1000, 1024, 1536, 2048, 4096, rng.randint(64, 1024), rng.randint(64, 4096)])


def draw(rng):
    op = rng.choice(["linear_q8", "linear_q8", "linear_q8", "add_norm", "norm_q8", "norm_q8", "local", "local", "local"])
    half = rng.choice(["bf16", "f16"])
    if op == "linear_q8":
        k, n = _width(rng), _width(rng)
        m = _logint(rng, 1, min(32768, 32768 * 1024 * 4096 // (k * n)))
        return dict(op=op, m=m, k=k, n=n, out=rng.choice([half, half, "f32"]),
                    act=rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"]), bias=rng.random() < 0.7,
                    residual=rng.random() < 0.4)
    if op == "local":
        hk = rng.choice([1, 2, 4, 12])
        hq = hk * rng.choice([1, 1, 2, 4] if hk < 12 else [1])
        d = rng.choice([32, 64, 64, 80, 96, 128])
        causal = rng.random() < 0.5
        left = rng.choice([64, 128, rng.randint(0, 100), _logint(rng, 1, 4096)])
        right = 0 if causal else rng.choice([left, rng.randint(0, 256)])
        sinks = rng.choice([0, 0, 4, rng.randint(1, 80)])
        hi = _logint(rng, 1, 32768)
        if causal and rng.random() < 0.4:
            batch = _logint(rng, 1, max(1, min(64, 64 * 32768 * 4 * 64 // (hi * hk * d))))
            return dict(op=op, batch=batch, lo=rng.randint(1, hi), hi=hi, new=rng.choice([1, 1, 2, 4]), hq=hq, hk=hk, d=d,
                        causal=True, left=left, right=0, sinks=sinks, dtype=half)
        seen = min(hi, left + right + 1) + sinks
        batch = _logint(rng, 1, max(1, min(512, 32768 * 4096 * 8 // (hi * max(seen, 256) * hq), 65536 // hi)))
        return dict(op=op, batch=batch, lo=rng.randint(1, hi), hi=hi, new=0, hq=hq, hk=hk, d=d, causal=causal, left=left,
                    right=right, sinks=sinks, dtype=half)
    dim = _width(rng)
    tokens = _logint(rng, 1, min(65536, 80_000_000 // dim))
    dtype = rng.choice([half, half, "f32"])
    rdtype = rng.choice([dtype, "f32"])
    if op == "add_norm":
        return dict(op=op, tokens=tokens, dim=dim, kind=rng.choice(["layer", "rms"]), dtype=dtype, rdtype=rdtype,
                    out=rng.choice([half, half, "f32"]))
    return dict(op=op, tokens=tokens, dim=dim, kind=rng.choice(["none", "layer", "rms", "rms"]), dtype=dtype,
                rdtype=rng.choice([None, rdtype]))


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

    def rand(*shape, scale=1.0, shift=0.0, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device="cuda").mul_(scale).add_(shift).to(dtype)

    if case["op"] == "linear_q8":
        m, k, n = case["m"], case["k"], case["n"]

        def codes(rows, scale):
            y = rand(rows, k, scale=scale)
            s = y.abs().amax(1) / 127
            return (y / s[:, None]).round_().to(torch.int8), s
        (x, sx), (w, sw) = codes(m, 1.0), codes(n, k ** -0.5)
        out = DTYPES[case["out"]]
        return dict(case=case, x=x, sx=sx, w=w, sw=sw, b=rand(n, scale=0.1) if case["bias"] else None,
                    r=rand(m, n, dtype=out) if case["residual"] else None)
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "local":
        lens = _lengths(case)
        new = [min(case["new"], n) for n in lens] if case["new"] else lens
        hq, hk, d = case["hq"], case["hk"], case["d"]
        cu_q, cu_k = _offsets(new), _offsets(lens)
        as_cu = lambda c: torch.tensor(c, dtype=torch.int32, device="cuda")  # noqa: E731
        kv = rand(cu_k[-1], 2 * hk, d, dtype=dtype)
        return dict(case=case, q=rand(cu_q[-1], hq, d, scale=1.5, dtype=dtype), k=kv[:, :hk], v=kv[:, hk:],
                    cu_q=as_cu(cu_q), cu_k=as_cu(cu_k), max_q=max(new), max_k=max(lens))
    t, dim = case["tokens"], case["dim"]
    return dict(case=case, x=rand(t, dim, scale=2.0, shift=0.3, dtype=dtype),
                r=rand(t, dim, scale=3.0, dtype=DTYPES[case["rdtype"]]) if case["rdtype"] else None,
                w=rand(dim, scale=0.1, shift=1.0) if case["kind"] != "none" else None,
                b=rand(dim, scale=0.1) if case["kind"] == "layer" else None)


# --------------------------------------------------------------------- run --
EPS = 1e-5


@functools.lru_cache(maxsize=1)
def _ops():
    from browservec_amd import DeviceContext, EmbedOps

    return EmbedOps(DeviceContext(0))


def run(state):
    case = state["case"]
    return (_own if own else _plain)[case["op"]](state, case)


def _own_linear_q8(s, c):
    return _ops().linear_q8(s["x"], s["sx"], s["w"], s["sw"], bias=s["b"], residual=s["r"], activation=c["act"],
                            out_dtype=DTYPES[c["out"]])


def _own_add_norm(s, c):
    y, total = _ops().add_norm(s["x"], s["r"], weight=s["w"], bias=s["b"], kind=c["kind"], eps=EPS,
                               out_dtype=DTYPES[c["out"]])
    return dict(y=y, total=total)


def _values(q, scales):
    """What codes and scales stand for, in 16 bits."""
    return torch.mul(q, scales[:, None], out=torch.empty(q.shape, dtype=torch.bfloat16, device=q.device))


def _own_norm_q8(s, c):
    q, scales, total = _ops().norm_q8(s["x"], residual=s["r"], weight=s["w"], bias=s["b"], kind=c["kind"], eps=EPS)
    return dict(y=_values(q, scales), scales=scales, total=total)


def _own_local(s, c):
    return _ops().attention(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], max_q=s["max_q"], max_k=s["max_k"],
                            causal=c["causal"], window=(c["left"], c["right"]), sinks=c["sinks"])


_own = dict(linear_q8=_own_linear_q8, add_norm=_own_add_norm, norm_q8=_own_norm_q8, local=_own_local)


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


def _plain_linear_q8(s, c):
    y = torch.matmul(s["x"].float(), s["w"].float().t())
    y = y * s["sx"][:, None] * s["sw"]
    if s["b"] is not None:
        y = y + s["b"]
    y = _act(y, c["act"])
    if s["r"] is not None:
        y = y + s["r"].float()
    return y.to(DTYPES[c["out"]])


def _plain_sum(s, c):
    t = s["x"].float()
    return t if s["r"] is None else t + s["r"].float()


def _normed(x, w, b, kind):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    if kind != "none":
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    if w is not None:
        x = x * w
    return x if b is None else x + b


def _plain_add_norm(s, c):
    t = _plain_sum(s, c)
    return dict(y=_normed(t, s["w"], s["b"], c["kind"]).to(DTYPES[c["out"]]), total=t.to(s["r"].dtype))


def _plain_norm_q8(s, c):
    t = _plain_sum(s, c)
    y = _normed(t, s["w"], s["b"], c["kind"])
    top = y.abs().amax(-1, keepdim=True)
    q = torch.where(top > 0, y * (127 / top), torch.zeros_like(y)).round().to(torch.int8)
    scales = top[:, 0] / 127
    return dict(y=_values(q, scales), scales=scales, total=None if s["r"] is None else t.to(s["r"].dtype))


def _plain_local(s, c):
    """Blocks of queries side by side, each with the keys that some of its queries see: the window's span, and the first keys."""
    q, k, v, cu_q, cu_k = s["q"], s["k"], s["v"], s["cu_q"].long(), s["cu_k"].long()
    hq, hk, d, lq, lk = c["hq"], c["hk"], c["d"], s["max_q"], s["max_k"]
    left, right = min(c["left"], lk), 0 if c["causal"] else min(c["right"], lk)
    batch, group, dev = cu_q.numel() - 1, c["hq"] // c["hk"], q.device
    size = min(lq, max(64, left + right))  # queries of a block
    blocks, span = (lq + size - 1) // size, size + left + right
    nq, nk = cu_q[1:] - cu_q[:-1], cu_k[1:] - cu_k[:-1]
    i = torch.arange(blocks, device=dev)[:, None] * size + torch.arange(size, device=dev)
    at_q = (cu_q[:-1, None, None] + i).clamp(max=q.shape[0] - 1)               # [batch, blocks, size]
    place = i + (nk - nq)[:, None, None]
    j = (place[:, :, :1] - left) + torch.arange(span, device=dev)               # [batch, blocks, span]
    j = torch.cat([torch.arange(c["sinks"], device=dev).expand(batch, blocks, c["sinks"]), j], -1)
    first = torch.arange(j.shape[-1], device=dev) < c["sinks"]
    keys = j.shape[-1]
    at_k = (cu_k[:-1, None, None] + j.clamp(min=0)).clamp(max=k.shape[0] - 1)
    near = (j[:, :, None, :] >= place[..., None] - left) & (j[:, :, None, :] <= place[..., None] + right)
    seen = torch.where(first, ~near & ((place[..., None] >= j[:, :, None, :]) | (not c["causal"])), near)
    seen = seen & (j >= 0)[:, :, None, :] & (j < nk[:, None, None])[:, :, None, :]
    many = batch * blocks * hk
    qs = q.float()[at_q].view(batch, blocks, size, hk, group, d).permute(0, 1, 3, 4, 2, 5).reshape(many, group * size, d)
    ks = k.float()[at_k].permute(0, 1, 3, 4, 2).reshape(many, d, keys)
    vs = v.float()[at_k].permute(0, 1, 3, 2, 4).reshape(many, keys, d)
    score = torch.matmul(qs, ks).mul_(d ** -0.5).view(batch, blocks, hq, size, keys)
    score.masked_fill_(~seen[:, :, None], float("-inf"))
    top = score.amax(-1, keepdim=True).clamp(min=-1e30)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(many, group * size, keys), vs).view(batch, blocks, hq, size, d)
    o = torch.where(total > 0, o / total, torch.zeros_like(o)).permute(0, 1, 3, 2, 4).reshape(batch, blocks * size, hq, d)
    t = torch.arange(q.shape[0], device=dev)
    of = (t[:, None] >= cu_q[1:]).sum(1)
    return o[of, t - cu_q[of]].to(q.dtype)


_plain = dict(linear_q8=_plain_linear_q8, add_norm=_plain_add_norm, norm_q8=_plain_norm_q8, local=_plain_local)


# -------------------------------------------------------------------- work --
def _pairs(case):
    """Visible pairs of a head, and the keys that some query sees."""
    left, right, sinks = case["left"], 0 if case["causal"] else case["right"], case["sinks"]
    pairs = keys = 0
    for n in _lengths(case):
        lq = min(case["new"], n) if case["new"] else n
        p = torch.arange(n - lq, n)
        a, e = (p - left).clamp(min=0), (p + right + 1).clamp(max=n)
        firsts = torch.minimum(a, torch.full_like(a, sinks))
        pairs += int((e - a + firsts).sum())
        keys += int(e[-1] - a[0]) + int(firsts[0])
    return pairs, keys


def work(case):
    if case["op"] == "linear_q8":
        m, k, n = case["m"], case["k"], case["n"]
        return dict(bytes=m * k + n * k + 4 * (m + n + n * case["bias"]) + m * n * (1 + case["residual"]) * BYTES[case["out"]],
                    flops=2 * m * n * k)
    if case["op"] == "local":
        pairs, keys = _pairs(case)
        rows = sum(min(case["new"], n) if case["new"] else n for n in _lengths(case))
        return dict(bytes=(2 * rows * case["hq"] + 2 * keys * case["hk"]) * case["d"] * BYTES[case["dtype"]],
                    flops=4 * pairs * case["d"] * case["hq"])
    n, b = case["tokens"] * case["dim"], BYTES[case["dtype"]]
    added = 2 * BYTES[case["rdtype"]] if case["rdtype"] else 0
    out = BYTES[case["out"]] if case["op"] == "add_norm" else 1
    return dict(bytes=n * (b + added + out) + (4 * case["tokens"] if case["op"] == "norm_q8" else 0), flops=10 * n)


# ------------------------------------------------------------------- exact --
def exact(case, seed):
    s = prepare(case, seed)
    f = lambda x: None if x is None else x.double()  # noqa: E731
    if case["op"] == "linear_q8":
        z = (f(s["x"]) * f(s["sx"])[:, None]) @ (f(s["w"]) * f(s["sw"])[:, None]).t().contiguous()
        z = z if s["b"] is None else z.add_(f(s["b"]))
        z = {"none": lambda z: z, "relu": lambda z: z.clamp(min=0), "gelu": lambda z: z * torch.special.ndtr(z),
             "gelu_tanh": lambda z: z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)),
             "silu": lambda z: z * torch.sigmoid(z)}[case["act"]](z)
        return z if s["r"] is None else z + f(s["r"])
    if case["op"] == "local":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        group, left, right = case["hq"] // case["hk"], case["left"], 0 if case["causal"] else case["right"]
        cu_q, cu_k = s["cu_q"].tolist(), s["cu_k"].tolist()
        for a, e, ka, ke in zip(cu_q, cu_q[1:], cu_k, cu_k[1:]):
            n, step = ke - ka, 2048
            for r in range(a, e, step):
                q = s["q"][r:min(e, r + step)]
                p = torch.arange(r, r + q.shape[0], device="cuda") - e + n  # the queries' places
                lo, hi = max(0, int(p[0]) - left), min(n, int(p[-1]) + right + 1)
                j = torch.cat([torch.arange(0, min(case["sinks"], lo), device="cuda"), torch.arange(lo, hi, device="cuda")])
                ok = ((j >= p[:, None] - left) | (j < case["sinks"])) & ((j <= p[:, None] + right) | ((j < case["sinks"]) & (not case["causal"])))
                for h in range(case["hk"]):
                    k, v = f(s["k"][ka + j, h]), f(s["v"][ka + j, h])
                    w = f(q[:, h * group:(h + 1) * group]).permute(1, 0, 2).reshape(-1, q.shape[2]) @ k.t().contiguous()
                    w = (w / math.sqrt(case["d"])).view(group, q.shape[0], j.numel()).masked_fill(~ok, -math.inf)
                    w = torch.nan_to_num(torch.softmax(w, -1), nan=0.0)
                    out[r:r + q.shape[0], h * group:(h + 1) * group] = torch.matmul(w, v).permute(1, 0, 2)
        return out
    t = f(s["x"]) if s["r"] is None else f(s["x"]) + f(s["r"])
    y = t
    if case["kind"] == "layer":
        y = (y - y.mean(-1, keepdim=True)) / torch.sqrt(y.var(-1, unbiased=False, keepdim=True) + EPS)
    elif case["kind"] == "rms":
        y = y / torch.sqrt(y.pow(2).mean(-1, keepdim=True) + EPS)
    y = y if s["w"] is None else y * f(s["w"])
    y = y if s["b"] is None else y + f(s["b"])
    if case["op"] == "add_norm":
        return dict(y=y, total=t)
    scales = torch.linalg.vector_norm(y, math.inf, dim=-1) / 127
    return dict(y=torch.round(y / scales[:, None]) * scales[:, None], scales=scales, total=None if s["r"] is None else t)
