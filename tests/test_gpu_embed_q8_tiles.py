"""EmbedOps.linear_q8 by every shape of tile that its plan chooses among, each ragged in
rows, columns and codes, alone and before and behind another (which size goes by which
shape is checked by test_embed_q8_plan.py)."""

import pytest
import torch

from tests.helpers import say
from tests.test_gpu_embed import BF, F32, HF, U, ops, rand  # noqa: F401
from tests.test_gpu_embed_q8 import ACTS, I8, floor_of

pytestmark = pytest.mark.gpu

# (m, n, k, activation): k % 16, n % 8 and the rows of a tile leave a rest in all but the
# last of them
TILES = [
    (7341, 70, 484, "gelu"), (35, 17, 1039, "gelu"), (37, 17, 2068, "none"),                # 64 x 64, steps of 512
    (35, 17, 10, "gelu"), (37, 18, 267, "silu"), (17504, 17, 1037, "none"),                 # 64 x 64, steps of 256
    (16349, 66, 3096, "none"),                                                              # 64 x 128
    (12999, 65, 19, "none"), (16403, 71, 291, "gelu"), (16641, 74, 563, "gelu_tanh"),       # 128 x 128
    (16406, 129, 11, "relu"), (17366, 129, 258, "none"), (19521, 135, 537, "none"),         # 128 x 256, one a CU
    (16043, 581, 212, "none"), (22318, 268, 277, "relu"), (17905, 398, 517, "none"),        # 192 x 256
    (21924, 137, 13, "gelu"), (22600, 132, 72, "silu"), (22318, 148, 271, "gelu"),          # 128 x 256, two a CU
    (12921, 2363, 260, "none"), (20893, 521, 468, "relu"), (15418, 809, 515, "none"),       # 256 x 256
    (16533, 279, 2614, "gelu"), (16729, 857, 456, "none"), (21803, 646, 261, "gelu"), (18630, 842, 2719, "none"),
    (23102, 588, 535, "gelu"), (4760, 4147, 1470, "gelu"), (17420, 1327, 2271, "none"),     # two shapes
    (20011, 1024, 4096, "none"),
]


def device(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def codes(rows, k, seed):
    return torch.randint(-128, 128, (rows, k), generator=device(seed), dtype=torch.int32, device="cuda").to(I8)


def within(got, want, bound, what):
    """On the card, as the results are large."""
    over = (got.double() - want).abs() - bound
    assert not torch.isnan(over).any() and over.max() <= 0, f"{what}: {int((over > 0).sum())} values outside, worst by {over.max():.3g}"


def product(x, sx, w, sw, b, r, act, out):
    """The result in 64 bits and its bound.  The whole sum is exact; rounded to 32 bits,
    multiplied by two scales and added to the bias: four roundings of 2^-24, whose size
    is at most that of the product and the bias.  The activations' slopes stay below 1.13;
    their own arithmetic is within 2^-20 of max(1, |z|).  The residual's addition rounds
    once in 32 bits, the result once to its type."""
    z = (x.double() @ w.double().t().contiguous()) * sx.double()[:, None] * sw.double()
    mag = z.abs()
    if b is not None:
        z, mag = z + b.double(), mag + b.double().abs()
    bound = 1.13 * 4 * 2.0 ** -24 * 1.01 * mag
    if act not in ("none", "relu"):
        bound = bound + 2.0 ** -20 * z.abs().clamp(min=1)
    y = ACTS[act](z)
    if r is not None:
        y = y + r.double()
        bound = bound + 2.0 ** -24 * (y.abs() + bound)
    return y, bound + U[out] * (y.abs() + bound) + floor_of(out)


@pytest.mark.parametrize("out", [BF, HF, F32])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("m,n,k,act", TILES)
def test_linear_q8_tiles(ops, m, n, k, act, out, residual):  # noqa: F811
    """The result lies in wider rows, whose other elements stay as they were; without a
    residual there is a bias."""
    say("linear_q8 tiles", m, n, k, act, out, residual)
    x, w = codes(m, k, 1), codes(n, k, 2)
    sx, sw = (torch.rand(rows, generator=device(3), device="cuda") * 0.02 + 1e-4 for rows in (m, n))
    b = None if residual else torch.randn(n, generator=device(4), device="cuda").to(out)
    wide = torch.full((m + 1, n + 5), 7.0, dtype=out, device="cuda")
    r = torch.randn(m, n, generator=device(5), device="cuda").to(out) if residual else None
    y = wide[:m, 2:n + 2]
    assert ops.linear_q8(x, sx, w, sw, bias=b, residual=r, activation=act, out=y) is y
    within(y, *product(x, sx, w, sw, b, r, act, out), f"{m} x {n}, k {k}")
    assert (wide[m:] == 7).all() and (wide[:, :2] == 7).all() and (wide[:, n + 2:] == 7).all()
    if residual:  # onto itself: the same bits
        y2 = r.clone()
        ops.linear_q8(x, sx, w, sw, residual=y2, activation=act, out=y2)
        assert torch.equal(y2, y)
