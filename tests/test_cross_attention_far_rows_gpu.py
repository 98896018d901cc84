"""Cross attention rows whose largest score is far from zero: samples whose keys are all masked additively, query rows of
a large constant bias, rows whose first or last keys lie far from the others.

Scores are fp32, so the reference rounds them to fp32: q and k hold -1, 0 and 1 and the scale is 1/8, which makes every
product exact, and a score that adds to the mask term or the bias is rounded once.  Its softmax does not change when a row
is shifted, so the bounds are those of rows near zero.
"""

import math

import pytest
import torch

from attention_reference import check, reference
from test_cross_attention_gpu import run, to_cuda

pytestmark = pytest.mark.gpu

SCALE = 0.125
SHIFTS = [-1e4, -1e6, -1e9, -1e10, -1e12, -1e30, 1e4, 1e6]
# b, nq, nk, h, hk, d, share, gate
ONE_TILE = (2, 130, 200, 2, 1, 32, 2, True)
WIDE = (2, 130, 200, 2, 1, 128, 2, True)
TWO_TILES = (80, 140, 150, 2, 2, 24, 1, False)
FEW = (2, 20, 300, 2, 2, 64, 1, True)
GENERIC = (4, 40, 50, 2, 2, 32, 2, True)
STEP = (2, 3, 200, 4, 2, 64, 2, False)
SHAPES = dict(one_tile=ONE_TILE, wide=WIDE, two_tiles=TWO_TILES, few=FEW, generic=GENERIC, step=STEP)


def exact_inputs(shape, dtype):
    b, nq, nk, h, hk, d, _, gate = shape
    g = torch.Generator().manual_seed(nq + nk + d)
    signs = lambda *s: torch.randint(-1, 2, s, generator=g).to(dtype)  # noqa: E731
    randn = lambda *s: torch.randn(*s, generator=g).to(dtype)  # noqa: E731
    x = dict(q=signs(b, nq, h, d), k=signs(b, nk, hk, d), v=randn(b, nk, hk, d), scale=SCALE, dy=randn(b, nq, h, d))
    if gate:
        x["gate"] = randn(b, nq, h, d)
    return x


def rounded_reference(x, terms):
    """:func:`reference` of scores rounded to fp32 after the ``terms`` (fp32 [b, h or 1, nq or 1, nk]) have been added one
    by one, in rows shifted to a largest score of 0 where it is past 1024; dbias per sample."""
    k = x["k"].double().repeat_interleave(x["q"].shape[2] // x["k"].shape[2], 2)
    s = SCALE * torch.einsum("bihd,bjhd->bhij", x["q"].double(), k)
    score = s.float()
    assert torch.equal(score.double(), s)
    for t in terms:
        score = score + t
    score = score.double()
    top = score.amax(-1, keepdim=True)
    score = score - torch.where(top.abs() > 1024, top, 0.0)
    # A probability that is 0 in fp32 whatever its score: keep the reference's bound from growing with that score.
    score = score.clamp(min=-300.0)
    given = {n: t for n, t in x.items() if n in ("q", "k", "v", "dy", "gate", "scale")}
    return reference(**given, bias=score - s)


def compare(x, value, bound, share):
    if share:
        for r in (value, bound):
            r["dbias"] = r["dbias"].unflatten(0, (-1, share)).sum(1)
    else:
        value.pop("dbias")
    actual = run(to_cuda(x))
    check(actual, value, bound)
    again = run(to_cuda(x))
    assert all(torch.equal(actual[n], again[n]) for n in actual)
    return actual


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("inf", [1e4, 1e6, 1e9, 1e10, 1e12])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_samples_masked_additively(shape, biased, inf, dtype):
    """Every key of the first sample masked, some of the others'."""
    shape = SHAPES[shape]
    b, nq, nk, h, share = *shape[:4], shape[6]
    x = exact_inputs(shape, dtype)
    g = torch.Generator().manual_seed(nk)
    x["mask"], x["inf"] = (torch.rand(b, nk, generator=g) < 0.7).float(), inf
    x["mask"][0] = 0
    terms = [torch.tensor(inf, dtype=torch.float32) * (x["mask"] - 1)[:, None, None]]
    if biased:  # of whole eighths: the sum with a score is exact
        x["bias"] = (torch.randint(-16, 17, (b // share, h, nq, nk), generator=g) / 8).to(dtype)
        terms.insert(0, x["bias"].float().repeat_interleave(share, 0))
    compare(x, *rounded_reference(x, terms), share if biased else 0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shift", SHIFTS)
@pytest.mark.parametrize("shape", SHAPES)
def test_bias_rows(shape, shift, dtype):
    """Rows of a constant bias, rows whose first 70 or last 70 keys have it, ordinary rows beside them."""
    shape = SHAPES[shape]
    b, nq, nk, h, share = *shape[:4], shape[6]
    x = exact_inputs(shape, dtype)
    bias = torch.zeros(b // share, h, nq, nk)
    bias[:, :, 0::4] = shift
    bias[:, :, 1::4, :70] = shift
    bias[:, :, 2::4, -70:] = shift
    x["bias"] = bias.to(dtype)
    terms = [x["bias"].float().repeat_interleave(share, 0)]
    actual = compare(x, *rounded_reference(x, terms), share)
    assert math.isfinite(float(actual["lse"].sum()))


ABOVE_ONE = [
    # b, nq, nk, h, hk, d, share, gate: query rows that do not fill the gradient kernels' tiles
    (2, 37, 70, 2, 1, 32, 1, True),
    (2, 37, 70, 2, 2, 128, 0, False),
    (4, 20, 96, 2, 2, 32, 2, True),  # fp32: the windows' kernel
    (1, 130, 200, 2, 1, 48, 1, True),
    (2, 3, 90, 4, 2, 64, 1, False),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", ABOVE_ONE)
def test_additive_masks_above_one(shape, dtype):
    """A mask of 2 adds inf to a key's scores: query rows past the last one must not see it."""
    b, nk, share = shape[0], shape[2], shape[6]
    x = exact_inputs(shape, dtype)
    x["mask"], x["inf"] = torch.ones(b, nk), 1e3
    x["mask"][:, 5], x["mask"][:, nk - 1], x["mask"][:, 7] = 2.0, 2.0, 0.0
    terms = [torch.tensor(x["inf"]) * (x["mask"] - 1)[:, None, None]]
    if share:
        x["bias"] = torch.zeros(b // share, shape[3], shape[1], nk, dtype=dtype)
    compare(x, *rounded_reference(x, terms), share)
