"""Softmax attention (qlka.softmax) where scores, biases and scales are as large or as small as they may be: forward and
gradients against the float64 oracle's bounds.

A row's probabilities depend on the differences of its scores alone, so cases are built whose differences are known exactly
(equal scores, or some so much larger than the others that these weigh 0), and the oracle forms the same probabilities from
scores of the ordinary size."""

import pytest
import torch

from oracle import softmax as oracle
from test_gpu_softmax import BF16, F32, check, make, run

pytestmark = pytest.mark.gpu

TYPES = pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])


def equal_scores(t, see, scale):
    """The oracle where every key in `see` (B, M, N) has the same score as the others of its row: a scale of 2^-80 leaves
    scores below 2^-70, whose exponentials are 1 within 2^-70; what is proportional to the scale is multiplied up again."""
    down = 2.0 ** -80
    want = oracle.attention(t["q"], t["k"], t["v"], down, see, t["g"])
    for d in (want, want["bound"]):
        for n in ("gq", "gk"):
            d[n] = d[n] * (scale / down)
    return want



def whole(t, seed=0, most=2):
    """q and k of small whole numbers: every score is exact before it is scaled, and scores are equal or 1 apart at least."""
    gen = torch.Generator().manual_seed(seed)
    for n in "qk":
        t[n] = torch.randint(-most, most + 1, t[n].shape, generator=gen).to(t[n].dtype)
    return t


def largest(t, see):
    """(B, H, M, N): the keys of the largest scores that a row sees."""
    k = t["k"].repeat_interleave(t["q"].shape[1] // t["k"].shape[1], 1)
    s = torch.matmul(t["q"].double(), k.double().transpose(-1, -2)).masked_fill(~see[:, None], float("-inf"))
    return see[:, None] & (s == s.amax(-1, keepdim=True))


@TYPES
@pytest.mark.parametrize("M,N", [(40, 256), (200, 300), (70, 4000), (1, 300), (2, 4100)])
@pytest.mark.parametrize("scale", [2.0 ** 12, 2.0 ** 20, 2.0 ** 30, -2.0 ** 30, 2.0 ** 96, 1e9])
@pytest.mark.parametrize("masked", [False, True], ids=["all", "keep"])
def test_large_scales_forward(dev, scale, M, N, masked, dtype):
    """The keys of a row's largest score share it, on tiles with and without a mask and for single tokens,
    split and whole."""
    t = whole(make(1, 2, 1, M, N, 64, dtype, seed=M, keep="random" if masked else None), most=2 if M > 4 else 9)
    see = oracle.visible(1, M, N, t["keep"])
    if scale < 0:
        t["q"] = -t["q"]
    top = largest(t, see)
    if scale < 0:
        t["q"] = -t["q"]
    for h in range(2):
        want = equal_scores({n: t[n][:, h:h + 1] if n in "qg" else t[n] for n in "qkvg"}, top[:, h], scale)
        if h == 0:
            out = run(dev, t, train=False, scale=scale)["out"]
        check({"out": out[:, h:h + 1]}, want)


@TYPES
@pytest.mark.parametrize("M", [1, 3, 70])
@pytest.mark.parametrize("scale", [2.0 ** 24, 2.0 ** 31, 2.0 ** 60])
def test_large_scales_of_any_values_stay_finite(dev, scale, M, dtype):
    """Scores whose roundings are larger than 1: which key takes the row is a matter of rounding, but it is a mean of values."""
    t = make(2, 2, 2, M, 700, 64, dtype, seed=3)
    out = run(dev, t, train=False, scale=scale)["out"].float().cpu()
    lo, hi = (f(t["v"].float(), 2, keepdim=True) for f in (torch.amin, torch.amax))
    slack = 2 ** -7 if dtype == BF16 else 2 ** -16
    assert (out >= lo - slack * lo.abs()).all() and (out <= hi + slack * hi.abs()).all()


@TYPES
@pytest.mark.parametrize("M", [1, 2, 40])
def test_equal_products_stay_equal(dev, M, dtype):
    """Keys of the same elements in another order against a query of equal ones: their sums are exact, so the scores are the
    same however large the scale is."""
    t = make(2, 2, 2, M, 200, 64, dtype, seed=4)
    t["q"] = torch.ones_like(t["q"])
    gen = torch.Generator().manual_seed(8)
    row = torch.randint(-9, 20, (64,), generator=gen)
    t["k"] = row[torch.rand(t["k"].shape, generator=gen).argsort(-1)].to(dtype)
    want = equal_scores(t, torch.ones(2, M, 200, dtype=torch.bool), 1e9)
    check(run(dev, t, train=False, scale=1e9), want, ["out"])
