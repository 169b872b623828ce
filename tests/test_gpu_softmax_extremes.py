"""Softmax attention (qlka.softmax) where scores, biases and scales are as large or as small as they may be: forward and
gradients against the float64 oracle's bounds.

A row's probabilities depend on the differences of its scores alone, so cases are built whose differences are known exactly
(equal scores, or some so much larger than the others that these weigh 0), and the oracle forms the same probabilities from
scores of the ordinary size."""

import math

import pytest
import torch

from oracle import softmax as oracle
from qlka.softmax import softmax_attention
from test_gpu_softmax import BF16, BOTH, F32, PAST, check, make, reference, run

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


@TYPES
@pytest.mark.parametrize("scale,bias", [(0.125, -1e38), (0.125, -4.5e37), (2.0 ** -96, 1e10), (2.0 ** -96, -1e10), (2.0 ** -90, 1e12)])
def test_log_sums_far_larger_than_the_scale(dev, scale, bias, dtype):
    """Rows of one key: its probability is 1 whatever its score."""
    t = make(2, 4, 2, 40, 1, 64, dtype, seed=1, bias=PAST)
    t["table"].fill_(bias)
    want = equal_scores(t, torch.ones(2, 40, 1, dtype=torch.bool), scale)
    check(run(dev, t, PAST, scale=scale), want, ["out", "gq", "gk", "gv"])


@TYPES
@pytest.mark.parametrize("M,N,causal", [(1, 50, False), (40, 50, False), (70, 300, True), (3, 4100, False), (600, 65, False)])
@pytest.mark.parametrize("scale,bias", [(0.125, -1e38), (0.125, 2e38), (0.125, -1e30), (2.0 ** -96, 1e10)])
def test_biases_that_swallow_the_scores(dev, scale, bias, M, N, causal, dtype):
    """A bias so large that scores next to it are all the same: n keys share a row by 1 / n each, in the gradients too."""
    t = make(2, 4, 2, M, N, 64, dtype, seed=1, bias=PAST, keep="random")
    t["table"].fill_(bias)
    start = N - M if causal else 0
    want = equal_scores(t, oracle.visible(2, M, N, t["keep"], causal, start), scale)
    check(run(dev, t, PAST, scale=scale, causal=causal, start=start), want, ["out", "gq", "gk", "gv"])


@TYPES
@pytest.mark.parametrize("M,N", [(40, 256), (200, 300), (1, 300)])
@pytest.mark.parametrize("scale", [2.0 ** 12, 2.0 ** 22, 2.0 ** 30, 2.0 ** 96])
@pytest.mark.parametrize("masked", [False, True], ids=["all", "keep"])
def test_large_scales_gradients(dev, scale, M, N, masked, dtype):
    t = whole(make(2, 1, 1, M, N, 64, dtype, seed=M, keep="random" if masked else None))
    t["g"] = t["g"] * 2.0 ** -40                   # so that the largest scale's gradients stay in range
    top = largest(t, oracle.visible(2, M, N, t["keep"]))
    check(run(dev, t, scale=scale), equal_scores(t, top[:, 0], scale))


@TYPES
@pytest.mark.parametrize("bias", [None, BOTH], ids=["plain", "bias"])
@pytest.mark.parametrize("size", [200.0, 3000.0])
@pytest.mark.parametrize("M,N", [(2, 90), (150, 200)])
def test_scores_of_thousands(dev, M, N, size, bias, dtype):
    """Where the log sums begin to be taken off in two steps: all values against the oracle."""
    t = make(2, 4, 2, M, N, 64, dtype, seed=6, bias=bias)
    if bias:
        t["table"] += size
        check(run(dev, t, bias), reference(t, bias))
    scale = size / 16
    t = dict(t, table=None)
    check(run(dev, t, scale=scale), reference(t, scale=scale))


@TYPES
@pytest.mark.parametrize("M", [1, 3, 70])
def test_gradients_of_large_scales_stay_finite(dev, M, dtype):
    """Scores whose roundings are larger than 1, formed once in the forward and again in the backward: no probability is
    larger than 1, so a value's gradient is at most the sum of its queries'."""
    t = make(2, 2, 2, M, 700, 64, dtype, seed=3)
    for scale in (2.0 ** 20, 2.0 ** 24, 2.0 ** 31):
        got = run(dev, t, scale=scale)
        for n in got:
            assert torch.isfinite(got[n]).all(), (n, scale)
        most = t["g"].double().abs().sum(2, keepdim=True)
        assert (got["gv"].double().cpu().abs() <= most * (1 + 2 ** -7)).all(), scale


def test_the_c_entries_with_lse_alone(dev):
    """lse is the log2 of a row's sum, and enough for the backward where that is of the ordinary size."""
    import ctypes

    from qlka import _lib
    lib = _lib.load()
    t = make(2, 2, 2, 50, 70, 64, F32, seed=2, keep="holes")
    want = reference(t)
    x = {n: t[n].to(dev) for n in "qkvg"}
    keep = t["keep"].to(dev)
    r = {n: torch.empty_like(x[m]) for n, m in (("out", "q"), ("g_q", "q"), ("g_k", "k"), ("g_v", "v"))}
    lse = torch.empty(2, 2, 50, device=dev)
    a = _lib.SoftmaxArgs(dtype=0, B=2, H=2, G=2, M=50, N=70, D=64, scale=0.125, lse=lse.data_ptr(),
                         keep=keep.data_ptr(), keep_stride=70)
    for n, y in [(n, x[n]) for n in "qkv"] + [("g_out", x["g"])] + list(r.items()):
        setattr(a, n, y.data_ptr())
        setattr(a, n + "_stride", (ctypes.c_int64 * 3)(*y.stride()[:3]))
    stream = torch.cuda.current_stream().cuda_stream
    for fn, need in ((lib.qlka_softmax_fwd, lib.qlka_softmax_fwd_ws_bytes),
                     (lib.qlka_softmax_bwd, lib.qlka_softmax_bwd_ws_bytes)):
        ws = torch.empty(max(need(ctypes.byref(a)), 16), dtype=torch.uint8, device=dev)
        assert fn(ctypes.byref(a), ws.data_ptr(), ws.numel(), stream) == 0
    check({"out": r["out"], "gq": r["g_q"], "gk": r["g_k"], "gv": r["g_v"]}, want)
    s = torch.matmul(t["q"].double(), t["k"].double().transpose(-1, -2)) * 0.125
    s = s.masked_fill(~t["keep"][:, None, None, :], float("-inf"))
    exact = torch.logsumexp(s, -1) / math.log(2)
    none = torch.isinf(exact)
    assert (lse.cpu()[none] == float("inf")).all()
    # 64 products and their sum, the change of units, up to 70 exponentials and their sum, log2 and the sum with the maximum
    size = 0.125 * torch.matmul(t["q"].double().abs(), t["k"].double().abs().transpose(-1, -2)).amax(-1)
    bound = oracle.U * ((64 + 16) * size * 1.5 + (2 * 70 + 32) + 4 * exact.abs())
    assert ((lse.cpu().double() - exact).abs() <= bound)[~none].all()


def highest(t, see, start, bias):
    """(B, H, M, N): the keys of the largest bias that a row sees."""
    B, M, N = see.shape
    value = t["table"].t()[:, oracle.bucket_map(M, N, start, *bias).flatten()].view(1, -1, M, N).expand(B, -1, M, N)
    value = value.masked_fill(~see[:, None], float("-inf"))
    return see[:, None] & (value == value.amax(-1, keepdim=True))


LOWEST, LOWEST_BF16 = torch.finfo(F32).min, torch.finfo(BF16).min
TABLES = {
    "lowest": lambda n: [LOWEST] * n, "lowest_bf16": lambda n: [LOWEST_BF16] * n, "largest": lambda n: [-LOWEST] * n,
    # which of two is the larger one has to be seen where both are below -2.36e38
    "two": lambda n: [LOWEST if i % 3 else LOWEST_BF16 for i in range(n)],
    "close": lambda n: [-2.5e38 if i % 2 else -2.4e38 for i in range(n)],
    "both_ends": lambda n: [LOWEST if i % 2 else -LOWEST for i in range(n)],
    "hidden": lambda n: [0.0] + [LOWEST] * (n - 1),
}


@TYPES
@pytest.mark.parametrize("M,N,causal", [(1, 50, True), (2, 300, False), (40, 50, False), (130, 300, True), (3, 4100, True), (600, 65, False)])
@pytest.mark.parametrize("kind", TABLES)
def test_biases_as_low_and_as_large_as_they_may_be(dev, kind, M, N, causal, dtype):
    """A bucket of the type's lowest value hides its keys from rows that see others, and not from those that do not: these
    see equal scores. "hidden" leaves some rows one bucket of ordinary scores (the queries are 0 there, so they are equal)."""
    t = make(2, 2, 2, M, N, 64, dtype, seed=1, bias=PAST, keep="random")
    t["table"] = torch.tensor(TABLES[kind](32))[:, None].repeat(1, 2)
    if kind == "hidden":
        t["q"] = torch.zeros_like(t["q"])
    start = N - M if causal else 0
    see = oracle.visible(2, M, N, t["keep"], causal, start)
    top = highest(t, see, start, PAST)[:, 0]
    check(run(dev, t, PAST, scale=0.125, causal=causal, start=start), equal_scores(t, top, 0.125), ["out", "gq", "gk", "gv"])


@pytest.mark.parametrize("M,N", [(1, 300), (40, 300), (200, 65), (3, 5000)])
def test_row_sums_of_unrounded_values(dev, M, N):
    """The row sums that the gradients take off, rowsum(dO * O), are formed from out before it is rounded to bfloat16. Scores are
    equal, so that no probability is rounded and out before its rounding is right to fp32; the bounds are then those
    with a table. Values and keys far from 0 show an error that is common to a row's dS."""
    t = make(2, 4, 2, M, N, 64, BF16, seed=9)
    t["q"] = torch.zeros_like(t["q"])
    t["k"] = (t["k"].float() / 8 + 4).to(BF16)
    t["v"] = (t["v"].float() / 8 + 8).to(BF16)
    zeros, none = torch.zeros(1, 4), torch.zeros(M, N, dtype=torch.long)
    want = oracle.attention(t["q"], t["k"], t["v"], 0.125, oracle.visible(2, M, N), t["g"], zeros, none)
    check(run(dev, t), want)
    kept = dict(t, table=torch.zeros(32, 4))                          # with a table that wants no gradient
    x = {n: kept[n].to(dev).requires_grad_(n in "qkv") for n in ("q", "k", "v", "g", "table")}
    out = softmax_attention(x["q"], x["k"], x["v"], table=x["table"], buckets=PAST)
    got = dict(zip(("gq", "gk", "gv"), torch.autograd.grad(out, [x[n] for n in "qkv"], x["g"].detach())), out=out.detach())
    check(got, want)


@TYPES
@pytest.mark.parametrize("D", [8, 32, 80, 128])
@pytest.mark.parametrize("M,N,causal", [(50, 90, True), (100, 300, False), (100, 300, True), (1, 700, True), (900, 70, False)])
def test_extremes_at_other_head_dimensions(dev, M, N, causal, D, dtype):
    """Every instance of the kernels, two and four waves a workgroup, whole and split: a bias of the lowest value everywhere, and
    a large scale of whole numbers, the mask's and the causal order's edges inside tiles."""
    start = N - M if causal else 0
    t = make(2, 4, 2, M, N, D, dtype, seed=D, bias=PAST, keep="random")
    see = oracle.visible(2, M, N, t["keep"], causal, start)
    t["table"].fill_(LOWEST)
    check(run(dev, t, PAST, scale=0.25, causal=causal, start=start), equal_scores(t, see, 0.25), ["out", "gq", "gk", "gv"])
    t = whole(make(2, 1, 1, M, N, D, dtype, seed=D, keep="random"))
    see = oracle.visible(2, M, N, t["keep"], causal, start)
    check(run(dev, t, scale=2.0 ** 30, causal=causal, start=start), equal_scores(t, largest(t, see)[:, 0], 2.0 ** 30))
