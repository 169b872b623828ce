"""Softmax attention (qlka.softmax) on the GPU against the float64 oracle, forward and gradients, within the bounds that
oracle/softmax.py derives; masks, lengths, strides, shared heads, the position bias and its table's gradient."""

import pytest
import torch

from oracle import softmax as oracle
from qlka.softmax import RelativeBuckets, relative_bias, softmax_attention

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
TINY = 1e-30


def make(B, H, G, M, N, D, dtype, seed=0, bias=None, keep=None):
    gen = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(s, generator=gen)  # noqa: E731
    t = {"q": (rand(B, H, M, D) * 1.5).to(dtype), "k": rand(B, G, N, D).to(dtype), "v": rand(B, G, N, D).to(dtype),
         "g": rand(B, H, M, D).to(dtype), "table": None, "keep": None}
    if bias:
        t["table"] = rand(bias.num_buckets, H)
    if keep == "random":
        t["keep"] = torch.rand(B, N, generator=gen) < 0.6
    elif keep == "padded":
        t["keep"] = torch.arange(N)[None, :] < torch.randint(1, N + 1, (B, 1), generator=gen)
    elif keep == "holes":                          # whole tiles without a key, and a batch without any
        t["keep"] = (torch.arange(N)[None, :] // 70 % 3 == 1).repeat(B, 1)
        t["keep"][0] = False
    return t


def reference(t, bias=None, causal=False, start=0, scale=None):
    B, H, M, D = t["q"].shape
    N = t["k"].shape[2]
    buckets = oracle.bucket_map(M, N, start, *bias) if bias else None
    return oracle.attention(t["q"], t["k"], t["v"], D ** -0.5 if scale is None else scale,
                            oracle.visible(B, M, N, t["keep"], causal, start), t["g"], t["table"], buckets)


def run(dev, t, bias=None, train=True, **kw):
    x = {n: None if a is None else a.to(dev) for n, a in t.items()}
    leaves = [x[n] for n in ("q", "k", "v", "table") if x[n] is not None]
    for a in leaves:
        a.requires_grad_(train)
    out = softmax_attention(x["q"], x["k"], x["v"], keep=x["keep"], table=x["table"], buckets=bias, **kw)
    r = {"out": out.detach()}
    if train:
        r.update(zip(("gq", "gk", "gv", "gtable"), torch.autograd.grad(out, leaves, x["g"])))
    return r


def check(got, want, names=None):
    for n in names or got:
        off = (got[n].double().cpu() - want[n]).abs()
        over = off / (want["bound"][n] + TINY)
        assert torch.isfinite(got[n]).all(), n
        assert off.numel() == 0 or over.max() <= 1, f"{n}: {over.max():.3g} times its bound ({off.max():.3g})"


BOTH, PAST = RelativeBuckets(), RelativeBuckets(bidirectional=False)

SHAPES = [
    # B, H, G, M, N, D
    (1, 1, 1, 1, 1, 1),
    (2, 3, 3, 1, 5, 8),
    (2, 2, 1, 5, 64, 64),
    (1, 2, 2, 33, 65, 32),
    (2, 4, 2, 65, 65, 32),
    (1, 3, 1, 100, 129, 64),
    (2, 2, 2, 64, 200, 17),
    (1, 2, 2, 200, 63, 80),
    (1, 2, 1, 130, 70, 128),
    (1, 1, 1, 97, 300, 127),
    (1, 2, 2, 300, 515, 64),
]


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("kind", ["plain", "keep", "causal", "bias", "bias_causal_keep"])
def test_matches_the_oracle(dev, kind, shape, dtype):
    bias = {"bias": BOTH, "bias_causal_keep": PAST}.get(kind)
    causal = "causal" in kind
    M, N = shape[3], shape[4]
    start = N - M if causal else (3 if bias else 0)
    t = make(*shape, dtype, seed=sum(shape), bias=bias, keep="random" if "keep" in kind else None)
    check(run(dev, t, bias, causal=causal, start=start), reference(t, bias, causal, start))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("M", [1, 2, 8, 9, 40, 200])
@pytest.mark.parametrize("keep", ["padded", "holes"])
def test_masked_rows_may_hold_anything(dev, keep, M, dtype):
    t = make(3, 4, 2, M, 333, 64, dtype, seed=M, bias=BOTH, keep=keep)
    want = reference(t, BOTH, start=40)
    clean = run(dev, t, BOTH, start=40)
    check(clean, want)
    hidden = ~t["keep"][:, None, :, None].expand_as(t["k"])
    t["k"] = t["k"].masked_fill(hidden, float("nan"))
    t["v"] = t["v"].masked_fill(hidden, float("inf"))
    dirty = run(dev, t, BOTH, start=40)
    for n in clean:
        assert torch.equal(clean[n], dirty[n]), n
    assert (dirty["gk"].cpu()[hidden] == 0).all() and (dirty["gv"].cpu()[hidden] == 0).all()
    if keep == "holes":
        assert (dirty["out"][0] == 0).all() and (dirty["gq"][0] == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("M,N,start", [(70, 90, -30), (5, 200, -3), (200, 40, -150), (1, 300, 4), (3, 70, -1), (64, 64, 500)])
def test_causal_rows_without_keys(dev, M, N, start, dtype):
    t = make(2, 4, 2, M, N, 64, dtype, seed=M + N, bias=PAST)
    got, want = run(dev, t, PAST, causal=True, start=start), reference(t, PAST, True, start)
    check(got, want)
    if start < 0:
        assert (got["out"][:, :, :-start] == 0).all() and (got["gq"][:, :, :-start] == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("B,M,N", [(2, 0, 5), (2, 5, 0), (0, 5, 5), (2, 0, 0)])
def test_empty(dev, B, M, N, dtype):
    t = make(B, 2, 1, M, N, 16, dtype, bias=BOTH)
    got = run(dev, t, BOTH)
    assert got["out"].shape == (B, 2, M, 16)
    for n in got:
        assert (got[n] == 0).all(), n


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("shape", [(1, 2, 2, 64, 4000, 64), (1, 1, 1, 20, 3001, 40), (2, 6, 2, 1, 33000, 64), (1, 4, 1, 2, 5000, 64), (2, 2, 1, 1, 4099, 128),
                                   (1, 2, 1, 1500, 40, 64), (1, 2, 2, 1200, 100, 32)],
                         ids=lambda s: "x".join(map(str, s)))
def test_split_axes(dev, shape, dtype):
    """Few rows against a long axis: partial sums joined afterwards."""
    t = make(*shape, dtype, seed=7, bias=BOTH, keep="padded")
    start = shape[4] // 2
    check(run(dev, t, BOTH, start=start), reference(t, BOTH, start=start))


@pytest.mark.parametrize("bias", [RelativeBuckets(2, 5), RelativeBuckets(4, 3), RelativeBuckets(1, 1, False),
                                  RelativeBuckets(3, 9, False), RelativeBuckets(256, 200), RelativeBuckets(64, 1000, False),
                                  RelativeBuckets(32, 20, True)], ids=str)
@pytest.mark.parametrize("M", [1, 150])
def test_bucket_counts(dev, bias, M):
    t = make(1, 2, 2, M, 400, 32, F32, seed=3, bias=bias)
    check(run(dev, t, bias, start=130), reference(t, bias, start=130))


@pytest.mark.parametrize("scale", [-0.3, 0.0, 2.0])
@pytest.mark.parametrize("M", [2, 70])
def test_scales(dev, scale, M):
    t = make(2, 2, 1, M, 90, 32, F32, keep="random")
    check(run(dev, t, scale=scale), reference(t, scale=scale))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("M", [1, 77])
@pytest.mark.parametrize("D", [64, 20])
def test_strides(dev, D, M, dtype):
    """Heads of a packed projection, a broadcast batch, rows of odd alignment, a mask cut out of a larger one."""
    t = make(2, 4, 2, M, 130, D, dtype, seed=5, keep="random")
    want = reference(t)
    x = {n: None if a is None else a.to(dev) for n, a in t.items()}

    def views(a, pad):
        B, H, S, D = a.shape
        buf = torch.full((B, S, H * D + pad), float("nan"), dtype=a.dtype, device=dev)
        view = buf[:, :, pad:].view(B, S, H, D) if pad == 0 else buf[:, :, pad:].unflatten(2, (H, D))
        view = view.transpose(1, 2)
        view.copy_(a)
        return view

    for pad in (0, 1, 8):
        leaves = [views(x[n], pad).requires_grad_(True) for n in "qkv"]
        keep = torch.zeros(2, 200, dtype=torch.bool, device=dev)[:, 3:133].copy_(x["keep"])
        out = softmax_attention(*leaves, keep=keep)
        got = dict(zip(("gq", "gk", "gv"), torch.autograd.grad(out, leaves, x["g"])), out=out.detach())
        check(got, want)
    # every batch and head shares one row of values; the gradient of what was broadcast is their sum
    one = {n: x[n][:1, :1].clone().requires_grad_(True) for n in "kv"}
    spread = [one[n].expand(2, 2, -1, -1) for n in "kv"]
    out = softmax_attention(x["q"], *spread)
    grads = torch.autograd.grad(out, [one["k"], one["v"]], x["g"])
    whole = [a.detach().clone().requires_grad_(True) for a in spread]
    out2 = softmax_attention(x["q"], *whole)
    assert torch.equal(out, out2)
    for a, b in zip(grads, torch.autograd.grad(out2, whole, x["g"])):
        # the sum of the four, in any order and rounded after each: half a step of the largest partial sum three times
        h = max(torch.finfo(dtype).eps / 2, 2 ** -24)
        size = b.double().abs().sum((0, 1), keepdim=True)
        assert ((a.double() - b.double().sum((0, 1), keepdim=True)).abs() <= 4 * h * size + TINY).all()


def test_columns_apart_are_copied(dev):
    t = make(1, 2, 2, 40, 50, 16, F32)
    want = reference(t)
    flip = lambda a: a.to(dev).transpose(2, 3).contiguous().transpose(2, 3).requires_grad_(True)  # noqa: E731
    leaves = [flip(t[n]) for n in "qkv"]
    out = softmax_attention(*leaves)
    grads = torch.autograd.grad(out, leaves, flip(t["g"]).detach())
    check(dict(zip(("out", "gq", "gk", "gv"), (out.detach(),) + grads)), want)


@pytest.mark.parametrize("M", [1, 100])
def test_minus_infinity_in_the_table(dev, M):
    """A bucket of -inf hides its keys; a row that keeps none gives zeros."""
    bias = RelativeBuckets(4, 3, True)              # buckets 0, 1 (0, >= 1 before), 2, 3 (none, >= 1 after)
    t = make(1, 2, 2, M, 60, 32, F32, seed=2, bias=bias)
    t["table"][1] = float("-inf")
    t["table"][3] = float("-inf")
    start = 0 if M > 1 else 200
    got, want = run(dev, t, bias, start=start), reference(t, bias, start=start)
    check(got, want, ["out", "gq", "gk", "gv"])
    assert torch.isfinite(got["gtable"]).all()


@pytest.mark.parametrize("M", [1, 100])
def test_nan_in_the_table_where_keys_are_masked(dev, M):
    bias = RelativeBuckets(4, 3, True)
    t = make(1, 2, 2, M, 90, 32, F32, seed=2, bias=bias)
    t["keep"] = (torch.arange(90) < 70)[None, :]
    clean = run(dev, dict(t, table=t["table"][:, :].clone()), bias, start=80)      # every kept key lies before the queries
    t["table"][2:] = float("nan")
    t["table"][0] = float("inf")
    dirty = run(dev, t, bias, start=80)
    for n in ("out", "gq", "gk", "gv"):
        assert torch.equal(clean[n], dirty[n]), n
    assert torch.equal(clean["gtable"][1], dirty["gtable"][1])


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
def test_large_scores(dev, dtype):
    """Scores of hundreds: one key takes the row; and the running maximum rises along the keys."""
    t = make(1, 2, 2, 70, 300, 64, dtype)
    t["k"] = (t["k"].float() * torch.linspace(0.1, 30, 300)[None, None, :, None]).to(dtype)
    for M in (70, 2):
        s = dict(t, q=t["q"][:, :, :M].contiguous(), g=t["g"][:, :, :M].contiguous())
        check(run(dev, s), reference(s))


def test_gradient_against_differences(dev):
    t = make(2, 4, 2, 40, 70, 32, F32, bias=BOTH, keep="random")
    x = {n: None if a is None else a.to(dev) for n, a in t.items()}
    got = run(dev, t, BOTH, start=10)
    loss = lambda y: (softmax_attention(y["q"], y["k"], y["v"], keep=x["keep"], table=y["table"], buckets=BOTH, start=10).double()  # noqa: E731
                      * x["g"].double()).sum().item()
    gen = torch.Generator().manual_seed(1)
    for n, name in (("q", "gq"), ("k", "gk"), ("v", "gv"), ("table", "gtable")):
        way = torch.randn(x[n].shape, generator=gen).to(dev)
        h = 1e-2 / way.norm().item() * 4
        diff = (loss({**x, n: x[n].detach() + h * way}) - loss({**x, n: x[n].detach() - h * way})) / (2 * h)
        want = (got[name].double() * way.double()).sum().item()
        # third derivative over 6 times a step of 0.04 squared, and 2^-22 of the loss's terms over the step
        terms = 2 ** -22 * x["g"].abs().sum().item() ** 0.5 * 4 / (2 * h)
        assert abs(diff - want) <= 0.04 ** 2 * got[name].norm().item() * way.norm().item() + terms, n


def test_only_what_is_asked_for(dev):
    t = make(1, 2, 1, 50, 60, 32, BF16, bias=BOTH)
    want = run(dev, t, BOTH)
    x = {n: a.to(dev) for n, a in t.items() if a is not None}
    for names in (["q"], ["k"], ["v"], ["table"], ["q", "v"]):
        y = {n: x[n].detach().clone().requires_grad_(n in names) for n in ("q", "k", "v", "table")}
        out = softmax_attention(y["q"], y["k"], y["v"], table=y["table"], buckets=BOTH)
        for n, a in zip(names, torch.autograd.grad(out, [y[n] for n in names], x["g"])):
            if "table" in names:                    # else the probabilities are rounded once more, within the bounds
                assert torch.equal(a, want["g" + n]), n
    with torch.no_grad():
        out = softmax_attention(x["q"], x["k"], x["v"], table=x["table"], buckets=BOTH)
    assert not out.requires_grad


def test_results_do_not_change(dev):
    t = make(2, 4, 2, 300, 700, 64, BF16, bias=BOTH, keep="padded")
    a, b = run(dev, t, BOTH), run(dev, t, BOTH)
    for n in a:
        assert torch.equal(a[n], b[n]), n


# ------------------------------------------------------------------------------------------------------ the map
@pytest.mark.parametrize("bias", [BOTH, PAST, RelativeBuckets(2, 5), RelativeBuckets(256, 300), RelativeBuckets(1, 1, False)], ids=str)
@pytest.mark.parametrize("M,N,start", [(1, 1, 0), (1, 700, 699), (65, 3, 0), (100, 130, -50), (64, 1024, 10), (131, 1025, 200),
                                       (7, 2050, 1000), (0, 5, 0), (5, 0, 0)])
def test_bias_map(dev, M, N, start, bias):
    gen = torch.Generator().manual_seed(M + N)
    table = torch.randn(bias.num_buckets, 3, generator=gen)
    g = torch.randn(3, M, N, generator=gen)
    buckets = oracle.bucket_map(M, N, start, *bias)
    want = table.t()[:, buckets.flatten()].view(3, M, N)
    leaf = table.to(dev).requires_grad_(True)
    out = relative_bias(leaf, M, N, bias, start=start)
    assert torch.equal(out.detach().cpu(), want)
    got = torch.autograd.grad(out, leaf, g.to(dev))[0].cpu().double()
    hot = torch.nn.functional.one_hot(buckets.flatten(), bias.num_buckets).double()
    exact, size = (torch.matmul(x.double().view(3, -1), hot).t() for x in (g, g.abs()))
    # a diagonal's rows, the lanes of a bucket, then the workgroups: no chain of sums is longer than this
    assert ((got - exact).abs() <= (64 + 16 + N / 256 + M / 64) * oracle.U * size).all()


def test_bias_map_is_the_attentions_bias(dev):
    t = make(2, 3, 3, 90, 120, 32, F32, bias=BOTH)
    x = {n: a.to(dev) for n, a in t.items() if a is not None}
    fused = softmax_attention(x["q"], x["k"], x["v"], table=x["table"], buckets=BOTH, start=7)
    bias = relative_bias(x["table"], 90, 120, BOTH, start=7)
    s = x["q"].double() @ x["k"].double().transpose(-1, -2) * 32 ** -0.5 + bias.double()
    want = torch.softmax(s, -1) @ x["v"].double()
    bound = reference(t, BOTH, start=7)["bound"]["out"]
    assert ((fused.double() - want).abs().cpu() <= bound + TINY).all()
