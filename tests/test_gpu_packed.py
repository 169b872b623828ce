"""Attention within packed sequences (qlka.packed) on the GPU against the float64 oracle, forward and gradients, within the
bounds that oracle/softmax.py derives; lengths from none to several tiles, rows outside, strides, shared heads, what one
sequence may hold without another one's noticing, graph replays with other offsets."""

import math

import pytest
import torch

from oracle import packed as oracle
from qlka.packed import packed_attention

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
TINY = 1e-30
TYPES = pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])


def offsets_of(lengths, before=0):
    at = [before]
    for n in lengths:
        at.append(at[-1] + n)
    return at


def make(H, G, T, D, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    rand = lambda n: torch.randn(n, T, D, generator=gen)  # noqa: E731
    return {"q": (rand(H) * 1.5).to(dtype), "k": rand(G).to(dtype), "v": rand(G).to(dtype), "g": rand(H).to(dtype)}


def reference(t, at, causal, scale=None):
    return oracle.attention(t["q"], t["k"], t["v"], at, t["q"].shape[2] ** -0.5 if scale is None else scale, causal, t["g"])


def run(dev, t, at, train=True, **kw):
    x = {n: a.to(dev) for n, a in t.items()}
    leaves = [x[n].requires_grad_(train) for n in ("q", "k", "v")]
    out = packed_attention(*leaves, torch.tensor(at, dtype=torch.int32, device=dev), **kw)
    r = {"out": out.detach()}
    if train:
        r.update(zip(("gq", "gk", "gv"), torch.autograd.grad(out, leaves, x["g"])))
    return r


def check(got, want):
    for n in got:
        off = (got[n].double().cpu() - want[n]).abs()
        over = off / (want["bound"][n] + TINY)
        assert torch.isfinite(got[n]).all(), n
        assert off.numel() == 0 or over.max() <= 1, f"{n}: {over.max():.3g} times its bound ({off.max():.3g})"


LENGTHS = {
    "one": [1], "none": [0], "empty_between": [3, 0, 0, 5, 0], "tiles": [64, 32, 128, 31, 33, 1],
    "ragged": [200, 1, 77, 300, 2], "long": [515], "short": [7] * 40 + [1, 0, 30],
}


@TYPES
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "whole"])
@pytest.mark.parametrize("heads", [(1, 1, 8), (2, 2, 32), (4, 2, 64), (3, 1, 17), (2, 1, 80), (2, 2, 128)],
                         ids=lambda h: "x".join(map(str, h)))
@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
def test_matches_the_oracle(dev, lengths, heads, causal, dtype):
    H, G, D = heads
    at = offsets_of(LENGTHS[lengths])
    t = make(H, G, at[-1], D, dtype, seed=at[-1] + D)
    check(run(dev, t, at, causal=causal), reference(t, at, causal))


@TYPES
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "whole"])
@pytest.mark.parametrize("lengths,before,behind", [([40, 90], 33, 130), ([5], 1, 1), ([0], 70, 0), ([0], 0, 5), ([], 64, 65)])
def test_rows_outside_every_sequence(dev, lengths, before, behind, causal, dtype):
    at = offsets_of(lengths, before)
    T = at[-1] + behind
    t = make(4, 2, T, 64, dtype, seed=T)
    want = reference(t, at, causal)
    for n in ("q", "k", "v", "g"):                # nothing there is used
        t[n][:, :at[0]] = float("nan")
        t[n][:, at[-1]:] = float("inf")
    got = run(dev, t, at, causal=causal)
    check(got, want)
    for n in got:
        assert (got[n][:, :at[0]] == 0).all() and (got[n][:, at[-1]:] == 0).all(), n


@TYPES
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "whole"])
@pytest.mark.parametrize("lengths", [[100, 30, 70], [9, 20, 8, 20]])
def test_a_sequence_does_not_change_another(dev, lengths, causal, dtype):
    at = offsets_of(lengths)
    t = make(2, 1, at[-1], 64, dtype, seed=3)
    clean = run(dev, t, at, causal=causal)
    bad = slice(at[1], at[2])
    t["k"][:, bad] = float("nan")
    t["v"][:, bad] = float("inf")
    t["g"][:, bad] = float("nan")
    dirty = run(dev, t, at, causal=causal)
    for n in clean:
        for part in (slice(0, at[1]), slice(at[2], at[-1])):
            assert torch.equal(clean[n][:, part], dirty[n][:, part]), n


@TYPES
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "whole"])
@pytest.mark.parametrize("longest", [30, 60])
@pytest.mark.parametrize("D", [32, 40, 64, 128])
def test_many_short_sequences(dev, D, longest, causal, dtype):
    """Enough of them for workgroups of one wave and of two."""
    gen = torch.Generator().manual_seed(longest + D)
    at = offsets_of([longest, 0] + torch.randint(1, longest + 1, (68,), generator=gen).tolist(), 1)
    t = make(8, 4, at[-1] + 2, D, dtype, seed=D)
    check(run(dev, t, at, causal=causal), reference(t, at, causal))


@TYPES
@pytest.mark.parametrize("D", [32, 48, 64, 128])
def test_many_short_sequences_of_whole_heads(dev, D, dtype):
    gen = torch.Generator().manual_seed(D)
    at = offsets_of([60, 0] + torch.randint(20, 61, (68,), generator=gen).tolist())
    t = make(8, 8, at[-1], D, dtype, seed=D + 1)
    check(run(dev, t, at, causal=True), reference(t, at, True))


@TYPES
@pytest.mark.parametrize("count", [61, 62, 63, 64, 65, 130, 253, 254, 255, 5000])
def test_many_sequences(dev, count, dtype):
    """More than a wave, and than a wave's square, looks at together."""
    gen = torch.Generator().manual_seed(count)
    lengths = torch.randint(0, 4 if count > 100 else 60, (count,), generator=gen).tolist()
    at = offsets_of(lengths)
    t = make(2, 1, at[-1], 32, dtype, seed=count)
    check(run(dev, t, at), reference(t, at, True))


@TYPES
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "whole"])
@pytest.mark.parametrize("lengths", [[3000], [2500, 10], [700, 900, 800]])
def test_split_axes(dev, lengths, causal, dtype):
    """Few heads and long sequences: partial sums joined afterwards."""
    at = offsets_of(lengths)
    t = make(1, 1, at[-1], 64, dtype, seed=5)
    check(run(dev, t, at, causal=causal), reference(t, at, causal))


@TYPES
@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0 ** -90, 1e6])
def test_scales(dev, scale, dtype):
    at = offsets_of([90, 41])
    t = make(2, 1, at[-1], 64, dtype, seed=9)
    if scale == 1e6:                              # one key far ahead in each row: the softmax picks it
        t["k"] = torch.sign(t["k"])
        t["q"] = torch.sign(t["q"])
    got = run(dev, t, at, train=scale != 1e6, scale=scale)
    if scale != 1e6:
        return check(got, reference(t, at, True, scale))
    want = oracle.attention(t["q"], t["k"], t["v"], at, scale, True)["out"]
    # scores are whole numbers of products times the scale, so equal ones stay equal: rounded once, and the shares of ties
    assert ((got["out"].double().cpu() - want).abs() <= 2.0 ** -8 * (want.abs() + t["v"].double().abs().amax())).all()


@TYPES
def test_strides_and_views(dev, dtype):
    at = torch.tensor([0, 50, 113, 113, 200], dtype=torch.int32, device=dev)
    t = make(4, 2, 200, 64, dtype, seed=2)
    want = reference(t, at.tolist(), True)
    x = {n: a.to(dev) for n, a in t.items()}
    by_rows = {n: a.transpose(0, 1).contiguous().transpose(0, 1) for n, a in x.items()}                 # (T, n, D)
    both = torch.cat([x["k"].transpose(0, 1), x["v"].transpose(0, 1)], 2)                               # one projection
    parts = {"k": both[..., :64].transpose(0, 1), "v": both[..., 64:].transpose(0, 1)}
    off = {n: torch.cat([torch.zeros_like(a[..., :1]), a], 2)[..., 1:] for n, a in x.items()}           # rows off 16 bytes
    for y in (by_rows, {**x, **parts}, off):
        leaves = [y[n].detach().requires_grad_(True) for n in "qkv"]
        out = packed_attention(*leaves, at)
        grads = torch.autograd.grad(out, leaves, y["g"])
        check(dict(zip(("out", "gq", "gk", "gv"), (out.detach(),) + grads)), want)
    shared = x["k"][:1].expand(2, -1, -1)                                                               # a stride of 0
    t["k"] = t["k"][:1].repeat(2, 1, 1)
    out = packed_attention(x["q"], shared, x["v"], at)
    check({"out": out}, reference(t, at.tolist(), True))


@TYPES
def test_parts_of_the_gradient(dev, dtype):
    at = torch.tensor([0, 70, 150], dtype=torch.int32, device=dev)
    x = {n: a.to(dev) for n, a in make(2, 2, 150, 64, dtype, seed=4).items()}
    full = [x[n].clone().requires_grad_(True) for n in "qkv"]
    want = torch.autograd.grad(packed_attention(*full, at), full, x["g"])
    for one in range(3):
        leaves = [x[n].clone().requires_grad_(i == one) for i, n in enumerate("qkv")]
        got, = torch.autograd.grad(packed_attention(*leaves, at), [leaves[one]], x["g"])
        same = torch.equal(got, want[one])
        assert same or one == 2 and dtype == BF16 and torch.allclose(got.float(), want[2].float(), rtol=2 ** -7)


def test_gradient_against_differences(dev):
    """fp32: the slope along a direction from two sides, h = 2^-6: h^2 of the third derivative, and roundings of 2^-20 / h."""
    at = torch.tensor([0, 20, 47], dtype=torch.int32, device=dev)
    t = make(2, 1, 47, 32, F32, seed=11)
    x = {n: a.to(dev) for n, a in t.items()}
    leaves = [x[n].requires_grad_(True) for n in "qkv"]
    grads = torch.autograd.grad(packed_attention(*leaves, at), leaves, x["g"])
    gen = torch.Generator().manual_seed(1)
    for i in range(3):
        step = torch.randn(leaves[i].shape, generator=gen).to(dev)
        step = step / step.norm()
        side = []
        for h in (2.0 ** -6, -2.0 ** -6):
            moved = [a.detach() + (h * step if j == i else 0) for j, a in enumerate(leaves)]
            side.append((packed_attention(*moved, at).double() * x["g"].double()).sum())
        slope = ((side[0] - side[1]) / 2.0 ** -5).item()
        want = (grads[i].double() * step.double()).sum().item()
        size = (grads[i].double() * step.double()).abs().sum().item()
        assert abs(slope - want) <= 2e-3 * (size + 1)


def test_runs_are_equal_and_second_derivatives_are_refused(dev):
    at = offsets_of([300, 5, 200])
    t = make(3, 3, at[-1], 64, BF16, seed=8)
    a, b = run(dev, t, at), run(dev, t, at)
    for n in a:
        assert torch.equal(a[n], b[n]), n
    x = {n: y.to(dev) for n, y in t.items()}
    q = x["q"].requires_grad_(True)
    out = packed_attention(q, x["k"], x["v"], torch.tensor(at, dtype=torch.int32, device=dev))
    with pytest.raises(RuntimeError, match="no second derivative"):
        torch.autograd.grad(out, [q], x["g"], create_graph=True)


@TYPES
def test_replays_with_other_offsets(dev, dtype):
    t = make(4, 2, 260, 64, dtype, seed=6)
    x = {n: a.to(dev) for n, a in t.items()}
    at = torch.tensor([0, 100, 180, 260], dtype=torch.int32, device=dev)
    leaves = [x[n].requires_grad_(True) for n in "qkv"]

    def step():
        out = packed_attention(*leaves, at)
        return (out.detach(),) + torch.autograd.grad(out, leaves, x["g"])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for new in ([0, 100, 180, 260], [0, 1, 259, 260], [10, 10, 200, 240], [0, 260, 260, 260]):
        at.copy_(torch.tensor(new, dtype=torch.int32))
        for y in held:
            y.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        eager = step()
        for y, z in zip(held, eager):
            assert torch.equal(y, z), new
        check(dict(zip(("out", "gq", "gk", "gv"), held)), reference(t, new, True))


def test_other_streams(dev):
    at = torch.tensor([0, 90, 400], dtype=torch.int32, device=dev)
    x = {n: a.to(dev) for n, a in make(4, 4, 400, 64, BF16, seed=1).items()}
    want = packed_attention(x["q"], x["k"], x["v"], at)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for s in streams:
        with torch.cuda.stream(s):
            outs.append(packed_attention(x["q"], x["k"], x["v"], at))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


@TYPES
def test_far_rows(dev, dtype):
    """Rows past 2^31 elements from the tensor's start."""
    T, wide = 40, (1 << 31) // 32 + 64
    t = make(2, 1, T, 64, dtype, seed=13)
    at = [0, 15, 40]
    big = torch.empty(T * wide, dtype=dtype, device=dev)
    far = {n: torch.as_strided(big, (t[n].shape[0], T, 64), (64, wide, 1), 256 * i) for i, n in enumerate("qkv")}
    for n in far:
        far[n].copy_(t[n])
    out = packed_attention(far["q"], far["k"], far["v"], torch.tensor(at, dtype=torch.int32, device=dev))
    check({"out": out}, reference(t, at, True))


@pytest.mark.parametrize("lengths", [[14, 25, 29], [2524]], ids=["short", "split"])
def test_gradients_divide_by_the_sum_of_whole_exponentials(dev, lengths):
    """bf16, one key in 29 of score 0 and others whose exponentials all lie just below the middle between 1/2 and the next
    bf16 number, so that rounding takes nearly 2^-8 of a row's sum; lengths at which P and the gradient of v round the same
    way as that would. A row's P is off by its own rounding alone, not by the sum's too."""
    at = offsets_of(lengths)
    score = torch.tensor(-math.log(2) + 2.0 ** -8 * 0.99, dtype=torch.float64)
    gen = torch.Generator().manual_seed(0)
    t = {n: torch.zeros(1, at[-1], 64, dtype=BF16) for n in "qk"}
    t["q"][..., :2] = 1
    t["k"][..., 0] = score.to(BF16)
    t["k"][..., 1] = (score - score.to(BF16).double()).to(BF16)
    for lo, hi in zip(at, at[1:]):
        t["k"][:, lo:hi:29] = 0
    t["v"] = torch.randn(1, at[-1], 64, generator=gen).to(BF16)
    t["g"] = torch.randn(1, 1, 64, generator=gen).to(BF16).expand(1, at[-1], 64).contiguous()
    check(run(dev, t, at, causal=False, scale=1.0), reference(t, at, False, 1.0))


@TYPES
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "whole"])
@pytest.mark.parametrize("count", [200, 300])
def test_one_long_sequence_among_short_ones(dev, count, causal, dtype):
    """Workgroups of few waves, which the average length asks for, go through a sequence of many tiles; in the order of work,
    and by number."""
    lengths = [10, 0] * (count // 4) + [1300] + [9] * (count // 2)
    at = offsets_of(lengths, 2)
    t = make(4, 2, at[-1] + 3, 64, dtype, seed=count)
    check(run(dev, t, at, causal=causal), reference(t, at, causal))
