"""Softmax attention as it is used: a decoder layer trained on an encoder's states and then run token by token, under graph
capture, on several streams, with keys past 2^31 elements, and gradients that take only part of the inputs."""

import pytest
import torch

from oracle import softmax as oracle
from qlka import modules
from qlka.softmax import RelativeBuckets, relative_bias, softmax_attention

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


class Layer(torch.nn.Module):
    """An encoder's self attention with a position bias, a decoder's causal one, and attention from one to the other."""

    def __init__(self, E=96, H=3):
        super().__init__()
        bias = lambda both: modules.RelativePositionBias(H, bidirectional=both)  # noqa: E731
        self.enc = modules.KernelMultiheadAttention(E, H, position_bias=bias(True))
        self.dec = modules.KernelMultiheadAttention(E, H, position_bias=bias(False))
        self.cross = modules.KernelMultiheadAttention(E, H)

    def encode(self, x, keep):
        return x + self.enc(x, keep)

    def forward(self, x, keep, y):
        states = self.encode(x, keep)
        y = y + self.dec(y, causal=True)
        return y + self.cross(y, keep, states)


def plain_layer(layer, x, keep, y):
    """The same in the layer's parameters' type, by elementary operations."""
    def attend(mod, q_in, kv_in, keep, causal):
        E, H = mod.out_proj.in_features, mod.num_heads
        w, b = mod.in_proj_weight, mod.in_proj_bias
        q, k, v = (torch.nn.functional.linear(z, w[i * E:(i + 1) * E], b[i * E:(i + 1) * E]).unflatten(-1, (H, -1)).transpose(1, 2)
                   for i, z in enumerate((q_in, kv_in, kv_in)))
        s = torch.matmul(q, k.transpose(-1, -2).contiguous()) * mod.tau ** -2
        if mod.position_bias is not None:
            at = oracle.bucket_map(q.shape[2], k.shape[2], 0, *mod.position_bias.buckets).to(q.device)
            s = s + mod.position_bias.weight[at].permute(2, 0, 1)
        see = oracle.visible(q.shape[0], q.shape[2], k.shape[2], None if keep is None else keep.cpu(), causal).to(q.device)
        p = torch.softmax(s.masked_fill(~see[:, None], float("-inf")), -1)
        return mod.out_proj(torch.matmul(p, v).transpose(1, 2).flatten(2))

    states = x + attend(layer.enc, x, x, keep, False)
    y = y + attend(layer.dec, y, y, None, True)
    return y + attend(layer.cross, y, states, keep, False)


def make_layer(dev):
    torch.manual_seed(0)
    layer = Layer()
    for m in layer.modules():
        if isinstance(m, modules.RelativePositionBias):
            torch.nn.init.normal_(m.weight)
    x, y = torch.randn(2, 150, 96), torch.randn(2, 70, 96)
    keep = torch.arange(150)[None, :] < torch.tensor([[150], [83]])
    return layer.to(dev), x.to(dev), keep.to(dev), y.to(dev)


def test_layer_and_its_gradients(dev):
    layer, x, keep, y = make_layer(dev)
    g = torch.randn(2, 70, 96, device=dev)
    params = list(layer.parameters())
    out = layer(x, keep, y)
    got = torch.autograd.grad(out, params, g)
    exact = Layer().to(dev).double()
    exact.load_state_dict(layer.state_dict())
    want_out = plain_layer(exact, x.double(), keep, y.double())
    want = torch.autograd.grad(want_out, list(exact.parameters()), g.double())
    # fp32 throughout: sums of up to 2 * 150 * 96 terms, whose roundings add up at random: a few hundred steps of 2^-24
    assert (out.double() - want_out).norm() <= 2e-5 * want_out.norm()
    for (n, _), a, b in zip(layer.named_parameters(), got, want):
        assert (a.double() - b).norm() <= 2e-5 * b.norm() + 1e-6, n      # the keys' bias has no gradient but rounding


def test_tokens_one_by_one(dev):
    layer, x, keep, y = make_layer(dev)
    with torch.no_grad():
        whole = layer(x, keep, y)
        states = layer.cross.project_context(layer.encode(x, keep))
        k, v = layer.dec.project_context(y)
        for i in (0, 1, 30, 69):
            t = y[:, i:i + 1]
            t = t + layer.dec(t, context=(k[:, :, :i + 1], v[:, :, :i + 1]), causal=True, start=i)
            t = t + layer.cross(t, keep, states)
            # two layers of sums over up to 150 keys and 96 features in fp32 by other kernels
            assert (t - whole[:, i:i + 1]).norm() <= 1e-5 * whole[:, i:i + 1].norm(), i


def leaves(dev, B, H, G, M, N, D, dtype, bias=None, seed=0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=gen).to(dtype).to(dev)  # noqa: E731
    table = torch.randn(bias.num_buckets, H, generator=gen).to(dev) if bias else None
    return {"q": r(B, H, M, D), "k": r(B, G, N, D), "v": r(B, G, N, D), "g": r(B, H, M, D), "table": table}


CAPTURED = [("step", (2, 4, 2, 1, 3000, 64), BF16, False), ("split", (1, 2, 2, 50, 4000, 64), F32, False),
            ("rows", (3, 4, 4, 200, 300, 64), BF16, False), ("train", (2, 4, 2, 150, 200, 64), BF16, True),
            ("train_fp32", (2, 4, 2, 65, 65, 32), F32, True), ("train_split", (1, 2, 1, 1500, 64, 64), BF16, True)]


@pytest.mark.parametrize("name,shape,dtype,train", CAPTURED, ids=[c[0] for c in CAPTURED])
def test_graph_replays_equal_eager(dev, name, shape, dtype, train):
    bias = RelativeBuckets(bidirectional=False)
    x = leaves(dev, *shape, dtype, bias)
    keep = torch.rand(shape[0], shape[4], device=dev) < 0.8
    names = ("q", "k", "v", "table")

    def call(y):
        kw = dict(keep=keep, table=y["table"], buckets=bias, causal=True, start=shape[4] - shape[3])
        if not train:
            return (softmax_attention(y["q"], y["k"], y["v"], **kw),)
        out = softmax_attention(y["q"], y["k"], y["v"], **kw)
        return (out.detach(),) + torch.autograd.grad(out, [y[n] for n in names], y["g"])

    def fresh():                                     # leaves of their own: no eager graph of the captured ones is alive
        return {n: a.clone().requires_grad_(train and n in names) for n, a in x.items()}

    eager = [t.clone() for t in call(fresh())]
    held = fresh()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            call(fresh())
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = call(held)
    for i in range(3):
        for t in outs:
            t.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(eager, outs):
            assert torch.equal(a, b), (name, i)
        call(fresh())                                # eager work between the replays
    # new values in the same places
    other = leaves(dev, *shape, dtype, bias, seed=5)
    with torch.no_grad():
        for n in held:
            held[n].copy_(other[n])
    graph.replay()
    torch.cuda.synchronize()
    want = call({n: a.clone().requires_grad_(train and n in names) for n, a in other.items()})
    for a, b in zip(want, outs):
        assert torch.equal(a, b)


def test_two_graphs_and_two_streams_keep_apart(dev):
    """Splits of two calls that overlap have workspaces of their own."""
    xs = [leaves(dev, 1, 4, 2, M, 5000, 64, BF16, seed=s) for s, M in ((1, 1), (2, 40))]
    want = [softmax_attention(x["q"], x["k"], x["v"]) for x in xs]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x in xs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(softmax_attention(x["q"], x["k"], x["v"]))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in xs]
    for _ in range(20):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(want, outs):
        assert torch.equal(a, b)
    eager = []
    for _ in range(10):
        for s, x in zip(streams, xs):
            with torch.cuda.stream(s):
                eager.append(softmax_attention(x["q"], x["k"], x["v"]))
    torch.cuda.synchronize()
    for i, a in enumerate(eager):
        assert torch.equal(a, want[i % 2])


@pytest.mark.parametrize("M", [1, 40])
def test_offsets_past_32_bits(dev, M):
    """A cache of 3 x 2^30 elements of which two far apart rows' worth is attended to."""
    B, N, D = 3, 1 << 24, 64                          # bf16: 6 GiB for k; v is a broadcast row
    k = torch.zeros(B, 1, N, D, dtype=BF16, device=dev)
    v = torch.randn(1, 1, 1, D, device=dev).to(BF16)
    vv = torch.zeros(B, 1, N, D, dtype=BF16, device=dev)
    keep = torch.zeros(B, N, dtype=torch.bool, device=dev)
    at = torch.tensor([5, 1 << 20, N - 2], device=dev)
    keep[:, at] = True
    vv[:, 0, at] = torch.arange(1, 4, device=dev).to(BF16)[None, :, None] * v[0, 0]
    q = torch.randn(B, 1, M, D, device=dev).to(BF16)
    out = softmax_attention(q, k, vv, keep=keep)
    want = (2 * v).float().expand(B, 1, M, D)         # equal scores: the mean of 1, 2, 3 times v
    assert ((out.float() - want).abs() <= 3 * 2 ** -8 * want.abs()).all()


def test_second_derivative_is_refused(dev):
    x = leaves(dev, 1, 2, 2, 10, 12, 32, F32)
    q = x["q"].requires_grad_(True)
    out = softmax_attention(q, x["k"], x["v"])
    with pytest.raises(RuntimeError, match="no second derivative"):
        torch.autograd.grad(out, q, x["g"], create_graph=True)
    table = torch.zeros(32, 2, device=dev, requires_grad=True)
    out = relative_bias(table, 3, 4)
    with pytest.raises(RuntimeError, match="no second derivative"):
        torch.autograd.grad(out.sum(), table, create_graph=True)


def test_refusals(dev):
    x = leaves(dev, 2, 4, 2, 5, 6, 32, F32)
    q, k, v = x["q"], x["k"], x["v"]
    for bad, message in (((q.double(), k.double(), v.double()), "float32 or bfloat16"), ((q, k.to(BF16), v), "same dtype"),
                         ((q[0], k, v), "4D"), ((q, k, v[:, :, :5]), "same shape"), ((q[:1], k, v), "batch size"),
                         ((q[..., :16], k, v), "same head dimension"), ((q[:, :3], k, v), "multiple of"),
                         ((q.repeat(1, 1, 1, 5), k.repeat(1, 1, 1, 5), v.repeat(1, 1, 1, 5)), "head dimension must be")):
        with pytest.raises(RuntimeError, match=message):
            softmax_attention(*bad)
    for kw, message in ((dict(keep=torch.ones(2, 5, dtype=torch.bool, device=dev)), "keep must be"),
                        (dict(keep=torch.ones(2, 6, dtype=torch.bool)), "keep must be on"),
                        (dict(table=torch.zeros(32, 3, device=dev)), "table must be"), (dict(start=1 << 29), "start"),
                        (dict(table=torch.zeros(32, 4)), "table must be on")):
        with pytest.raises(RuntimeError, match=message):
            softmax_attention(q, k, v, **kw)


def test_saved_inputs_are_guarded(dev):
    x = leaves(dev, 1, 2, 2, 10, 12, 32, F32)
    q = x["q"].requires_grad_(True)
    k = x["k"].clone()
    out = softmax_attention(q, k, x["v"])
    k.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def test_bfloat16_table_and_numeric_mask(dev):
    bias = RelativeBuckets()
    x = leaves(dev, 2, 2, 2, 30, 40, 32, BF16, bias)
    keep = torch.rand(2, 40, device=dev) < 0.5
    a = softmax_attention(x["q"], x["k"], x["v"], keep=keep, table=x["table"].to(BF16), buckets=bias)
    b = softmax_attention(x["q"], x["k"], x["v"], keep=keep.float(), table=x["table"].to(BF16).float(), buckets=bias)
    assert torch.equal(a, b)
    table = x["table"].to(BF16).requires_grad_(True)
    out = softmax_attention(x["q"], x["k"], x["v"], keep=keep, table=table, buckets=bias)
    assert torch.autograd.grad(out, table, x["g"])[0].dtype == BF16


def test_forward_mode_is_refused(dev):
    import torch.autograd.forward_ad as fwAD
    x = leaves(dev, 1, 2, 2, 10, 12, 32, F32, RelativeBuckets())
    for wants in (False, True):                       # whether another input wants a gradient
        k = x["k"].clone().requires_grad_(wants)
        with fwAD.dual_level():
            q = fwAD.make_dual(x["q"], torch.ones_like(x["q"]))
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                softmax_attention(q, k, x["v"])
            table = fwAD.make_dual(x["table"], torch.ones_like(x["table"]))
            with pytest.raises(RuntimeError, match="jvp"):
                relative_bias(table, 3, 4)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("M", [1, 2, 5, 40, 200])
@pytest.mark.parametrize("start", [-300, -3, 0, 37, 250])
@pytest.mark.parametrize("bias", [None, RelativeBuckets(bidirectional=False)], ids=["plain", "bias"])
def test_a_cache_longer_than_its_tokens(dev, bias, start, M, dtype):
    """Rows of a cache that no token has reached may hold anything: the same result as without them, and zeros as their
    gradients."""
    N, cache = max(0, M + start), 600
    x = leaves(dev, 2, 4, 2, M, cache, 64, dtype, bias, seed=M)
    dirty = {n: x[n].clone() for n in "kv"}
    dirty["k"][:, :, N:], dirty["v"][:, :, N:] = float("nan"), float("inf")

    def call(k, v):
        y = {"q": x["q"].clone(), "k": k.clone(), "v": v.clone()}
        if bias:
            y["table"] = x["table"].clone()
        for a in y.values():
            a.requires_grad_(True)
        out = softmax_attention(y["q"], y["k"], y["v"], table=y.get("table"), buckets=bias, causal=True, start=start)
        with torch.no_grad():
            assert torch.equal(softmax_attention(y["q"], y["k"], y["v"], causal=True, start=start), out) or bias
        return (out.detach(),) + torch.autograd.grad(out, list(y.values()), x["g"])

    want = call(x["k"][:, :, :N], x["v"][:, :, :N])
    got = call(dirty["k"], dirty["v"])
    for i, (a, b) in enumerate(zip(got, want)):
        if i in (2, 3):                               # keys and values
            assert (a[:, :, N:] == 0).all(), i
            a = a[:, :, :N]
        assert torch.isfinite(a).all(), i
        # the axes may be split otherwise: sums of up to 250 terms of one size, and each result's rounding
        h = torch.finfo(dtype).eps if a.dtype == BF16 else 2 ** -17
        assert (a.double() - b.double()).abs().max() <= 2 * h * b.double().abs().max() if b.numel() else True, i
