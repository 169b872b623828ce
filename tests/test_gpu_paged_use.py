"""Packed sequences and the cache in pages as they are used: a layer of a decoder trained on packed documents, then run on prompts,
chunks and tokens over a cache, against the same layer on whole sequences; heads read back for attention with a position
bias; a captured decoding step."""

import pytest
import torch

from qlka import modules
from qlka.packed import packed_attention
from qlka.paged import PagedCache, paged_attention
from qlka.softmax import RelativeBuckets, softmax_attention

pytestmark = pytest.mark.gpu

F32, BF16, I8, E4 = torch.float32, torch.bfloat16, torch.int8, torch.float8_e4m3fn
E, H = 96, 3


def i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def sums(lengths):
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return at


def make_layer(dev, dtype=F32):
    torch.manual_seed(0)
    layer = modules.KernelMultiheadAttention(E, H, tau=32 ** 0.25)
    torch.nn.init.normal_(layer.in_proj_bias, std=0.3)
    return layer.to(dev).to(dtype)


def plain(layer, x, causal=True):
    """The layer on one sequence (S, E) in its parameters' type, by elementary operations."""
    q, k, v = (t[0] for t in layer.split_heads(x[None]))
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()) * layer.tau ** -2
    if causal:
        s = s.masked_fill(torch.ones_like(s, dtype=torch.bool).triu(1), float("-inf"))
    return layer.out_proj(torch.matmul(torch.softmax(s, -1), v).transpose(0, 1).flatten(1))


@pytest.mark.parametrize("causal", [True, False], ids=["causal", "whole"])
def test_training_on_packed_documents(dev, causal):
    layer, lengths = make_layer(dev), [90, 1, 40, 130]
    at = sums(lengths)
    x, g = torch.randn(at[-1], E, device=dev), torch.randn(at[-1], E, device=dev)
    params = list(layer.parameters())
    out = layer(x, offsets=i32(at, dev), causal=causal)
    got = torch.autograd.grad(out, params, g)
    exact = make_layer(dev).double()
    want_out = torch.cat([plain(exact, x[a:b].double(), causal) for a, b in zip(at, at[1:])])
    want = torch.autograd.grad(want_out, list(exact.parameters()), g.double())
    # fp32 throughout: sums of up to 261 * 96 terms, whose roundings add up at random: a few hundred steps of 2^-24
    assert (out.double() - want_out).norm() <= 2e-5 * want_out.norm()
    for (n, _), a, b in zip(layer.named_parameters(), got, want):
        assert (a.double() - b).norm() <= 2e-5 * b.norm() + 1e-6, n     # the keys' bias has no gradient but rounding


@pytest.mark.parametrize("dtype,held,bound", [(F32, F32, 2e-5), (BF16, BF16, 2e-2), (F32, I8, 2e-2), (F32, E4, 8e-2)],
                         ids=["fp32", "bf16", "fp32_int8", "fp32_e4m3"])
def test_prompts_chunks_and_tokens(dev, dtype, held, bound):
    """A batch of sequences goes through a cache as a server has it: prompts, then more of one prompt beside tokens of others,
    a sequence that ends and one that takes its pages, tokens. Bounds: bf16 roundings of states, weights and results add up
    to a few 2^-8 of the norm; int8 rounds each element by at most 2^-8 of its block's largest, e4m3 by 2^-4 of itself,
    which keys pass on to the scores and values to the result."""
    layer, page_size = make_layer(dev, dtype), 16
    cache = PagedCache.new(40, page_size, H, E // H, held)
    total = [100, 70, 46, 60]
    x = [torch.randn(n, E, device=dev).to(dtype) for n in total]
    exact = make_layer(dev, dtype).double()
    want = [plain(exact, y.double()) for y in x]
    free = torch.randperm(40).tolist()
    tables = torch.full((3, 8), -1, dtype=torch.int32)
    have, who = [0, 0, 0], [0, 1, 2]                     # tokens in each place of the batch, and whose they are
    got = [[] for _ in total]

    def step(new):
        for b, n in enumerate(new):
            have[b] += n
            for i in range(-(-have[b] // page_size)):
                if tables[b, i] < 0:
                    tables[b, i] = free.pop()
        rows = torch.cat([x[who[b]][have[b] - n:have[b]] for b, n in enumerate(new)])
        at = sums(new)
        with torch.no_grad():
            given = None if new == [1] * 3 else i32(at, dev)
            out = layer(rows, cache=(cache, tables.to(dev), i32(have, dev)), offsets=given)
        for b, n in enumerate(new):
            got[who[b]].append(out[at[b]:at[b + 1]])

    step([40, 69, 1])
    step([30, 0, 44])                                    # more of the first prompt, most of the third
    step([1, 1, 0])
    free.extend(tables[1][tables[1] >= 0].tolist())      # the second ended: a fourth takes its place, and its pages
    tables[1], have[1], who[1] = -1, 0, 3
    step([1, 58, 0])
    step([1, 1, 1])
    step([27, 1, 0])
    for y, z in zip(got, want):
        y = torch.cat(y).double()
        assert y.shape == z.shape
        assert (y - z).norm() <= bound * z.norm()


@pytest.mark.parametrize("held", [BF16, I8, E4], ids=["bf16", "int8", "e4m3"])
def test_packed_prompt_then_pages_agree(dev, held):
    """The last row of a prompt from packed attention over its own rows, and as a token over the pages that hold them: equal to
    the rounding of what 8 bits hold (bf16: of P and the result)."""
    gen = torch.Generator().manual_seed(3)
    lengths, G, D = [300, 77, 64], 2, 64
    at = sums(lengths)
    q, k, v = (torch.randn(n, at[-1], D, generator=gen).to(BF16).to(dev) for n in (4, G, G))
    cache = PagedCache.new(32, 16, G, D, held)
    tables = torch.full((3, 19), -1, dtype=torch.int32)
    order = torch.randperm(32, generator=gen).tolist()
    for b, n in enumerate(lengths):
        for i in range(-(-n // 16)):
            tables[b, i] = order.pop()
    tables, lens, offsets = tables.to(dev), i32(lengths, dev), i32(at, dev)
    cache.write(k, v, tables, lens, offsets)
    last = torch.tensor(at[1:], device=dev) - 1
    token = paged_attention(q[:, last], cache, tables, lens)
    # what is held, as rows again, is what packed attention takes
    kept = cache.read(tables, lens, 300)
    rows = [torch.cat([y[b, :, :n] for b, n in enumerate(lengths)], 1) for y in kept]
    want = packed_attention(q, *rows, offsets)[:, last]
    assert (token.float() - want.float()).norm() <= 2 ** -7 * want.float().norm()
    whole = paged_attention(q, cache, tables, lens, offsets)
    assert (whole.float() - packed_attention(q, *rows, offsets).float()).norm() <= 2 ** -7 * whole.float().norm()


@pytest.mark.parametrize("held", [F32, I8, E4], ids=["fp32", "int8", "e4m3"])
def test_heads_read_back_for_attention_with_a_bias(dev, held):
    """What qlka.paged has no kernel for, a position bias, runs on the heads that the cache gives back, as the layer's context."""
    torch.manual_seed(1)
    bias = modules.RelativePositionBias(H, bidirectional=False)
    torch.nn.init.normal_(bias.weight)
    layer = modules.KernelMultiheadAttention(E, H, tau=32 ** 0.25, position_bias=bias).to(dev)
    cache = PagedCache.new(12, 16, H, E // H, held)
    lengths = [60, 60]
    tables = torch.randperm(12)[:8].view(2, 4).int().to(dev)
    x = torch.randn(2, 60, E, device=dev)
    with torch.no_grad():
        k, v = layer.project_context(x)                                             # (B, H, N, Dh)
        pack = lambda t: t.transpose(0, 1).flatten(1, 2)  # noqa: E731
        cache.write(pack(k), pack(v), tables, i32(lengths, dev), i32([0, 60, 120], dev))
        heads = cache.read(tables, i32(lengths, dev), 60, F32)
        got = layer(x[:, 50:], context=heads, causal=True, start=50)
        q, = layer._heads(x[:, 50:], 0, 1)
        want = softmax_attention(q, *heads, scale=layer.tau ** -2, table=bias.weight,
                                 buckets=RelativeBuckets(bidirectional=False), causal=True, start=50)
        want = layer.out_proj(want.transpose(1, 2).flatten(2))
        assert torch.equal(got, want)
        whole = layer(x, causal=True)[:, 50:]
        assert (got - whole).norm() <= {F32: 1e-5, I8: 2e-2, E4: 8e-2}[held] * whole.norm()


def test_a_captured_decoding_step(dev):
    """One token for each sequence through a layer, captured once: lengths, tables and inputs change between the replays."""
    layer = make_layer(dev, BF16)
    caches = [PagedCache.new(30, 16, H, E // H, I8) for _ in range(2)]
    tables = torch.arange(24, dtype=torch.int32, device=dev).view(4, 6)
    lengths, x = i32([1, 5, 16, 17], dev), torch.randn(4, E, device=dev).to(BF16)
    with torch.no_grad():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            layer(x, cache=(caches[1], tables, lengths))
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layer(x, cache=(caches[0], tables, lengths))
        for i in range(20):
            x.copy_(torch.randn(4, E, device=dev))
            out.fill_(float("nan"))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, layer(x, cache=(caches[1], tables, lengths))), i
            lengths += 1


def test_what_the_layer_refuses(dev):
    layer = make_layer(dev)
    cache = PagedCache.new(4, 16, H, E // H, F32)
    x, at = torch.randn(5, E, device=dev), i32([0, 5], dev)
    held = (cache, i32([[0]], dev), i32([5], dev))
    with pytest.raises(RuntimeError, match="must not require"):
        layer(x, cache=held, offsets=at)
    with torch.no_grad():
        with pytest.raises(ValueError, match="no keep, context or start"):
            layer(x, offsets=at, start=3)
        with pytest.raises(ValueError, match=r"must be \(T, E\)"):
            layer(x[None], offsets=at)
        with pytest.raises(RuntimeError, match="rows must be B"):
            layer(x, cache=held)
        with pytest.raises(RuntimeError, match="offsets must be int32"):
            layer(x, offsets=at.long())
        with pytest.raises(NotImplementedError, match="without a position bias"):
            modules.KernelMultiheadAttention(E, H, position_bias=modules.RelativePositionBias(H)).to(dev)(x, offsets=at)
        with pytest.raises(NotImplementedError, match="'softmax' kernel"):
            modules.KernelMultiheadAttention(E, H, kernel="add_riesz").to(dev)(x, offsets=at)


def test_refusals(dev):
    z = lambda *s, d=BF16: torch.zeros(s, dtype=d, device=dev)  # noqa: E731
    k, e = z(4, 2, 16, 64), z(4, 2, 16, 2, d=torch.uint8)
    for args, match in [((k, z(4, 2, 16, 32)), "one dtype, shape"), ((k.half(), k.half()), "must be float32"),
                        ((k[0], k[0]), "must be 4D"), ((z(4, 2, 16, 60), z(4, 2, 16, 60)), "multiple of 8"),
                        ((k, k, e, e), "go with pages of 8 bits"), ((k.to(I8), k.to(I8)), "need exponents"),
                        ((k.to(I8), k.to(I8), e[..., :1], e), "exponents must be"), ((k.to(I8), k.to(I8), e.int(), e), "must be uint8"),
                        ((k.transpose(2, 3), k.transpose(2, 3)), "page_size|next to each other|multiple of 8"),
                        ((k.clone().requires_grad_(), k), "must not require one")]:
        with pytest.raises(RuntimeError, match=match):
            PagedCache.of(*args)

    cache = PagedCache.of(k, k.clone())
    tables, lengths, at, q = i32([[0, 1], [2, 3]], dev), i32([3, 9], dev), i32([0, 1, 2], dev), z(4, 2, 64)
    for args, match in [((q, cache, tables.long(), lengths), "must be int32"), ((q, cache, tables, lengths[:1]), "tables must be|rows must be B"),
                        ((q, cache, tables[0], lengths), "tables must be"), ((q, cache, tables, lengths, at[:2]), r"offsets must be \(B \+ 1\)"),
                        ((q[..., :32], cache, tables, lengths), "with the pages' D"), ((z(3, 2, 64), cache, tables, lengths), "multiple of those"),
                        ((q.float(), cache, tables, lengths), "tokens' dtype or 8 bits"), ((q.half(), cache, tables, lengths), "must be float32 or bfloat16"),
                        ((q.cpu(), cache, tables, lengths), "on the pages' device"), ((q, cache, tables.t(), lengths), "contiguous"),
                        ((q.detach().requires_grad_(), cache, tables, lengths), "must not require")]:
        with pytest.raises(RuntimeError, match=match):
            paged_attention(*args)
    with pytest.raises(RuntimeError, match="have the heads of the pages"):
        cache.write(q, q, tables, lengths)
    with pytest.raises(RuntimeError, match="number of positions"):
        cache.read(tables, lengths, -1)
    with pytest.raises(RuntimeError, match="tokens' dtype or 8 bits"):
        cache.read(tables, lengths, 4, F32)
    with torch.no_grad():
        version = cache.k._version
        cache.write(z(2, 2, 64), z(2, 2, 64), tables, lengths)
        assert cache.k._version > version                    # what autograd saved of the pages is known to have changed
