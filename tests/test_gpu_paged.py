"""A cache of keys and values in pages (qlka.paged) and attention over it, on the GPU: what is written and read back to the bit,
attention against the float64 oracle within its bounds, pages that do not exist, tables and offsets of every kind, views,
far pages, replays."""

import math

import pytest
import torch

from oracle import paged as oracle
from qlka.paged import PagedCache, paged_attention

pytestmark = pytest.mark.gpu

F32, BF16, I8, E4 = torch.float32, torch.bfloat16, torch.int8, torch.float8_e4m3fn
TINY = 1e-30
KINDS = pytest.mark.parametrize("dtype,held", [(F32, F32), (BF16, BF16), (F32, I8), (BF16, I8), (F32, E4), (BF16, E4)],
                                ids=["fp32", "bf16", "fp32_int8", "bf16_int8", "fp32_e4m3", "bf16_e4m3"])


def i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def as_bytes(x):
    return x if x.dtype in (F32, BF16) or x.dtype == torch.uint8 else x.view(torch.uint8)


def sums(lengths, before=0):
    at = [before]
    for n in lengths:
        at.append(at[-1] + n)
    return at


def tables_of(lengths, page_size, gen, spare=3):
    """Tables of as many pages as the lengths need, in any order, -1 behind them; and the number of pages."""
    need = [-(-n // page_size) for n in lengths]
    order = torch.randperm(sum(need) + spare, generator=gen).tolist()
    t = torch.full((len(need), max(need + [0]) + 1), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        for i in range(n):
            t[b, i] = order.pop()
    return t, sum(need) + spare


def filled(num_pages, page_size, G, D, dtype, held, gen, dev):
    """A cache whose every row holds something (random rows as the definition stores them)."""
    def one():
        x = torch.randn(num_pages, G, page_size, D, generator=gen).to(dtype)
        if held in (F32, BF16):
            return x, None
        return oracle.quantise(x, held)
    (k, ke), (v, ve) = one(), one()
    put = lambda x: None if x is None else x.to(dev)  # noqa: E731
    view = lambda x: put(x) if held in (F32, BF16) else put(x).view(held)  # noqa: E731
    return PagedCache.of(view(k), view(v), put(ke), put(ve)), (k, v, ke, ve)


def attend(dev, t, cache, tables, lengths, offsets, **kw):
    return paged_attention(t.to(dev), cache, tables.to(dev), i32(lengths, dev), None if offsets is None else i32(offsets, dev), **kw)


def close(got, want, bound):
    assert torch.isfinite(got).all()
    over = (got.double().cpu() - want).abs() / (bound + TINY)
    assert over.numel() == 0 or over.max() <= 1, f"{over.max():.3g} times its bound"


# ------------------------------------------------------------------------------------------------- write and read
def written(cpu, k, v, held, tables, lengths, offsets):
    """What the pages hold after a write, in place on the CPU copies."""
    pages, exps = cpu[:2], cpu[2:]
    for b, length in enumerate(lengths):
        n = offsets[b + 1] - offsets[b]
        for i in range(n):
            at = oracle.place(tables, b, length - n + i, pages[0].shape[2], pages[0].shape[0])
            if at is None:
                continue
            for x, p, e in zip((k, v), pages, exps):
                row = x[:, offsets[b] + i]
                if held in (F32, BF16):
                    p[at[0], :, at[1]] = row
                else:
                    code, power = oracle.quantise(row, held)
                    p[at[0], :, at[1]], e[at[0], :, at[1]] = code, power


@KINDS
@pytest.mark.parametrize("G,D,page_size", [(1, 8, 16), (2, 32, 7), (3, 40, 16), (12, 64, 32), (2, 72, 1), (2, 96, 48), (5, 128, 64)])
def test_writes_what_the_definition_says(dev, G, D, page_size, dtype, held):
    gen = torch.Generator().manual_seed(G * D + page_size)
    lengths, new = [70, 1, 33, 5, 90], [70, 1, 2, 0, 40]
    tables, num_pages = tables_of(lengths, page_size, gen)
    tables[4, 1] = num_pages                                        # pages that do not exist
    tables[0, 0] = -7
    offsets = sums(new, 3)
    T = offsets[-1] + 5
    cache, cpu = filled(num_pages, page_size, G, D, dtype, held, gen, dev)
    k, v = (torch.randn(G, T, D, generator=gen) * torch.exp2(torch.randint(-12, 12, (G, T, 1), generator=gen).float()) for _ in "kv")
    k, v = k.to(dtype), v.to(dtype)
    cache.write(k.to(dev), v.to(dev), tables.to(dev), i32(lengths, dev), i32(offsets, dev))
    written(cpu, k, v, held, tables, lengths, offsets)
    for got, want in zip(cache, cpu):
        assert (got is None) == (want is None)
        if want is not None:
            assert torch.equal(as_bytes(got).cpu(), want)
    # and back
    for out in (F32, BF16) if held in (I8, E4) else (dtype,):
        got = cache.read(tables.to(dev), i32(lengths, dev), 100, out)
        for x, pages, e in zip(got, cpu[:2], cpu[2:]):
            for b, n in enumerate(lengths):
                want, _ = oracle.rows(pages, e, held, tables, b, n)
                assert torch.equal(x[b, :, :n].cpu().double(), want) and (x[b, :, n:] == 0).all()


@pytest.mark.parametrize("held", [I8, E4], ids=["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
def test_blocks_of_every_kind(dev, dtype, held):
    """Ties, zeros of either sign, the largest and the smallest numbers, single elements, infinities and NaN."""
    gen = torch.Generator().manual_seed(1)
    blocks = [torch.zeros(32), -torch.zeros(32)]
    for top in (127.0, 448.0, 126.5, 449.0, 1.0, 3.0e38, 1e-38, 1e-40, 2.0 ** -100, 2.0 ** -94, 2.0 ** -95 * 1.99):
        x = torch.randn(32, generator=gen)
        blocks += [x / x.abs().max() * top, torch.full((32,), top), torch.arange(32) * (top / 32)]
    blocks.append(torch.cat([torch.arange(16) + 0.5, 127 - torch.arange(16).float()]))                # int8's ties
    blocks.append(torch.cat([(torch.arange(31) + 8) * 1.0 + 0.5, torch.tensor([448.0])]))             # e4m3's
    blocks.append(torch.cat([(torch.arange(31) + 0.5) * 2.0 ** -9, torch.tensor([300.0])]))           # and its smallest
    for bad in (math.inf, -math.inf, math.nan):
        x = torch.randn(32, generator=gen)
        x[7] = bad
        blocks.append(x)
    x = torch.stack(blocks).to(dtype)
    x[torch.isinf(x) & torch.isfinite(torch.stack(blocks))] = 3e38
    x = torch.cat([x, x.flip(0)], 1)[None]                           # (1, T, 64): neighbours differ
    T = x.shape[1]
    cache = PagedCache.new(T // 8 + 1, 8, 1, 64, held)
    tables, lengths, offsets = torch.arange(T // 8 + 1, dtype=torch.int32)[None].to(dev), i32([T], dev), i32([0, T], dev)
    cache.write(x.to(dev), -x.to(dev), tables, lengths, offsets)
    code, power = oracle.quantise(x, held)
    got = as_bytes(cache.k).cpu().transpose(0, 1).reshape(1, -1, 64)[:, :T]
    exps = cache.k_exp.cpu().transpose(0, 1).reshape(1, -1, 2)[:, :T]
    fine = (power != 255).repeat_interleave(32, -1)
    assert torch.equal(exps, power) and torch.equal(got[fine], code[fine])
    want = oracle.values(code, power, held)
    for out in (F32, BF16):
        k, v = cache.read(tables, lengths, T, out)
        assert torch.equal(k[0].cpu().double().nan_to_num(nan=1234.0), want.nan_to_num(nan=1234.0))
        assert torch.equal(v[0].cpu().double().nan_to_num(nan=1234.0), (-want).nan_to_num(nan=1234.0))


@KINDS
def test_tokens_at_the_edge(dev, dtype, held):
    """One token for each sequence: at position 0, at a page's first and last row, past the table, at no position."""
    gen = torch.Generator().manual_seed(0)
    tables = torch.tensor([[4, -1], [1, 2], [3, 5], [0, 7], [6, 8], [9, 1]], dtype=torch.int32)
    lengths = [1, 16, 17, 33, 0, -5]
    cache, cpu = filled(10, 16, 2, 64, dtype, held, gen, dev)
    k, v = (torch.randn(2, 6, 64, generator=gen).to(dtype) for _ in "kv")
    cache.write(k.to(dev), v.to(dev), tables.to(dev), i32(lengths, dev))
    written(cpu, k, v, held, tables, lengths, sums([1] * 6))
    for got, want in zip(cache, cpu):
        if want is not None:
            assert torch.equal(as_bytes(got).cpu(), want)
    q = torch.randn(4, 6, 64, generator=gen).to(dtype)
    want, bound = oracle.attention(q, *cpu, held, tables, lengths, sums([1] * 6), 0.125)
    got = attend(dev, q, cache, tables, lengths, None)
    close(got, want, bound)
    assert (got[:, 4:] == 0).all()
    assert cache.read(tables.to(dev), i32(lengths, dev), 0)[0].shape == (6, 2, 0, 64)


# ---------------------------------------------------------------------------------------------------- attention
BATCHES = {
    # new tokens and lengths of each sequence, rows before and behind; pages are of 16 unless said
    "tokens": ([1] * 6, [1, 2, 33, 64, 100, 300], 0, 0, 16),
    "few": ([1, 3, 0, 2, 4], [40, 3, 9, 200, 131], 2, 3, 16),
    "chunks": ([70, 130, 40], [70, 400, 41], 0, 0, 48),
    "mixed": ([1, 90, 1, 0, 1, 5, 200], [33, 500, 1, 7, 300, 5, 200], 1, 40, 7),
    "pages_of_1": ([2, 50], [40, 60], 0, 0, 1),
    "large_pages": ([1, 60, 1], [129, 70, 3], 0, 0, 100),
    "too_short": ([5, 40, 1], [3, 20, 0], 0, 0, 16),      # fewer tokens than new ones: the first are at no position
}


@KINDS
@pytest.mark.parametrize("heads", [(1, 1, 8), (4, 2, 32), (12, 4, 64), (3, 3, 64), (2, 2, 40), (8, 1, 128), (4, 4, 80)],
                         ids=lambda h: "x".join(map(str, h)))
@pytest.mark.parametrize("batch", BATCHES, ids=str)
def test_attention_matches_the_oracle(dev, batch, heads, dtype, held):
    H, G, D = heads
    new, lengths, before, behind, page_size = BATCHES[batch]
    gen = torch.Generator().manual_seed(sum(lengths) + D)
    offsets = sums(new, before)
    T = offsets[-1] + behind
    tables, num_pages = tables_of(lengths, page_size, gen)
    cache, cpu = filled(num_pages, page_size, G, D, dtype, held, gen, dev)
    q = (torch.randn(H, T, D, generator=gen) * 1.5).to(dtype)
    want, bound = oracle.attention(q, *cpu, held, tables, lengths, offsets, D ** -0.5)
    plain = all(n == 1 for n in new) and T == len(new)
    for given in [offsets] + [None] * plain:
        for longest in (0, max(new), 1):                    # a hint, also a wrong one
            got = attend(dev, q, cache, tables, lengths, given, longest=longest)
            close(got, want, bound)
            assert (got[:, :before] == 0).all() and (got[:, offsets[-1]:] == 0).all()


@KINDS
@pytest.mark.parametrize("new", [[1, 1, 1, 1], [40, 1, 300, 2], [200, 90, 150, 80]], ids=str)
def test_pages_that_do_not_exist(dev, new, dtype, held):
    gen = torch.Generator().manual_seed(5)
    lengths = [300, 100, 310, 700]
    tables, num_pages = tables_of(lengths, 32, gen)
    tables[0, 0], tables[0, 5], tables[2, 3], tables[3, 10:13] = -1, num_pages, 1 << 30, -(1 << 31)
    tables[1] = -1                                          # a sequence without any page
    offsets = sums(new)
    cache, cpu = filled(num_pages, 32, 2, 64, dtype, held, gen, dev)
    q = torch.randn(4, offsets[-1], 64, generator=gen).to(dtype)
    want, bound = oracle.attention(q, *cpu, held, tables, lengths, offsets, 0.125)
    got = attend(dev, q, cache, tables, lengths, offsets)
    close(got, want, bound)
    assert (got[:, offsets[1]:offsets[2]] == 0).all()


@KINDS
@pytest.mark.parametrize("new", [[1, 1, 1], [20, 1, 90], [200, 150, 199]], ids=str)
def test_what_is_not_seen_may_hold_anything(dev, new, dtype, held):
    """Rows past a sequence's tokens in its last page, pages of others, rows outside: NaN and infinities there."""
    gen = torch.Generator().manual_seed(6)
    lengths = [100, 45, 333]
    tables, num_pages = tables_of(lengths, 64, gen)
    offsets = sums(new, 4)
    cache, _ = filled(num_pages, 64, 2, 64, dtype, held, gen, dev)
    q = torch.randn(4, offsets[-1] + 6, 64, generator=gen).to(dtype)
    clean = attend(dev, q, cache, tables, lengths, offsets)
    used = torch.zeros(num_pages, 64, dtype=torch.bool)
    for b, n in enumerate(lengths):
        for i in range(n):
            used[oracle.place(tables, b, i, 64, num_pages)] = True
    unused = ~used[:, None, :, None].to(dev)
    if held in (F32, BF16):
        cache.k.masked_fill_(unused, math.nan)
        cache.v.masked_fill_(unused, math.inf)
    else:
        cache.k_exp.masked_fill_(unused, 255)
        cache.v_exp.masked_fill_(unused, 255)
    q[:, :4], q[:, offsets[-1]:] = math.nan, math.inf
    assert torch.equal(attend(dev, q, cache, tables, lengths, offsets), clean)


@KINDS
@pytest.mark.parametrize("new", [[1, 1], [40, 1], [64, 64]], ids=str)
def test_long_sequences_are_split(dev, new, dtype, held):
    gen = torch.Generator().manual_seed(7)
    lengths = [3000, 1333]
    tables, num_pages = tables_of(lengths, 24, gen)
    offsets = sums(new)
    cache, cpu = filled(num_pages, 24, 1, 64, dtype, held, gen, dev)
    q = torch.randn(2, offsets[-1], 64, generator=gen).to(dtype)
    want, bound = oracle.attention(q, *cpu, held, tables, lengths, offsets, 0.125)
    close(attend(dev, q, cache, tables, lengths, offsets), want, bound)


@KINDS
@pytest.mark.parametrize("case", ["65_tokens", "130_few", "200_mixed", "129_empty"])
def test_many_sequences(dev, case, dtype, held):
    """More than a wave's lanes look up at once."""
    gen = torch.Generator().manual_seed(13)
    B = int(case.split("_")[0])
    draw = lambda lo, hi: torch.randint(lo, hi + 1, (B,), generator=gen).tolist()  # noqa: E731
    new = [1] * B if "tokens" in case else draw(0, 3) if "few" in case else [0] * B
    if "mixed" in case:
        new = [[1, 0, 1, 1, 2][b % 5] for b in range(B)]
        new[3], new[70], new[199] = 60, 45, 90
    if "empty" in case:
        new[64], new[128] = 1, 40
    lengths = [n + m for n, m in zip(new, draw(0, 40))]
    lengths[B - 1], lengths[B // 2] = 1200, 900             # some in parts
    offsets = sums(new, 2)
    tables, num_pages = tables_of(lengths, 16, gen)
    cache, cpu = filled(num_pages, 16, 1, 64, dtype, held, gen, dev)
    q = torch.randn(2, offsets[-1] + 3, 64, generator=gen).to(dtype)
    want, bound = oracle.attention(q, *cpu, held, tables, lengths, offsets, 0.125)
    close(attend(dev, q, cache, tables, lengths, offsets), want, bound)
    k, v = (torch.randn(1, offsets[-1] + 3, 64, generator=gen).to(dtype) for _ in "kv")
    cache.write(k.to(dev), v.to(dev), tables.to(dev), i32(lengths, dev), i32(offsets, dev))
    written(cpu, k, v, held, tables, lengths, offsets)
    for got, want in zip(cache, cpu):
        assert want is None or torch.equal(as_bytes(got).cpu(), want)


@pytest.mark.parametrize("dtype,held", [(F32, F32), (BF16, BF16), (BF16, E4)], ids=["fp32", "bf16", "bf16_e4m3"])
@pytest.mark.parametrize("B", [255, 256, 1024, 1025, 2100])
@pytest.mark.parametrize("kind", ["tokens", "mixed", "sparse"])
def test_hundreds_of_sequences(dev, kind, B, dtype, held):
    gen = torch.Generator().manual_seed(B)
    new = [1] * B
    if kind != "tokens":
        new = torch.randint(0, 3, (B,), generator=gen).tolist() if kind == "mixed" else [0] * B
        new[0], new[B // 2], new[B - 1] = 0, 70, 40
    lengths = [n + m for n, m in zip(new, torch.randint(0, 20, (B,), generator=gen).tolist())]
    lengths[B - 1], lengths[B // 3] = 1500, 700
    offsets = sums(new, 1)
    tables, num_pages = tables_of(lengths, 16, gen)
    cache, cpu = filled(num_pages, 16, 2, 32, dtype, held, gen, dev)
    q = torch.randn(4, offsets[-1] + 2, 32, generator=gen).to(dtype)
    want, bound = oracle.attention(q, *cpu, held, tables, lengths, offsets, 0.2)
    got = attend(dev, q, cache, tables, lengths, offsets, scale=0.2)
    close(got, want, bound)
    assert (got[:, :1] == 0).all() and (got[:, offsets[-1]:] == 0).all()


@pytest.mark.parametrize("dtype,held", [(F32, F32), (BF16, BF16), (BF16, I8)], ids=["fp32", "bf16", "bf16_int8"])
@pytest.mark.parametrize("new,length,heads", [([1], 20000, (2, 1, 32)), ([3, 1], 18000, (2, 2, 128)), ([400], 10000, (12, 4, 64)),
                                              ([700], 5000, (7, 7, 32)), ([600, 1], 4000, (8, 1, 128))], ids=str)
def test_parts_beyond_what_is_joined_at_once(dev, new, length, heads, dtype, held):
    """Rows whose parts are more than the lanes that look at them, many rows and few."""
    H, G, D = heads
    gen = torch.Generator().manual_seed(length)
    lengths, offsets = [length] * len(new), sums(new)
    tables, num_pages = tables_of(lengths, 64, gen)
    cache, cpu = filled(num_pages, 64, G, D, dtype, held, gen, dev)
    q = torch.randn(H, offsets[-1], D, generator=gen).to(dtype)
    want, bound = oracle.attention(q, *cpu, held, tables, lengths, offsets, D ** -0.5)
    close(attend(dev, q, cache, tables, lengths, offsets), want, bound)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("held", [I8, E4], ids=["int8", "e4m3"])
@pytest.mark.parametrize("new", [[1, 1], [40, 50]], ids=str)
def test_blocks_that_were_not_finite(dev, new, held, dtype):
    """A block marked as such is NaN: in the keys it makes the rows that see it NaN, in the values its 32 elements of them."""
    gen = torch.Generator().manual_seed(14)
    lengths = [60, 70]
    tables, num_pages = tables_of(lengths, 16, gen)
    cache, _ = filled(num_pages, 16, 1, 64, dtype, held, gen, dev)
    q = torch.randn(2, sum(new), 64, generator=gen).to(dtype)
    clean = attend(dev, q, cache, tables, lengths, sums(new))
    cache.v_exp[int(tables[0, 0]), 0, 3, 1] = 255           # sequence 0, position 3
    as_bytes(cache.v)[int(tables[0, 0]), 0, 3] = 0          # (whatever its codes are)
    got = attend(dev, q, cache, tables, lengths, sums(new))
    assert got[:, :new[0], 32:].isnan().all() and got[:, :new[0], :32].isfinite().all() and got[:, new[0]:].isfinite().all()
    cache.v_exp[int(tables[0, 0]), 0, 3, 1] = 127
    cache.k_exp[int(tables[1, 0]), 0, 5, 0] = 255           # sequence 1, position 5
    got = attend(dev, q, cache, tables, lengths, sums(new))
    assert got[:, new[0]:].isnan().all() and not got[:, :new[0]].isnan().any()
    assert clean.isfinite().all()


@KINDS
@pytest.mark.parametrize("new", [[1, 1], [100, 90]], ids=str)
@pytest.mark.parametrize("scale", [0.0, -0.2, 1e5])
def test_scales(dev, scale, new, dtype, held):
    gen = torch.Generator().manual_seed(8)
    lengths = [120, 99]
    tables, num_pages = tables_of(lengths, 16, gen)
    offsets = sums(new)
    cache, cpu = filled(num_pages, 16, 1, 32, dtype, held, gen, dev)
    q = torch.randn(2, offsets[-1], 32, generator=gen).to(dtype)
    if scale == 1e5:                                        # one key and its copies ahead of all others: shares are equal
        for b in range(2):
            for n in range(lengths[b]):
                at = oracle.place(tables, b, n, 16, num_pages)
                for x in [cpu[0], as_bytes(cache.k)] + ([cpu[2], cache.k_exp] if cpu[2] is not None else []):
                    x[at[0], :, at[1]] = x[int(tables[0, 0]), :, 0].clone()
    want, bound = oracle.attention(q, *cpu, held, tables, lengths, offsets, scale)
    if scale == 1e5:                                        # no score's rounding counts: those of the mean, of P and of out
        bound = torch.full_like(bound, 2.0 ** -8 if dtype == BF16 else 2.0 ** -18) * 6
    close(attend(dev, q, cache, tables, lengths, offsets, scale=scale), want, bound)


@KINDS
@pytest.mark.parametrize("new", [[1, 1, 1], [30, 1, 60]], ids=str)
def test_views(dev, new, dtype, held):
    """Pages by token (num_pages, page_size, G, D), every other page, q by rows and off 16 bytes, tables as part of larger ones."""
    gen = torch.Generator().manual_seed(9)
    lengths = [50, 7, 120]
    tables, num_pages = tables_of(lengths, 16, gen)
    offsets = sums(new)
    cache, cpu = filled(num_pages, 16, 2, 64, dtype, held, gen, dev)
    q = torch.randn(4, offsets[-1], 64, generator=gen).to(dtype)
    want = attend(dev, q, cache, tables, lengths, offsets)

    def turned(x):
        if x is None:
            return None
        y = as_bytes(x)
        wide = torch.zeros(2 * y.shape[0], y.shape[2], y.shape[1], y.shape[3], dtype=y.dtype, device=dev)
        wide[::2] = y.transpose(1, 2)
        return wide[::2].transpose(1, 2).view(x.dtype) if x.dtype != y.dtype else wide[::2].transpose(1, 2)

    other = PagedCache.of(*(turned(x) for x in cache))
    large = torch.full((6, tables.shape[1] + 9), 1 << 20, dtype=torch.int32)
    large[::2, 4:4 + tables.shape[1]] = tables
    part = large.to(dev)[::2, 4:4 + tables.shape[1]]
    qs = [q.to(dev), q.to(dev).transpose(0, 1).contiguous().transpose(0, 1), torch.cat([torch.zeros_like(q[..., :1]), q], 2).to(dev)[..., 1:]]
    for x in qs:
        assert torch.equal(paged_attention(x, other, part, i32(lengths, dev), i32(offsets, dev)), want)
    k, v = (torch.randn(2, offsets[-1], 64, generator=gen).to(dtype).to(dev) for _ in "kv")
    for c, t in ((cache, tables.to(dev)), (other, part)):
        c.write(k, v.transpose(0, 1).contiguous().transpose(0, 1), t, i32(lengths, dev), i32(offsets, dev))
    for x, y in zip(cache, other):
        assert x is None or torch.equal(as_bytes(x), as_bytes(y))
    for x, y in zip(cache.read(tables.to(dev), i32(lengths, dev), 130), other.read(part, i32(lengths, dev), 130)):
        assert torch.equal(x, y)


@pytest.mark.parametrize("dtype,held", [(BF16, BF16), (BF16, I8), (BF16, E4)], ids=["bf16", "int8", "e4m3"])
def test_far_pages(dev, dtype, held):
    """Pages past 2^31 elements of the pool."""
    gen = torch.Generator().manual_seed(10)
    page_size, G, D = 1024, 16, 128
    num_pages = (1 << 31) // (page_size * G * D) + 6
    cache = PagedCache.new(num_pages, page_size, G, D, held)
    small, cpu = filled(6, page_size, G, D, dtype, held, gen, dev)
    for big, x in zip(cache, small):
        if big is not None:
            as_bytes(big)[-6:] = as_bytes(x)
    lengths, new = [2000, 1500], [1, 60]
    near = torch.tensor([[0, 3], [5, 1]], dtype=torch.int32)
    far = near + num_pages - 6
    q = torch.randn(16, 61, D, generator=gen).to(dtype)
    want = attend(dev, q, small, near, lengths, sums(new))
    assert torch.equal(attend(dev, q, cache, far, lengths, sums(new)), want)
    k, v = (torch.randn(G, 61, D, generator=gen).to(dtype).to(dev) for _ in "kv")
    for c, t in ((small, near), (cache, far)):
        c.write(k, v, t.to(dev), i32(lengths, dev), i32(sums(new), dev))
    for x, y in zip(small.read(near.to(dev), i32(lengths, dev), 2000), cache.read(far.to(dev), i32(lengths, dev), 2000)):
        assert torch.equal(x, y)


# ---------------------------------------------------------------------------------------------------------- use
@KINDS
def test_replays_follow_the_tables(dev, dtype, held):
    """A captured step (write, attend) goes on as lengths, tables and offsets change, with eager calls between the replays."""
    gen = torch.Generator().manual_seed(11)
    H, G, D, page_size, B = 4, 2, 64, 16, 3
    cache = PagedCache.new(40, page_size, G, D, held)
    other = PagedCache.new(40, page_size, G, D, held)
    tables = torch.full((B, 12), -1, dtype=torch.int32, device=dev)
    lengths, offsets = i32([1] * B, dev), i32(sums([2, 1, 0]), dev)
    q, k, v = (torch.randn(n, 3, D, generator=gen).to(dtype).to(dev) for n in (H, G, G))

    def step(c):
        c.write(k, v, tables, lengths, offsets)
        return paged_attention(q, c, tables, lengths, offsets)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(other)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held_out = step(cache)
    order = torch.randperm(40, generator=gen).tolist()
    have = [0] * B
    for i in range(12):
        new = [[2, 1, 0], [1, 1, 1], [0, 3, 0], [0, 0, 2]][i % 4]
        for b in range(B):
            have[b] += new[b]
            while (tables[b] >= 0).sum() * page_size < have[b]:
                tables[b, int((tables[b] >= 0).sum())] = order.pop()
        lengths.copy_(i32(have, dev))
        offsets.copy_(i32(sums(new), dev))
        for x, n in ((q, H), (k, G), (v, G)):
            x.copy_(torch.randn(n, 3, D, generator=gen).to(dtype))
        held_out.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held_out, step(other)), i
        for x, y in zip(cache, other):
            assert x is None or torch.equal(as_bytes(x), as_bytes(y))


def test_two_streams_at_once(dev):
    gen = torch.Generator().manual_seed(12)
    lengths = [3000, 2000]
    tables, num_pages = tables_of(lengths, 16, gen)
    cache, _ = filled(num_pages, 16, 2, 64, BF16, I8, gen, dev)
    q = torch.randn(4, 2, 64, generator=gen).to(BF16).to(dev)
    tables, lengths = tables.to(dev), i32(lengths, dev)
    want = paged_attention(q, cache, tables, lengths)
    torch.cuda.synchronize()
    outs = []
    for s in [torch.cuda.Stream() for _ in range(3)]:
        with torch.cuda.stream(s):
            outs += [paged_attention(q, cache, tables, lengths) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


@KINDS
def test_nothing_to_do(dev, dtype, held):
    cache = PagedCache.new(4, 16, 2, 32, held if held not in (F32, BF16) else dtype)
    none = torch.zeros(0, dtype=torch.int32, device=dev)
    empty = torch.zeros(2, 0, 32, dtype=dtype, device=dev)
    cache.write(empty, empty, torch.zeros(0, 3, dtype=torch.int32, device=dev), none)
    assert paged_attention(empty, cache, torch.zeros(0, 3, dtype=torch.int32, device=dev), none).shape == (2, 0, 32)
    # no sequence but rows, no table but a sequence, no page but a table
    x = torch.ones(2, 3, 32, dtype=dtype, device=dev)
    assert (paged_attention(x, cache, torch.zeros(0, 3, dtype=torch.int32, device=dev), none, i32([0], dev)) == 0).all()
    short = torch.zeros(3, 0, dtype=torch.int32, device=dev)
    cache.write(x, x, short, i32([1, 2, 3], dev))
    assert (paged_attention(x, cache, short, i32([1, 2, 3], dev)) == 0).all()
    bare = PagedCache.new(0, 16, 2, 32, cache.k.dtype)
    full = torch.zeros(3, 2, dtype=torch.int32, device=dev)
    bare.write(x, x, full, i32([1, 2, 3], dev))
    assert (paged_attention(x, bare, full, i32([1, 2, 3], dev)) == 0).all()
    assert (paged_attention(torch.ones(2, 90, 32, dtype=dtype, device=dev), bare, full[:1], i32([90], dev), i32([0, 90], dev)) == 0).all()
    assert (bare.read(full, i32([1, 2, 3], dev), 4)[0] == 0).all()


@pytest.mark.parametrize("dtype,held", [(F32, F32), (BF16, BF16), (BF16, I8)], ids=["fp32", "bf16", "bf16_int8"])
@pytest.mark.parametrize("B", [193, 256, 257, 319, 320, 321])
@pytest.mark.parametrize("kind", ["tokens", "mixed"])
def test_as_many_sequences_as_are_looked_up_at_once(dev, kind, B, dtype, held):
    """The last ones that every workgroup looks up by itself (320), and the first that a kernel does before the others."""
    gen = torch.Generator().manual_seed(B)
    new = [1] * B
    if kind == "mixed":
        new[0], new[255 % B], new[B - 2], new[B - 1] = 0, 50, 70, 30
    lengths = [n + m for n, m in zip(new, torch.randint(0, 20, (B,), generator=gen).tolist())]
    lengths[B - 1], lengths[192] = 1500, 900                # in parts
    offsets = sums(new, 1)
    tables, num_pages = tables_of(lengths, 16, gen)
    cache, cpu = filled(num_pages, 16, 2, 64, dtype, held, gen, dev)
    q = torch.randn(4, offsets[-1] + 2, 64, generator=gen).to(dtype)
    want, bound = oracle.attention(q, *cpu, held, tables, lengths, offsets, 0.125)
    got = attend(dev, q, cache, tables, lengths, offsets)
    close(got, want, bound)
    assert (got[:, :1] == 0).all() and (got[:, offsets[-1]:] == 0).all()


@KINDS
@pytest.mark.parametrize("chunk", [500, 520])
def test_tokens_beside_one_chunk(dev, chunk, dtype, held):
    """A chunk that takes its tokens to the tiles (12 / 4 heads, six sequences: from 512 on), and one that does not."""
    gen = torch.Generator().manual_seed(chunk)
    new = [1, 1, chunk - 5, 1, 1, 1]
    lengths = [1, 700, 900, 33, 400, 64]
    offsets = sums(new)
    tables, num_pages = tables_of(lengths, 32, gen)
    cache, cpu = filled(num_pages, 32, 4, 64, dtype, held, gen, dev)
    q = torch.randn(12, offsets[-1], 64, generator=gen).to(dtype)
    want, bound = oracle.attention(q, *cpu, held, tables, lengths, offsets, 0.125)
    close(attend(dev, q, cache, tables, lengths, offsets), want, bound)


@pytest.mark.parametrize("dtype,held", [(F32, F32), (BF16, BF16), (BF16, I8)], ids=["fp32", "bf16", "bf16_int8"])
@pytest.mark.parametrize("parts,new,heads", [(n, [1], (1, 1, 128)) for n in (3, 17, 31, 33, 34, 47, 63, 64, 65, 99, 127)]
                         + [(n, [2], (2, 1, 80)) for n in (33, 49)] + [(n, [1], (2, 1, 64)) for n in (33, 65)]
                         + [(n, [1], (1, 1, 32)) for n in (9, 71)] + [(n, [40], (1, 1, 128)) for n in (33, 35)], ids=str)
def test_every_number_of_parts(dev, parts, new, heads, dtype, held):
    """Parts of 128 positions (256 with chunks), odd numbers of them too, which the lanes that add them up share unevenly."""
    H, G, D = heads
    gen = torch.Generator().manual_seed(parts)
    lengths = [(128 if new[0] < 16 else 256) * parts - 5]
    offsets = sums(new)
    tables, num_pages = tables_of(lengths, 64, gen)
    cache, cpu = filled(num_pages, 64, G, D, dtype, held, gen, dev)
    q = torch.randn(H, offsets[-1], D, generator=gen).to(dtype)
    want, bound = oracle.attention(q, *cpu, held, tables, lengths, offsets, D ** -0.5)
    close(attend(dev, q, cache, tables, lengths, offsets), want, bound)
