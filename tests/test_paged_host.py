"""CPU checks of the cache in pages: the oracle of its 8 bits, what the Python and the C entry points refuse before any kernel
runs, the division by the page size."""

import ctypes
import math
import os
import random

import pytest
import torch

from oracle import paged as oracle
from qlka import _lib
from qlka.paged import PagedCache, paged_attention


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        from qlka import build
        build.build()
    return _lib.load()


# --------------------------------------------------------------------------------------------------------- oracle
def test_e4m3_values_are_torchs():
    codes = torch.arange(256, dtype=torch.uint8)
    want = codes.view(torch.float8_e4m3fn).double()
    assert torch.equal(oracle.E4M3.nan_to_num(nan=1e9), want.nan_to_num(nan=1e9))


@pytest.mark.parametrize("held", [torch.int8, torch.float8_e4m3fn], ids=["int8", "e4m3"])
def test_quantised_rows(held):
    gen = torch.Generator().manual_seed(0)
    x = torch.randn(50, 72, generator=gen) * torch.exp2(torch.randint(-20, 20, (50, 1), generator=gen).float())
    codes, exps = oracle.quantise(x, held)
    y = oracle.values(codes, exps, held)
    for i in range(3):
        part, back, unit = x[:, 32 * i:32 * i + 32].double(), y[:, 32 * i:32 * i + 32], torch.exp2(exps[:, i].double() - 127)
        most = part.abs().amax(1)
        assert (most <= oracle.LARGEST[held] * unit).all() and (most > oracle.LARGEST[held] * unit / 2).all()
        # half a step: of int8 the unit, of e4m3 2^-3 of the value's power of two, 2^-9 at least
        step = unit[:, None] if held == torch.int8 else unit[:, None] * torch.exp2(
            torch.floor(torch.log2((part / unit[:, None]).abs().clamp_min(2.0 ** -6))) - 3)
        assert ((part - back).abs() <= step / 2).all()
    if held == torch.float8_e4m3fn:                  # torch rounds the scaled numbers alike
        scaled = x.double() / torch.exp2(exps.double() - 127).repeat_interleave(32, 1)[:, :72]
        assert torch.equal(scaled.float().to(held).view(torch.uint8), codes)


def test_values_that_are_not_finite():
    x = torch.zeros(3, 64)
    x[0, 3], x[1, 40], x[2, 0] = math.nan, math.inf, 5.0
    for held in (torch.int8, torch.float8_e4m3fn):
        y = oracle.values(*oracle.quantise(x, held), held)
        assert y[0, :32].isnan().all() and (y[0, 32:] == 0).all() and y[1, 32:].isnan().all() and y[2, 0] == 5


def test_division_by_the_page_size():
    """n / size as the high word of 2 n * magic, shifted, for n below 2^31 (its ends, multiples and their neighbours)."""
    rng = random.Random(0)
    for size in list(range(1, 300)) + [rng.randint(300, 65536) for _ in range(300)] + [65535, 65536]:
        shift = (size - 1).bit_length()
        magic = -(-(1 << 31 + shift) // size)
        assert magic < 1 << 32
        for n in [0, 1, size - 1, size, size + 1, (1 << 28) - 1, 1 << 28, (1 << 31) - 1] + [
                rng.randint(0, (1 << 31) // size - 1) * size + d for d in (-1, 0, 1) for _ in range(30)]:
            if n >= 0:
                assert (2 * n * magic >> 32) >> shift == n // size


# ------------------------------------------------------------------------------------------------------- refusals
def test_python_refusals():
    x = torch.zeros(4, 2, 16, 32)
    with pytest.raises(RuntimeError, match="pages must be CUDA tensors"):
        PagedCache.of(x, x)
    with pytest.raises(ValueError, match="dtype must be one of"):
        PagedCache.new(4, 16, 2, 32, torch.float16, device="cpu")
    with pytest.raises(RuntimeError, match="pages must be CUDA tensors"):
        paged_attention(torch.zeros(2, 3, 32), PagedCache(x, x), torch.zeros(3, 1, dtype=torch.int32), torch.zeros(3, dtype=torch.int32))


def args(**kw):
    """Arguments of a small valid call on addresses that nothing reads: every case here fails before a launch."""
    a = _lib.PagedArgs()
    a.dtype, a.held, a.B, a.H, a.G, a.T, a.D, a.scale = 1, 2, 3, 4, 2, 5, 64, 0.125
    a.page_size, a.num_pages, a.table_len, a.N = 16, 9, 4, 50
    for n in ("tables", "lengths", "offsets", "k_pages", "v_pages", "k_exp", "v_exp", "q", "k", "v", "out", "out_k", "out_v"):
        setattr(a, n, 1 << 12)
    a.table_stride = 4
    for n in ("k_pages", "v_pages"):
        setattr(a, n + "_stride", (ctypes.c_int64 * 3)(2048, 1024, 64))
    for n in ("k_exp", "v_exp"):
        setattr(a, n + "_stride", (ctypes.c_int64 * 3)(64, 32, 2))
    for n in ("q", "k", "v", "out"):
        setattr(a, n + "_stride", (ctypes.c_int64 * 2)(320, 64))
    for n in ("out_k", "out_v"):
        setattr(a, n + "_stride", (ctypes.c_int64 * 3)(6400, 3200, 64))
    for n, x in kw.items():
        if n.endswith("_stride") and n != "table_stride":
            x = (ctypes.c_int64 * len(x))(*x)
        setattr(a, n, x)
    return a


def calls(lib, a):
    return {"write": lambda: lib.qlka_paged_write(a, None), "read": lambda: lib.qlka_paged_read(a, None),
            "attention": lambda: lib.qlka_paged_attention(a, 1 << 12, 1 << 50, None)}


WRONG = [
    (dict(dtype=2), "dtype must be"), (dict(held=0), "held must be dtype"), (dict(held=4), "held must be dtype"),
    (dict(B=-1), "must be >= 0"), (dict(T=-1), "must be >= 0"), (dict(G=0), "H and G >= 1"), (dict(G=3), "H must be a multiple"),
    (dict(D=60), "multiple of 8"), (dict(D=136), "multiple of 8"), (dict(T=(1 << 28) + 1), "2^28"),
    (dict(H=1 << 20, T=1 << 20), "must fit int32"), (dict(page_size=0), "page_size must be"), (dict(page_size=65537), "page_size must be"),
    (dict(num_pages=-1), "must be >= 0"), (dict(table_len=-1), "must be >= 0"), (dict(longest=-1), "longest must be"),
    (dict(offsets=None), "T must be B"), (dict(k_pages=None), "k_pages must be non-null"),
    (dict(k_pages=(1 << 12) + 8), "rows of k_pages must be aligned to 16"), (dict(v_pages_stride=(2048, 1024, 72)), "rows of v_pages must be aligned to 16"),
    (dict(D=40, v_pages_stride=(2048, 1024, 36)), "rows of v_pages must be aligned to 8"),
    (dict(k_pages_stride=(-2048, 1024, 64)), "strides of k_pages must be in"),
    (dict(v_pages_stride=(1 << 33, 1024, 64)), "strides of v_pages must be in"), (dict(k_exp_stride=(1 << 32, 32, 2)), "strides of k_exp"),
    (dict(v_pages_stride=(1 << 62, 1024, 64)), "strides of v_pages must be in"),
    (dict(k_exp=None), "k_exp and v_exp must be non-null"), (dict(v_exp_stride=(64, -1, 2)), "strides of k_exp and v_exp must be in"),
    (dict(lengths=None), "tables and lengths must be"), (dict(tables=None), "tables and lengths must be"),
    (dict(table_stride=-4), "table_stride must not"),
]


@pytest.mark.parametrize("wrong,message", WRONG, ids=[m + str(i) for i, (_, m) in enumerate(WRONG)])
def test_wrong_arguments(lib, wrong, message):
    for name, call in calls(lib, ctypes.byref(args(**wrong))).items():
        assert call() == 1, name
        assert message in lib.qlka_last_error().decode(), name


@pytest.mark.parametrize("name,wrong,message", [
    ("write", dict(k=None), "k and v must be non-null"), ("write", dict(v=(1 << 12) + 4), "rows of v must be aligned"),
    ("write", dict(k_stride=(320, 63)), "rows of k must be aligned"), ("write", dict(k_stride=(-320, 64)), "must not be negative"),
    ("read", dict(out_k=None), "out_k and out_v must be"), ("read", dict(out_v=(1 << 12) + 4), "rows of out_v must be aligned"),
    ("read", dict(N=(1 << 28) + 1), "2^28"), ("read", dict(B=1 << 14, N=1 << 20), "must fit int32"),
    ("attention", dict(q=None), "q and out must be"), ("attention", dict(out=(1 << 12) + 2), "rows of out must be aligned"),
    ("attention", dict(scale=float("inf")), "scale must be 0 or"), ("attention", dict(scale=1e-38), "scale must be 0 or"),
])
def test_wrong_arguments_of_one(lib, name, wrong, message):
    assert calls(lib, ctypes.byref(args(**wrong)))[name]() == 1
    assert message in lib.qlka_last_error().decode()


def test_workspaces(lib):
    a = args(B=1, T=1, H=2, G=1, offsets=None, table_len=4096)
    need = lib.qlka_paged_attention_ws_bytes(ctypes.byref(a))
    assert need > 0 and lib.qlka_paged_attention(ctypes.byref(a), 1 << 12, need - 1, None) == 2
    assert lib.qlka_paged_attention(ctypes.byref(a), None, need, None) == 2
    assert "workspace" in lib.qlka_last_error().decode()
    assert lib.qlka_paged_attention_ws_bytes(None) == 0 and lib.qlka_paged_attention_ws_bytes(ctypes.byref(args(D=3))) == 0
    assert lib.qlka_paged_attention_ws_bytes(ctypes.byref(args(table_len=2))) == 0           # nothing to split


@pytest.mark.parametrize("H,G,D", [(12, 12, 64), (12, 4, 64), (32, 32, 128)])
def test_workspace_of_a_chunk_among_many_tokens(lib, H, G, D):
    """Parts' places go by the sequences that can have them: a chunk among single tokens takes no more than both apart and
    a block of 128 rows for each sequence long enough for the tiles; sequences without a token take none."""
    def need(**kw):
        return lib.qlka_paged_attention_ws_bytes(ctypes.byref(args(H=H, G=G, D=D, held=1, page_size=64, table_len=128, **kw)))
    apart = need(B=2000, T=2000, offsets=None) + need(B=1, T=512)
    share, few = H // G, 16
    long_enough = 2511 // (few // share + 1)
    assert need(B=2000, T=2511) <= apart + 2 * long_enough * G * 128 * (D + 2) * 4
    assert need(B=2000, T=20) <= need(B=20, T=20) + (1 << 20)


def test_one_round_of_workgroups(lib):
    """fp32 rows of 128: a compute unit has room for one workgroup (96 KB of LDS, or more than 256 registers), so parts are
    cut, and have places, for 256 of them."""
    sizes = dict(dtype=0, H=8, G=8, D=128, T=1, B=1, offsets=None, table_len=4096)
    pages = {n + "_stride": (16 * 8 * 128, 16 * 128, 128) for n in ("k_pages", "v_pages")}
    place = 16 * (128 + 2) * 4
    need = lambda held: lib.qlka_paged_attention_ws_bytes(ctypes.byref(args(held=held, **sizes, **pages)))  # noqa: E731
    assert 250 * place < need(0) <= (256 + 2 * 8) * place + 512
    assert need(2) > 500 * place                            # of 8 bits: two


def test_nothing_to_do(lib):
    a = args(B=0, T=0, N=0, offsets=None, tables=None, lengths=None, q=None, k=None, v=None, out=None, out_k=None, out_v=None)
    for name, call in calls(lib, ctypes.byref(a)).items():
        assert call() == 0, name
