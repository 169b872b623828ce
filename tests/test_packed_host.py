"""CPU checks of packed attention: the numbering of blocks, what the Python and the C entry points refuse before any kernel."""

import ctypes
import os
import random

import pytest
import torch

from qlka import _lib
from qlka.packed import packed_attention


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        from qlka import build
        build.build()
    return _lib.load()


@pytest.mark.parametrize("share,rows", [(1, 32), (1, 128), (3, 128), (4, 16), (12, 32)])
def test_every_row_has_one_block(share, rows):
    """The numbers that csrc/segments.h gives to the blocks: each row in one, none twice, all below the launch's size."""
    rng = random.Random(share * rows)
    for _ in range(300):
        B, T = rng.randint(0, 9), rng.choice([0, 1, 31, 32, 33, 200, 1000])
        offsets = sorted(rng.randint(0, T) for _ in range(B + 1))
        edge = [0] + offsets + [T]
        starts = [edge[j] * share // rows + j for j in range(B + 2)]
        assert starts[0] == 0 and all(a < b for a, b in zip(starts, starts[1:]))
        most, seen = T * share // rows + B + 2, set()
        for number in range(most):
            j = max(i for i in range(B + 2) if starts[i] <= number)
            mine, block = (edge[j + 1] - edge[j]) * share, number - starts[j]
            for r in range(block * rows, min((block + 1) * rows, mine)):
                assert (j, r) not in seen
                seen.add((j, r))
        assert len(seen) == T * share


def test_python_refusals():
    x, at = torch.zeros(2, 4, 8), torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="q, k and v must be CUDA tensors"):
        packed_attention(x, x, x, at)


def args(**kw):
    """Arguments of a small valid call on addresses that nothing reads: every case here fails before a launch."""
    a = _lib.PackedArgs()
    a.dtype, a.B, a.H, a.G, a.T, a.D, a.scale = 0, 2, 4, 2, 5, 64, 0.125
    for n in ("q", "k", "v", "out", "g_out", "g_q", "g_k", "g_v", "log_sums", "offsets"):
        setattr(a, n, 1 << 12)
    for n in ("q", "k", "v", "out", "g_out", "g_q", "g_k", "g_v"):
        setattr(a, n + "_stride", (ctypes.c_int64 * 2)(5 * 64, 64))
    for n, x in kw.items():
        setattr(a, n, (ctypes.c_int64 * 2)(*x) if n.endswith("_stride") else x)
    return a


WRONG = [
    (dict(dtype=2), "dtype must be"), (dict(B=-1), "B and T must be >= 0"), (dict(T=-1), "B and T must be >= 0"),
    (dict(G=0), "H and G >= 1"), (dict(G=3), "H must be a multiple of G"), (dict(D=0), "multiple of 8"),
    (dict(D=60), "multiple of 8"), (dict(D=136), "multiple of 8"), (dict(T=(1 << 28) + 1), "2^28"),
    (dict(B=(1 << 28) + 1), "2^28"), (dict(H=1 << 20, T=1 << 20), "must fit int32"), (dict(scale=float("nan")), "scale must be 0 or"),
    (dict(scale=1e-38), "scale must be 0 or"), (dict(q=(1 << 12) + 4), "rows of q must be aligned"),
    (dict(v_stride=(320, 66)), "rows of v must be aligned"), (dict(k_stride=(-320, 64)), "strides of k must not be negative"),
    (dict(out_full=1 << 12), "out_full goes with"), (dict(k=None), "must be non-null"), (dict(offsets=None), "offsets must be non-null"),
    (dict(H=1 << 20, G=1, T=1 << 10, B=1 << 12), "too many workgroups"),
]


@pytest.mark.parametrize("wrong,message", WRONG, ids=[m + str(i) for i, (_, m) in enumerate(WRONG)])
def test_wrong_arguments(lib, wrong, message):
    a = args(**wrong)
    for fn in (lib.qlka_packed_fwd, lib.qlka_packed_bwd):
        assert fn(ctypes.byref(a), 1 << 12, 1 << 50, None) == 1
        assert message in lib.qlka_last_error().decode()


def test_backward_refusals(lib):
    for wrong, message in ((dict(g_v=None), "both or neither"), (dict(log_sums=None), "must be non-null"),
                           (dict(g_out=None), "must be non-null")):
        a = args(**wrong)
        assert lib.qlka_packed_bwd(ctypes.byref(a), 1 << 12, 1 << 50, None) == 1
        assert message in lib.qlka_last_error().decode()
    assert lib.qlka_packed_fwd(None, None, 0, None) == 1 and lib.qlka_packed_bwd(None, None, 0, None) == 1


def test_workspaces(lib):
    a = args(T=4096, H=1, G=1, B=1)
    need = lib.qlka_packed_bwd_ws_bytes(ctypes.byref(a))
    assert need > 0 and lib.qlka_packed_bwd(ctypes.byref(a), 1 << 12, need - 1, None) == 2
    assert lib.qlka_packed_bwd(ctypes.byref(a), None, need, None) == 2
    assert lib.qlka_packed_bwd(ctypes.byref(a), (1 << 12) + 8, need, None) == 2
    assert "workspace" in lib.qlka_last_error().decode()
    fwd = lib.qlka_packed_fwd_ws_bytes(ctypes.byref(a))
    assert fwd > 0 and lib.qlka_packed_fwd(ctypes.byref(a), 1 << 12, fwd - 1, None) == 2          # split
    assert lib.qlka_packed_fwd_ws_bytes(None) == 0 and lib.qlka_packed_bwd_ws_bytes(ctypes.byref(args(D=7))) == 0


def test_nothing_to_do(lib):
    a = args(T=0, q=None, k=None, v=None, out=None)
    assert lib.qlka_packed_fwd(ctypes.byref(a), None, 0, None) == 0
