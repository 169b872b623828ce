"""CPU checks of softmax attention and the position bias: the bucket borders, what the Python and the C entry points refuse
before any kernel runs, and the modules' plumbing against torch's own attention."""

import ctypes
import math
import os

import pytest
import torch

from oracle import softmax as oracle
from qlka import _lib, modules
from qlka.softmax import RelativeBuckets, relative_bias, softmax_attention


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        from qlka import build
        build.build()
    return _lib.load()


# --------------------------------------------------------------------------------------------------------- buckets
@pytest.mark.parametrize("num,distance,both", [(32, 128, True), (32, 128, False), (64, 500, True), (16, 9, False), (4, 3, True),
                                               (2, 1, True), (1, 1, False), (3, 5, False), (255, 4096, False), (256, 300, True)])
def test_borders_are_where_the_bucket_changes(num, distance, both):
    borders = RelativeBuckets(num, distance, both).borders
    side = num // 2 if both else num
    assert len(borders) == side - 1 and list(borders) == sorted(borders)
    row = oracle.bucket_map(1, 600, 599, num, distance, both)[0].flip(0)           # distances 0 .. 599 of earlier keys
    for dist in range(600):
        assert sum(b <= dist for b in borders) == row[dist], dist


def test_borders_against_the_logarithm():
    # away from exact ties the formula in floating point gives the same buckets
    borders = RelativeBuckets(32, 128, False).borders
    for dist in range(1, 127):
        want = dist if dist < 16 else min(31, 16 + math.floor(math.log(dist / 16) / math.log(8) * 16 + 1e-9))
        assert sum(b <= dist for b in borders) == want


@pytest.mark.parametrize("args", [(3, 128, True), (0, 5, False), (258, 999, True), (257, 999, False), (32, 8, True), (8, 4, False)])
def test_buckets_that_do_not_exist(args):
    with pytest.raises(ValueError, match="num_buckets|max_distance"):
        RelativeBuckets(*args).borders
    with pytest.raises(ValueError):
        modules.RelativePositionBias(2, *args)


# ------------------------------------------------------------------------------------------------- Python refusals
def test_python_refusals():
    x = torch.zeros(1, 2, 4, 8)
    with pytest.raises(RuntimeError, match="q, k and v must be CUDA tensors"):
        softmax_attention(x, x, x)
    with pytest.raises(RuntimeError, match="table must be a CUDA tensor"):
        relative_bias(torch.zeros(32, 2), 4, 4)
    with pytest.raises(ValueError, match="buckets without a table"):
        softmax_attention(x, x, x, buckets=RelativeBuckets())


# ------------------------------------------------------------------------------------------------------- C refusals
def args(**kw):
    """Arguments of a small valid call on addresses that nothing reads: every case here fails before a launch."""
    a = _lib.SoftmaxArgs()
    a.dtype, a.B, a.H, a.G, a.M, a.N, a.D, a.scale = 0, 2, 4, 2, 5, 7, 64, 0.125
    for n in ("q", "k", "v", "out", "g_out", "g_q", "g_k", "g_v"):
        setattr(a, n, 1 << 12)
    a.lse = 1 << 12
    for n, heads, rows in (("q", 4, 5), ("k", 2, 7), ("v", 2, 7), ("out", 4, 5), ("g_out", 4, 5), ("g_q", 4, 5), ("g_k", 2, 7), ("g_v", 2, 7)):
        setattr(a, n + "_stride", (ctypes.c_int64 * 3)(heads * rows * 64, rows * 64, 64))
    a.keepalive = []
    for n, x in kw.items():
        if n.endswith("_stride") and n != "keep_stride":
            x = (ctypes.c_int64 * 3)(*x)
        if n == "border":
            x = (ctypes.c_int * len(x))(*x)
            a.keepalive.append(x)
            a.num_borders = len(x)
            x = ctypes.cast(x, ctypes.POINTER(ctypes.c_int))
        setattr(a, n, x)
    return a


WRONG = [
    (dict(dtype=2), "dtype must be"), (dict(B=-1), "B, M and N must be >= 0"), (dict(M=-1), "must be >= 0"),
    (dict(G=0), "H and G >= 1"), (dict(G=3), "H must be a multiple of G"), (dict(D=0), "multiple of 8"),
    (dict(D=60), "multiple of 8"), (dict(D=136), "multiple of 8"), (dict(N=(1 << 28) + 1), "2^28"), (dict(start=-(1 << 28) - 1), "2^28"),
    (dict(B=1 << 20, M=1 << 20), "must fit int32"), (dict(scale=float("nan")), "scale must be 0 or"),
    (dict(scale=float("inf")), "scale must be 0 or"), (dict(scale=1e-38), "scale must be 0 or"),
    (dict(q=(1 << 12) + 4), "rows of q must be aligned"), (dict(v_stride=(896, 448, 66)), "rows of v must be aligned"),
    (dict(table=1 << 12, border=[3, 2]), "border must be positive"), (dict(table=1 << 12, border=[0]), "border must be positive"),
    (dict(table=1 << 12, border=list(range(1, 257))), "at most 256 buckets"),
    (dict(table=1 << 12, border=list(range(1, 129)), bidirectional=1), "at most 256 buckets"),
    (dict(table=1 << 12, num_borders=3), "border must be non-null"), (dict(k=None), "must be non-null"),
    (dict(out_full=1 << 12), "out_full goes with"),
]


@pytest.mark.parametrize("wrong,message", WRONG, ids=[m + str(i) for i, (_, m) in enumerate(WRONG)])
def test_wrong_arguments(lib, wrong, message):
    a = args(**wrong)
    for fn in (lib.qlka_softmax_fwd, lib.qlka_softmax_bwd):
        assert fn(ctypes.byref(a), 1 << 12, 1 << 40, None) == 1
        assert message in lib.qlka_last_error().decode()


def test_backward_refusals(lib):
    for wrong, message in ((dict(g_v=None), "both or neither"), (dict(g_table=1 << 12), "g_table needs the table"),
                           (dict(lse=None), "must be non-null"), (dict(g_out=None), "must be non-null"),
                           (dict(dtype=1, table=1 << 12, border=[1], g_table=1 << 12), "g_table needs out_full")):
        a = args(**wrong)
        assert lib.qlka_softmax_bwd(ctypes.byref(a), 1 << 12, 1 << 40, None) == 1
        assert message in lib.qlka_last_error().decode()
    assert lib.qlka_softmax_fwd(None, None, 0, None) == 1 and lib.qlka_softmax_bwd(None, None, 0, None) == 1
    assert lib.qlka_softmax_fwd_ws_bytes(None) == 0


def test_workspaces(lib):
    a = args(B=1, M=1, N=100000)                                   # few rows, many keys: split
    need = lib.qlka_softmax_fwd_ws_bytes(ctypes.byref(a))
    assert need > 0
    assert lib.qlka_softmax_fwd(ctypes.byref(a), 1 << 12, need - 1, None) == 2
    assert "workspace" in lib.qlka_last_error().decode()
    assert lib.qlka_softmax_fwd(ctypes.byref(a), None, need, None) == 2
    assert lib.qlka_softmax_fwd(ctypes.byref(a), (1 << 12) + 4, need, None) == 2
    a = args(B=64, M=1024, N=1024)
    assert lib.qlka_softmax_fwd_ws_bytes(ctypes.byref(a)) == 0
    need = lib.qlka_softmax_bwd_ws_bytes(ctypes.byref(a))
    assert need >= 64 * 4 * 1024 * 4                               # a row sum a query
    assert lib.qlka_softmax_bwd(ctypes.byref(a), 1 << 12, need - 1, None) == 2
    only_q = args(B=64, M=1024, N=1024, g_k=None, g_v=None)
    assert lib.qlka_softmax_bwd_ws_bytes(ctypes.byref(only_q)) <= need


def test_nothing_to_do(lib):
    for empty in (dict(B=0), dict(M=0)):
        a = args(**empty)
        assert lib.qlka_softmax_fwd(ctypes.byref(a), None, 0, None) == 0


def test_map_refusals(lib):
    border = (ctypes.c_int * 2)(1, 2)
    ok = dict(table=1 << 12, border=border, n=2, both=0, out=1 << 12, H=2, M=3, N=4, start=0)

    def fwd(**kw):
        a = {**ok, **kw}
        return lib.qlka_bias_map_fwd(a["table"], a["border"], a["n"], a["both"], a["out"], a["H"], a["M"], a["N"], a["start"], None)

    for wrong, message in ((dict(H=0), "H must be"), (dict(M=-1), "M and N"), (dict(N=(1 << 21) + 1), "M and N"),
                           (dict(start=1 << 29), "start"), (dict(n=-1), "buckets"), (dict(n=256), "buckets"), (dict(table=None), "non-null")):
        assert fwd(**wrong) == 1 and message in lib.qlka_last_error().decode(), wrong
    assert fwd(M=0) == 0
    need = lib.qlka_bias_map_bwd_ws_bytes(2, 0, 2, 3, 4)
    assert lib.qlka_bias_map_bwd(1 << 12, border, 2, 0, 1 << 12, 2, 3, 4, 0, 1 << 12, need - 1, None) == 2
    assert lib.qlka_bias_map_bwd(None, border, 2, 0, 1 << 12, 2, 3, 4, 0, 1 << 12, need, None) == 1


# ---------------------------------------------------------------------------------------------------------- modules
def test_cross_attention_equals_nn_multihead_attention():
    torch.manual_seed(0)
    E, H = 32, 4
    ref = torch.nn.MultiheadAttention(E, H, batch_first=True)
    torch.nn.init.normal_(ref.in_proj_bias)
    mod = modules.KernelMultiheadAttention(E, H, kernel="softmax", tau=(E // H) ** 0.25)
    mod.load_state_dict(ref.state_dict())
    x, states = torch.randn(3, 5, E), torch.randn(3, 11, E)
    keep = torch.rand(3, 11) < 0.7
    keep[:, 0] = True
    want, _ = ref(x, states, states, key_padding_mask=~keep, need_weights=False)
    torch.testing.assert_close(mod(x, keep, states), want, rtol=1e-5, atol=1e-6)
    torch.testing.assert_close(mod(x, keep, mod.project_context(states)), want, rtol=1e-5, atol=1e-6)
    # token by token over its own heads
    causal = torch.ones(5, 5, dtype=torch.bool).triu(1)
    want, _ = ref(x, x, x, attn_mask=causal, need_weights=False)
    torch.testing.assert_close(mod(x, causal=True), want, rtol=1e-5, atol=1e-6)
    k, v = mod.project_context(x)
    steps = [mod(x[:, i:i + 1], context=(k[:, :, :i + 1], v[:, :, :i + 1]), causal=True, start=i) for i in range(5)]
    torch.testing.assert_close(torch.cat(steps, 1), want, rtol=1e-5, atol=1e-6)


def test_what_the_additive_kernels_do_not_do():
    mod = modules.KernelMultiheadAttention(32, 4, kernel="add_riesz")
    x = torch.randn(1, 5, 32)
    for kw in (dict(context=x), dict(causal=True)):
        with pytest.raises(NotImplementedError, match="softmax"):
            mod(x, **kw)
    with pytest.raises(NotImplementedError, match="softmax"):
        modules.KernelMultiheadAttention(32, 4, kernel="add_bump", position_bias=modules.RelativePositionBias(4))


def test_position_bias_parameters():
    mod = modules.KernelMultiheadAttention(32, 4, position_bias=modules.RelativePositionBias(4, 16, 64, False))
    assert mod.state_dict()["position_bias.weight"].shape == (16, 4)
    assert sorted(n for n, _ in modules.KernelMultiheadAttention(32, 4).named_parameters()) == sorted(
        n for n, _ in mod.named_parameters() if not n.startswith("position_bias"))
    with pytest.raises(RuntimeError, match="CUDA"):
        mod(torch.randn(1, 5, 32))


@pytest.mark.parametrize("borders", [-5, 256, 1 << 30])
def test_workspace_of_impossible_buckets_is_none(borders):
    a = args(table=1 << 12, g_table=1 << 12)
    a.num_borders = borders
    assert _lib.load().qlka_softmax_bwd_ws_bytes(ctypes.byref(a)) == 0
    assert _lib.load().qlka_bias_map_bwd_ws_bytes(borders, 0, 2, 30, 40) == 0


# --------------------------------------------------------------------------------------------- strides, sizes, launches
@pytest.mark.parametrize("name,heads,rows", [("q", 4, 5), ("k", 2, 7), ("v", 2, 7), ("out", 4, 5), ("g_out", 4, 5), ("g_q", 4, 5),
                                             ("g_k", 2, 7), ("g_v", 2, 7)])
def test_negative_strides_are_refused(lib, name, heads, rows):
    # rows of a tile are found by unsigned offsets from its first one
    good = (heads * rows * 64, rows * 64, 64)
    for i in range(3):
        a = args(**{name + "_stride": [-s if i == j else s for j, s in enumerate(good)]})
        for fn in (lib.qlka_softmax_fwd, lib.qlka_softmax_bwd):
            assert fn(ctypes.byref(a), 1 << 12, 1 << 40, None) == 1
            assert f"strides of {name} must not be negative" in lib.qlka_last_error().decode()


def test_strides_of_single_rows_may_be_anything(lib):
    a = args(B=1, H=1, G=1, M=0, N=1, **{n + "_stride": (-8, -8, -8) for n in ("q", "k", "v", "out")})
    assert lib.qlka_softmax_fwd(ctypes.byref(a), None, 0, None) == 0           # nothing to do, and nothing refused


def refused(lib, fn, message, **kw):
    a = args(**kw)
    assert fn(ctypes.byref(a), 1 << 12, 1 << 44, None) == 1
    assert message in lib.qlka_last_error().decode()


def test_launches_past_2_32_threads_are_refused(lib):
    """B * G single tokens take a workgroup of 256 threads each, and a launch less than 2^32 threads."""
    one = dict(H=1, G=1, D=8, table=None)
    many = "too many workgroups"
    refused(lib, lib.qlka_softmax_fwd, many, **one, B=1 << 24, M=1, N=1)                        # a workgroup a token
    refused(lib, lib.qlka_softmax_fwd, many, **one, B=1 << 24, M=5, N=1)                        # a workgroup 128 rows
    nothing = dict(g_q=None, g_k=None, g_v=None)
    for wanted in (dict(g_q=1 << 12), dict(g_k=1 << 12, g_v=1 << 12)):                          # two waves a workgroup
        refused(lib, lib.qlka_softmax_bwd, many, **{**one, **nothing, **wanted}, B=1 << 25, M=1, N=1)
    wide = {**one, **nothing, "B": 1 << 26, "M": 1, "N": 0}                                     # row sums: a wave 32 rows
    refused(lib, lib.qlka_softmax_bwd, many, **wide)
    refused(lib, lib.qlka_softmax_bwd, many, H=1 << 24, G=1, B=1, M=0, N=1, D=8, g_q=None, g_k=None, g_v=None, table=1 << 12,
            g_table=1 << 12, border=[1])                                                       # a workgroup a head and bucket


@pytest.mark.parametrize("name", ["q", "k", "v", "table"])
@pytest.mark.parametrize("D", [8, 5])
def test_forward_mode_is_refused(name, D):
    """Not dropped: a tangent on an input that wants no gradient would be lost without a word."""
    import torch.autograd.forward_ad as fwAD
    x = {n: torch.zeros(1, 2, 4, D) for n in "qkv"}
    x["table"] = torch.zeros(32, 2)
    with fwAD.dual_level():
        x[name] = fwAD.make_dual(x[name], torch.ones_like(x[name]))
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            softmax_attention(x["q"], x["k"], x["v"], table=x["table"])


def test_start_goes_with_a_context():
    """Without one the keys are x's own, from position 0 on: queries placed after them would see tokens to come."""
    x = torch.randn(1, 5, 32)
    for mod in (modules.KernelMultiheadAttention(32, 4),
                modules.KernelMultiheadAttention(32, 4, position_bias=modules.RelativePositionBias(4, bidirectional=False))):
        for causal in (False, True):
            with pytest.raises(ValueError, match="start 3 without a context"):
                mod(x, causal=causal, start=3)
    mod = modules.KernelMultiheadAttention(32, 4)
    torch.testing.assert_close(mod(x, start=0), mod(x))
