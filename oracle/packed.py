"""Softmax attention within packed sequences in float64, with its gradients and bounds: oracle/softmax.py, sequence by
sequence.
TEST INFRASTRUCTURE ONLY.
"""

import torch

from . import softmax


def attention(q, k, v, offsets, scale, causal, g=None):
    """q (H, T, D), k and v (G, T, D), offsets a list: {"out", "gq", "gk", "gv"} and their "bound"; rows outside the
    sequences are zeros with the bound 0."""
    names = ("out",) if g is None else ("out", "gq", "gk", "gv")
    like = {"out": q, "gq": q, "gk": k, "gv": v}
    r = {n: torch.zeros(like[n].shape, dtype=torch.float64) for n in names}
    r["bound"] = {n: torch.zeros(like[n].shape, dtype=torch.float64) for n in names}
    for lo, hi in zip(offsets, offsets[1:]):
        if lo == hi:
            continue
        part = [x[None, :, lo:hi] for x in (q, k, v)]
        see = softmax.visible(1, hi - lo, hi - lo, causal=causal)
        one = softmax.attention(*part, scale, see, None if g is None else g[None, :, lo:hi])
        for n in names:
            r[n][:, lo:hi] = one[n][0]
            r["bound"][n][:, lo:hi] = one["bound"][n][0]
    return r
