"""Softmax attention within packed sequences in float64, with its gradients and bounds: oracle/softmax.py sequence by sequence.
TEST INFRASTRUCTURE ONLY.

With bfloat16 the rows' sums, by which the probabilities of the gradients are divided, are those of the rounded exponentials:
every term is off by at most h = 2^-8 of its size, all of them positive, so the sum l by at most h l, and P = E / l by at most
h P / (1 - h) before its own rounding. That is another h of the terms of gv = P^T g, and of dS = P (dP - delta), from which gq
and gk are. Rows of few keys come near it (the roundings of many average out).
"""

import torch

from . import softmax


def attention(q, k, v, offsets, scale, causal, g=None):
    """q (H, T, D), k and v (G, T, D), offsets a list: {"out", "gq", "gk", "gv"} and their "bound"; rows outside the sequences are
    zeros with the bound 0."""
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
        if g is not None and softmax.ROUND[q.dtype]:
            _add_sums(one["bound"], *part, g[None, :, lo:hi], scale, see)
        for n in names:
            r[n][:, lo:hi] = one[n][0]
            r["bound"][n][:, lo:hi] = one["bound"][n][0]
    return r


def _add_sums(bound, q, k, v, g, scale, see):
    """The share of the rows' sums in the bounds of the gradients (above)."""
    h = softmax.ROUND[q.dtype]
    share = q.shape[1] // k.shape[1]
    q, g, k, v = q.double(), g.double(), k.double().repeat_interleave(share, 1), v.double().repeat_interleave(share, 1)
    P = torch.softmax((q @ k.transpose(-1, -2) * scale).masked_fill(~see[:, None], float("-inf")), -1)
    dP = g @ v.transpose(-1, -2)
    dS = P * (dP - (P * dP).sum(-1, keepdim=True))
    per = lambda x: x.unflatten(1, (-1, share)).sum(2)  # noqa: E731
    more = h / (1 - h)
    bound["gv"] += more * per(P.transpose(-1, -2) @ g.abs())
    bound["gq"] += more * abs(scale) * (dS.abs() @ k.abs())
    bound["gk"] += more * abs(scale) * per(dS.abs().transpose(-1, -2) @ q.abs())
