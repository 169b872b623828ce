"""Softmax attention with a bucketed position bias in float64, with its gradients, and how far a computation in a given type
may be from them. TEST INFRASTRUCTURE ONLY.

Everything is formed whole, on the CPU, from the definitions. `bounds` follows a computation whose products and sums are
fp32 (relative error u = 2^-24 an operation, sums of n terms n u of the sum of the terms' sizes) and which, for bfloat16
operands, rounds P and dS for their products and each result at its end by at most h = 2^-8 of its size.
"""

import torch

U = 2.0 ** -24
ROUND = {torch.float32: 0.0, torch.bfloat16: torch.finfo(torch.bfloat16).eps / 2}


def bucket_map(M, N, start, num_buckets, max_distance, bidirectional):
    """(M, N) bucket of every (query, key), one at a time, in whole numbers."""
    side = num_buckets // 2 if bidirectional else num_buckets
    single = side // 2
    steps = side - single

    def of(dist):
        if dist < single or side == 1:
            return min(dist, side - 1)
        j = 0
        while j + 1 < steps and dist ** steps >= max_distance ** (j + 1) * single ** (steps - j - 1):
            j += 1
        return single + j if single else 0

    seen = {}

    def bucket(d):
        if d not in seen:
            dist = abs(d) if bidirectional else max(-d, 0)
            seen[d] = of(dist) + (side if bidirectional and d > 0 else 0)
        return seen[d]

    return torch.tensor([[bucket(n - m - start) for n in range(N)] for m in range(M)], dtype=torch.long).view(M, N)


def visible(B, M, N, keep=None, causal=False, start=0):
    see = torch.ones(B, M, N, dtype=torch.bool)
    if keep is not None:
        see &= (keep != 0)[:, None, :]
    if causal:
        see &= torch.arange(N)[None, None, :] <= torch.arange(M)[None, :, None] + start
    return see


def attention(q, k, v, scale, see, g=None, table=None, buckets=None):
    """{"out", "gq", "gk", "gv", "gtable"} in float64, and under "bound" the same names' bounds. buckets: bucket_map's."""
    dtype = q.dtype
    h = ROUND[dtype]
    B, H, M, D = q.shape
    G, N = k.shape[1], k.shape[2]
    share = H // G
    # rows that no query of the batch sees may hold anything
    used = see.any(1)[:, None, :, None]
    q, k, v = q.double(), torch.where(used, k.double(), 0.0), torch.where(used, v.double(), 0.0)
    K, V = k.repeat_interleave(share, 1), v.repeat_interleave(share, 1)
    bias = torch.zeros(H, M, N, dtype=torch.float64) if table is None else table.double().t()[:, buckets.flatten()].view(H, M, N)
    S = (q @ K.transpose(-1, -2)) * scale + bias
    see4 = see[:, None]
    S = S.masked_fill(~see4, float("-inf"))
    top = S.amax(-1, keepdim=True) if N else torch.zeros(B, H, M, 1, dtype=torch.float64)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    E = torch.exp(S - top)
    l = E.sum(-1, keepdim=True)
    P = torch.where(l > 0, E / torch.where(l > 0, l, 1.0), torch.zeros_like(E))
    out = P @ V
    r = {"out": out}

    # score: D products and sums, the bias, the change to log2 units; exp2; the row's sum of N
    size = abs(scale) * (q.abs() @ K.abs().transpose(-1, -2)) + torch.where(torch.isfinite(bias), bias, 0.0).abs()
    size = torch.where(see4, size, torch.zeros_like(size))
    top_size = size.amax(-1, keepdim=True) if N else torch.zeros(B, H, M, 1, dtype=torch.float64)
    e = 2 * ((D + 16) * U * top_size + 8 * U) + (2 * N + 32) * U
    PV = P @ V.abs()
    err_out = (e + h) * PV
    b = {"out": err_out + h * out.abs()}
    if g is not None:
        g = g.double()
        dP = g @ V.transpose(-1, -2)
        delta = (g * out).sum(-1, keepdim=True)
        dS = P * (dP - delta)
        r["gq"] = dS @ K * scale
        per = lambda x: x.view(B, G, share, N, D).sum(2)  # noqa: E731
        r["gk"] = per(dS.transpose(-1, -2) @ q * scale)
        r["gv"] = per(P.transpose(-1, -2) @ g)
        small = 2.0 ** -15 if h else 0.0                     # with the table: P and out to 16 bits
        err_delta = (g.abs() * (((e + small) * PV) if table is not None else b["out"])).sum(-1, keepdim=True)
        err_delta = err_delta + (D + 16) * U * (g.abs() * out.abs()).sum(-1, keepdim=True)
        err_dP = (D + 16) * U * (g.abs() @ V.abs().transpose(-1, -2))
        err_S = P * (e * (dP.abs() + delta.abs()) + err_dP + err_delta)
        b["gq"] = abs(scale) * ((err_S + (h + (N + 8) * U) * dS.abs()) @ K.abs()) + h * r["gq"].abs()
        b["gk"] = per(abs(scale) * ((err_S + (h + (share * M + 8) * U) * dS.abs()).transpose(-1, -2) @ q.abs())) + h * r["gk"].abs()
        b["gv"] = per((P * (e + h + (share * M + 8) * U)).transpose(-1, -2) @ g.abs()) + h * r["gv"].abs()
        if table is not None:
            num = table.shape[0]
            hot = torch.nn.functional.one_hot(buckets.flatten(), num).double()              # (M N, num)
            r["gtable"] = (dS.sum(0).view(H, -1) @ hot).t()
            err = err_S.sum(0) + (N + B * M + 64) * U * dS.abs().sum(0)
            b["gtable"] = (err.view(H, -1) @ hot).t()
    r["bound"] = b
    return r
