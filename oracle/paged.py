"""A cache of keys and values in pages on the CPU, from the definitions: what 8 bits hold of a row, where a token goes, what a
sequence reads back, and attention over it in float64. TEST INFRASTRUCTURE ONLY."""

import math

import torch

from . import softmax

BLOCK = 32
LARGEST = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
TOP = {torch.int8: 248, torch.float8_e4m3fn: 246}
LEAST = 27


def _e4m3_values():
    got = []
    for code in range(256):
        e, m = code >> 3 & 15, code & 7
        if code & 127 == 127:
            got.append(math.nan)
        else:
            x = (m / 8) * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
            got.append(-x if code & 128 else x)
    return torch.tensor(got, dtype=torch.float64)


E4M3 = _e4m3_values()


def quantise(x, held):
    """(codes as bytes, exponents) of rows x (..., D): blocks of 32, one at a time in float64."""
    D = x.shape[-1]
    rows = x.double().reshape(-1, D)
    codes = torch.zeros(rows.shape, dtype=torch.uint8)
    exps = torch.zeros(rows.shape[0], -(-D // BLOCK), dtype=torch.uint8)
    for i in range(exps.shape[1]):
        part = rows[:, i * BLOCK:(i + 1) * BLOCK]
        most = part.abs().amax(1)
        bad = ~torch.isfinite(part).all(1)
        e = torch.full(most.shape, LEAST, dtype=torch.long)
        for step in range(LEAST, TOP[held]):
            e = torch.where((most > LARGEST[held] * 2.0 ** (step - 127)) & (e == step), e + 1, e)
        y = (torch.where(bad[:, None], 0.0, part) / torch.exp2(e.double() - 127)[:, None]).clamp(-LARGEST[held], LARGEST[held])
        if held == torch.int8:
            code = torch.round(y).to(torch.int8).view(torch.uint8)
        else:
            # the nearest value, of two the one with the even code
            dist = (y[..., None].abs() - E4M3[:127].view(1, 1, -1)).abs()
            near = dist.amin(-1, keepdim=True)
            pick = torch.where(dist == near, torch.arange(127), 1000)
            even = torch.where((dist == near) & (torch.arange(127) % 2 == 0), torch.arange(127), 1000)
            code = torch.where(even.amin(-1) < 1000, even.amin(-1), pick.amin(-1))
            code = (code + 128 * torch.signbit(part if not bad.any() else y)).to(torch.uint8)
        codes[:, i * BLOCK:(i + 1) * BLOCK] = code
        exps[:, i] = torch.where(bad, 255, e).to(torch.uint8)
    return codes.view(x.shape), exps.view(*x.shape[:-1], -1)


def values(codes, exps, held):
    """float64 of held rows: codes as bytes (or the rows themselves) and exponents."""
    if held not in LARGEST:
        return codes.double()
    x = codes.view(torch.int8).double() if held == torch.int8 else E4M3[codes.long()]
    scale = torch.where(exps == 255, math.nan, torch.exp2(exps.double() - 127))
    return x * scale.repeat_interleave(BLOCK, -1)[..., :x.shape[-1]]


def place(tables, b, n, page_size, num_pages):
    """(page, row) of position n of sequence b, or None."""
    i = n // page_size
    if n < 0 or i >= tables.shape[1]:
        return None
    page = int(tables[b, i])
    return (page, n % page_size) if 0 <= page < num_pages else None


def rows(pages, exps, held, tables, b, count):
    """(G, count, D) float64 of the first `count` positions and which of them have a page."""
    num_pages, _, page_size, _ = pages.shape
    n = torch.arange(count)
    index = n // page_size
    page = torch.where(index < tables.shape[1], tables[b, index.clamp_max(max(tables.shape[1] - 1, 0))].long(), -1)
    there = (0 <= page) & (page < num_pages)
    pick = lambda x: x[page.clamp(0, num_pages - 1), :, n % page_size].transpose(0, 1)  # noqa: E731
    x = values(pick(pages), None if exps is None else pick(exps), held)
    return torch.where(there[None, :, None], x, 0.0), there


def attention(q, k_pages, v_pages, k_exp, v_exp, held, tables, lengths, offsets, scale):
    """(out, bound) of q (H, T, D), everything on the CPU, pages of 8 bits as bytes."""
    H, T, D = q.shape
    out, bound = torch.zeros(H, T, D, dtype=torch.float64), torch.zeros(H, T, D, dtype=torch.float64)
    for b, length in enumerate(lengths):
        lo, hi = offsets[b], offsets[b + 1]
        if lo == hi:
            continue
        count = max(0, min(length, tables.shape[1] * k_pages.shape[2]))
        k, there = rows(k_pages, k_exp, held, tables, b, count)
        v, _ = rows(v_pages, v_exp, held, tables, b, count)
        see = softmax.visible(1, hi - lo, count, there[None, :], True, length - (hi - lo))
        one = softmax.attention(q[None, :, lo:hi], k[None], v[None], scale, see)
        out[:, lo:hi], bound[:, lo:hi] = one["out"][0], one["bound"]["out"][0]
    return out, bound
