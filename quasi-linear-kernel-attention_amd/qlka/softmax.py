"""Softmax attention to a sequence of another length, with a learned relative position bias, over libqlka's kernels.

  * softmax_attention(q, k, v, ...): q (B, H, M, D) against keys and values (B, G, N, D) of another length, one key head for
    every H / G query heads, key mask, causal order, position bias; differentiable. One query (a decoder's token) and long
    prompts take kernels of their own.
  * RelativeBuckets and relative_bias(table, M, N, ...): the bias as a map (H, M, N); differentiable.

The additive layers next to it (qlka.layers) are fp32; these take float32 and bfloat16. The reference has torch's
scaled_dot_product_attention in this place (Experiments/kernel_attention/attention.py:99-102) and no position bias.
"""

from functools import lru_cache
from typing import NamedTuple

import torch

from . import _lib

MAX_BUCKETS = 256       # QLKA_MAX_BUCKETS


@lru_cache(maxsize=64)
def _borders(num_buckets, max_distance, bidirectional):
    if bidirectional and num_buckets % 2:
        raise ValueError(f"num_buckets must be even for both sides, got {num_buckets}")
    side = num_buckets // 2 if bidirectional else num_buckets
    if not 1 <= side or num_buckets > MAX_BUCKETS:
        raise ValueError(f"num_buckets must be in [{2 if bidirectional else 1}, {MAX_BUCKETS}], got {num_buckets}")
    single = side // 2
    if side > 1 and not single < max_distance <= 1 << 28:
        raise ValueError(f"max_distance must be in [{single + 1}, 2^28], got {max_distance}")
    found = list(range(1, single + 1))
    steps, d = side - single, single
    for j in range(1, steps if single else 0):
        # the least d with (d / single)^steps >= (max_distance / single)^j, in whole numbers
        need = max_distance ** j * single ** (steps - j)
        hi = max_distance
        while d < hi:
            mid = (d + hi) // 2
            d, hi = (d, mid) if mid ** steps >= need else (mid + 1, hi)
        found.append(d)
    return tuple(found)


class RelativeBuckets(NamedTuple):
    """How key - query distances fall into buckets: half of a side's buckets hold one distance each, from 0 on, the others
    grow with the logarithm up to max_distance, the last one takes all beyond. bidirectional: one half of the buckets for
    keys up to the query, the other for keys after it; else keys after the query are in bucket 0. Borders are found in
    whole numbers, so no rounding moves one."""
    num_buckets: int = 32
    max_distance: int = 128
    bidirectional: bool = True

    @property
    def borders(self):
        """First distance of each bucket of a side but the first."""
        return _borders(int(self.num_buckets), int(self.max_distance), bool(self.bidirectional))


def softmax_attention(q, k, v, scale=None, keep=None, table=None, buckets=None, causal=False, start=0):
    """softmax(scale q k^T + bias) v: q (B, H, M, D), k and v (B, G, N, D), H a multiple of G -> (B, H, M, D).

    float32 or bfloat16, D up to 128, any strides. scale: D ** -0.5 by default; 0 or of a size in [2^-96, 2^96]. keep (B, N):
    nonzero marks the keys to attend to (others are not read). table (num_buckets, H) with buckets (RelativeBuckets): the
    learned position bias table[bucket(n - (m + start)), h], finite or -inf (a bucket that is not attended to). causal: query
    m sees the keys n <= m + start; start is the position of the first query among the keys, of which those past
    the last query are not read (a cache may be longer than its tokens). A row that sees no key gives zeros and has no
    gradient. Differentiable once, backward, in q, k, v and table; results and gradients do not change from run to run."""
    if q.dim() == 4 and scale is None:
        scale = max(q.shape[3], 1) ** -0.5
    border, both = (), False
    if table is not None:
        if buckets is None:
            buckets = RelativeBuckets()
        border, both = buckets.borders, bool(buckets.bidirectional)
        table = table.float().contiguous()
    elif buckets is not None:
        raise ValueError("buckets without a table")
    if keep is not None and keep.dtype not in (torch.bool, torch.uint8):
        keep = keep != 0
    return _lib.torch_ext().softmax_attention(q, k, v, table, keep, 1.0 if scale is None else float(scale), bool(causal),
                                              int(start), border, both)


def relative_bias(table, M, N, buckets=RelativeBuckets(), start=0):
    """The position bias as a map (H, M, N) float32: table[bucket(n - (m + start)), h] of table (num_buckets, H).
    Differentiable in table."""
    return _lib.torch_ext().relative_bias(table.float(), int(M), int(N), int(start), buckets.borders,
                                          bool(buckets.bidirectional))
