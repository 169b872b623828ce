"""A cache of keys and values in pages, in the tokens' own type or in 8 bits, and softmax attention of tokens over it.

  * PagedCache: pages of page_size tokens that sequences take as they grow, in any order. write() puts the heads of new
    tokens at their positions (quantised on the way where 8 bits are held), read() gives whole sequences back, as a
    padded batch.
  * paged_attention(q, cache, ...): new tokens (one for each sequence, chunks of prompts, or both in a batch) over all
    that their sequences hold.

New tokens of a batch lie one after the other, without padding, as in qlka.packed: rows of all sequences, with offsets.
Where each sequence's pages are (tables) and how many tokens it holds with the new ones (lengths) is read on the device:
nothing waits for it, and captured calls may be replayed with other contents. The reference has no decoder.
"""

from typing import NamedTuple, Optional

import torch

from . import _lib

BLOCK = 32              # elements of a row that share a power of two
HELD = (torch.float32, torch.bfloat16, torch.int8, torch.float8_e4m3fn)


class PagedCache(NamedTuple):
    """Pages of keys and values (num_pages, G, page_size, D), and for 8 bits the exponents of their blocks of 32
    elements (num_pages, G, page_size, ceil(D / 32)). new() makes an empty one, of() takes tensors that are there (any
    strides whose rows start at multiples of 16 bytes; of 8 where rows of 8 bits are no multiple of 16). D: a multiple
    of 8 up to 128.

    With int8 and float8_e4m3fn a block's elements are code * 2^(e - 127): the least e in [27, 248] (246) with which the
    largest code (127; 448) reaches the largest element, the nearest codes, ties to the even one. Such values are exact
    in bfloat16. A block that holds an infinity or NaN reads as NaN.

    In every call: tables (B, P) int32, the numbers of each sequence's pages in order; lengths (B) int32, its tokens
    with the new ones; offsets (B + 1) int32, where the new tokens of each one begin among the T rows, or None: one for
    each, T = B.
    Page numbers outside [0, num_pages) are pages that do not exist (-1 pads a row of tables): nothing is written there,
    keys there are not seen, reading gives zeros; so are positions past the end of a row of tables."""
    k: torch.Tensor
    v: torch.Tensor
    k_exp: Optional[torch.Tensor] = None
    v_exp: Optional[torch.Tensor] = None

    @classmethod
    def new(cls, num_pages, page_size, heads, head_dim, dtype=torch.bfloat16, device="cuda"):
        """An empty cache; dtype float32, bfloat16 (that of the tokens), int8 or float8_e4m3fn."""
        if dtype not in HELD:
            raise ValueError(f"dtype must be one of {HELD}, got {dtype}")
        def rows(size, dtype):
            return torch.zeros(num_pages, heads, page_size, size, dtype=dtype, device=device)

        k, v = rows(head_dim, dtype), rows(head_dim, dtype)
        if dtype.itemsize > 1:
            return cls.of(k, v)
        blocks = -(-head_dim // BLOCK)
        return cls.of(k, v, rows(blocks, torch.uint8), rows(blocks, torch.uint8))

    @classmethod
    def of(cls, k, v, k_exp=None, v_exp=None):
        """The cache that tensors are; refuses what is none."""
        _lib.torch_ext().check_pages(k, v, k_exp, v_exp)
        return cls(k, v, k_exp, v_exp)

    @property
    def page_size(self):
        return self.k.shape[2]

    def write(self, k, v, tables, lengths, offsets=None):
        """Puts the new tokens' heads k, v (G, T, D) at their positions: row offsets[b] + i of sequence b is token
        lengths[b] - n + i, n = offsets[b + 1] - offsets[b]. Rows outside every sequence, and what has no page, are left
        out; the rest of the pages stays as it is. No two sequences of a call may write to one place."""
        _lib.torch_ext().paged_write(k, v, *self, tables, lengths, offsets)

    def read(self, tables, lengths, longest, dtype=None):
        """(k, v), each (B, G, longest, D): the first `longest` positions of every sequence, zeros from its length on.
        dtype: that of the pages, or float32 or bfloat16 where they hold 8 bits (bfloat16 by default). For attention
        that takes contiguous keys: softmax_attention with a position bias, or with a gradient."""
        if dtype is None:
            dtype = self.k.dtype if self.k_exp is None else torch.bfloat16
        return _lib.torch_ext().paged_read(*self, tables, lengths, int(longest), dtype)


def paged_attention(q, cache, tables, lengths, offsets=None, longest=0, scale=None):
    """softmax(scale q k^T) v of new tokens q (H, T, D) over what their sequences hold in the cache -> (H, T, D), H a
    multiple of the cache's key heads.

    The tokens' own keys and values have been written before (PagedCache.write with the same tables, lengths and
    offsets); each sees the keys up to its own position. Rows that see none, and rows outside every sequence, give
    zeros. Infinities and NaN that a sequence holds can make any of its new rows NaN, no other sequence's. float32 or
    bfloat16 q; the pages hold that type or 8 bits. longest: the most new tokens of a sequence where the caller knows
    it: it decides which kernels run, and changes no result by more than its rounding. scale: D ** -0.5 by default; 0 or
    of a size in [2^-96, 2^96]. No gradient (a captured graph, several streams and repeated calls give the same
    results)."""
    if q.dim() == 3 and scale is None:
        scale = max(q.shape[2], 1) ** -0.5
    return _lib.torch_ext().paged_attention(q, *cache, tables, lengths, offsets, int(longest),
                                            1.0 if scale is None else float(scale))
