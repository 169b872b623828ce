"""Softmax attention within sequences of different lengths that lie one after the other, over libqlka's kernels.

A batch of prompts or documents needs no padding this way: rows of all sequences are one tensor, and `offsets` says
where each one begins. Next to qlka.softmax (padded batches, attention to another sequence, the position bias) and
qlka.paged (a cache in pages, filled from such rows). The reference pads its documents
(Experiments/text_transformer/pareto.py:46-65).
"""

from . import _lib


def packed_attention(q, k, v, offsets, scale=None, causal=True):
    """softmax(scale q k^T) v within each sequence: q (H, T, D), k and v (G, T, D), H a multiple of G -> (H, T, D).

    offsets (B + 1) int32 on q's device, not decreasing: sequence b is rows offsets[b] to offsets[b + 1], which may be
    none; rows before the first and behind the last one get zeros and have no gradient. causal: a row sees the keys of
    its sequence up to itself, else all of them. float32 or bfloat16, D up to 128, any strides (rows that do not start
    at multiples of 16 bytes are copied). scale: D ** -0.5 by default; 0 or of a size in [2^-96, 2^96]. What one
    sequence holds, infinities and NaN too, changes no other one's results (it can make any row of its own NaN, earlier
    ones too).

    Differentiable once, backward, in q, k and v; results and gradients do not change from run to run. The offsets are
    read on the device: nothing waits for them, and a captured call may be replayed with others (a backward pass too,
    with those of its forward). How rows are shared out goes by T and B: lengths far from their average, and many empty
    sequences, cost time."""
    if q.dim() == 3 and scale is None:
        scale = max(q.shape[2], 1) ** -0.5
    return _lib.torch_ext().packed_attention(q, k, v, offsets, 1.0 if scale is None else float(scale), bool(causal))
