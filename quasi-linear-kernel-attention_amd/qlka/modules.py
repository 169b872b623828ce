"""Model-level integration: kernel attention for the experiment models, over the fused additive layers.

The reference's experiments (Experiments/kernel_attention) reach the weighted abs / Laplace sums through three
entries, provided here with the same names and arguments:

  * attention(q, k, v, kernel, tau, keep=None, impl="efficient") (attention.py:95-126), on (B, H, S, D) fp32
    tensors; keep (B, S) marks the real keys. The additive kernels (add_laplace, add_riesz, add_bump) run as one
    fused libqlka call each (qlka.layers); "softmax" is scaled dot-product attention with scale tau**-2
    (attention.py:99-102). TAU holds the default temperatures (kernels.py:13-25).
  * KernelMultiheadAttention(embed_dim, num_heads, kernel, tau, impl) (vision_transformer.py:19-44): self-attention
    whose state_dict is nn.MultiheadAttention's (in_proj_weight, in_proj_bias, out_proj), so trained weights load. With
    the "softmax" kernel it also attends to another sequence (context), to earlier positions alone (causal) and with a
    learned relative position bias (position_bias, a RelativePositionBias), on the kernels of qlka.softmax; to sequences
    of different lengths without padding (offsets), on those of qlka.packed; and to a cache in pages (cache), on those
    of qlka.paged. The last two, like the bias, run on the GPU alone; the others fall back to torch on the CPU.
  * use_kernel_attention(model, kernel, tau, impl) and KernelAttention(config, kernel, tau, impl) (nomic.py:9-40):
    kernel attention inside a HF NomicBertModel with its own weights.

The nomic integration goes through transformers' attention-function registry instead of replacing modules: the
registry entry "qlka" is an attention function (q, k, v after the layer's projections and rotary embedding, in
(B, H, S, D)) that reads the kernel from the calling attention module, and the model's attention implementation is
switched to it. The layers keep their own NomicBertAttention objects and parameters; the key mask is the boolean
SDPA-style mask the model builds for "sdpa" (the same mask builder is registered for "qlka").
"""

import copy

import torch
import torch.nn as nn
import torch.nn.functional as F

from . import layers, packed, paged, softmax

TAU = {"softmax": 64 ** 0.25, "add_laplace": 0.5, "add_riesz": 1.0, "add_bump": 1.5}   # kernels.py:13-25
KERNELS = tuple(TAU)
IMPLS = ("naive", "efficient")


def _softmax(q, k, v, tau, keep):
    mask = None if keep is None else keep.bool()[:, None, None, :]
    return F.scaled_dot_product_attention(q, k, v, attn_mask=mask, scale=tau ** -2)


def attention(q, k, v, kernel, tau, keep=None, impl="efficient"):
    """Kernel attention of (B, H, S, D) fp32 q, k, v; keep (B, S), nonzero = real key, or None."""
    assert q.dtype == k.dtype == v.dtype == torch.float32, "kernel attention runs in fp32 only"
    assert impl in IMPLS, f"impl must be one of {IMPLS}"
    if kernel == "softmax":
        return _softmax(q, k, v, tau, keep)
    if kernel not in layers.LAYERS:
        raise NotImplementedError(f"kernel {kernel!r} does not run on the weighted abs / Laplace sums; "
                                  f"available: {sorted(KERNELS)}")
    if impl == "naive":
        raise NotImplementedError("impl='naive' (the dense kernel matrix) is not part of this package; "
                                  "use impl='efficient'")
    return layers.attention(q, k, v, kernel, tau, keep)


def _resolve_tau(kernel, tau):
    if tau is not None:
        return float(tau)
    if kernel not in TAU:
        raise NotImplementedError(f"kernel {kernel!r} has no default temperature; available: {sorted(KERNELS)}")
    return TAU[kernel]


# --------------------------------------------------------------------------------------------- vision transformer
class RelativePositionBias(nn.Module):
    """A learned position bias for each head and bucket of key - query distance: weight (num_buckets, num_heads).
    forward(M, N, start) is the bias as a map (num_heads, M, N), for M queries from position start on and N keys."""

    def __init__(self, num_heads, num_buckets=32, max_distance=128, bidirectional=True):
        super().__init__()
        self.buckets = softmax.RelativeBuckets(num_buckets, max_distance, bidirectional)
        self.buckets.borders                             # refuses what has no buckets
        self.weight = nn.Parameter(torch.zeros(num_buckets, num_heads))

    def forward(self, M, N, start=0):
        return softmax.relative_bias(self.weight, M, N, self.buckets, start=start)


class KernelMultiheadAttention(nn.Module):
    """x (B, S, E) -> (B, S, E) attention with a chosen kernel. Parameters and their initialisation follow
    nn.MultiheadAttention (packed q/k/v input projection, output projection), so its state_dict loads both ways; a
    position_bias (RelativePositionBias, "softmax" only) adds its own parameter.

    forward(x, keep): self-attention. With the "softmax" kernel also
      * forward(x, keep, context): attention to context (B, N, E), a sequence of another length, or to its heads as
        project_context(context) gives them, which a decoder computes once and passes at every token; keep (B, N) marks
        context's real positions;
      * causal=True: the query at position start + m sees the keys up to its own position. For a decoder's next tokens,
        context holds the heads of all tokens up to them and start is the position of x's first one (without a context,
        where the keys are x's own, there is no other position than 0);
      * forward(x, offsets=offsets): x (T, E) on the GPU, sequences one after the other (qlka.packed), each attending to
        itself (causal or not) -> (T, E);
      * forward(x, cache=(pages, tables, lengths), offsets=offsets): x (T, E), the new tokens of sequences whose heads a
        qlka.paged.PagedCache of num_heads key heads holds, one each without offsets. Their own heads are written there,
        then each attends to its sequence up to itself. No gradient (call it under torch.no_grad())."""

    def __init__(self, embed_dim, num_heads, kernel="softmax", tau=None, impl="efficient", position_bias=None):
        super().__init__()
        if embed_dim % num_heads:
            raise ValueError(f"embed_dim {embed_dim} is not a multiple of num_heads {num_heads}")
        if position_bias is not None and kernel != "softmax":
            raise NotImplementedError(f"a position bias runs on the 'softmax' kernel, not on {kernel!r}")
        self.num_heads = num_heads
        self.kernel, self.tau, self.impl = kernel, _resolve_tau(kernel, tau), impl
        self.in_proj_weight = nn.Parameter(nn.init.xavier_uniform_(torch.empty(3 * embed_dim, embed_dim)))
        self.in_proj_bias = nn.Parameter(torch.zeros(3 * embed_dim))
        self.out_proj = nn.Linear(embed_dim, embed_dim)
        nn.init.xavier_uniform_(self.out_proj.weight)
        nn.init.zeros_(self.out_proj.bias)
        self.position_bias = position_bias

    def _heads(self, x, first, count):
        """`count` of the packed projections of x from the first-th on, as (B, H, S, E / H) tensors."""
        E = self.out_proj.in_features
        part = slice(first * E, (first + count) * E)
        packed = F.linear(x, self.in_proj_weight[part], self.in_proj_bias[part])    # [q | k | v] along the last dim
        per_head = packed.unflatten(-1, (count, self.num_heads, -1))                 # (B, S, count, H, Dh)
        return per_head.permute(2, 0, 3, 1, 4).unbind(0)

    def split_heads(self, x):
        """The packed projection of x as three (B, H, S, E / H) tensors q, k, v."""
        return self._heads(x, 0, 3)

    def project_context(self, context):
        """The heads (k, v) of context (B, N, E), each (B, H, N, E / H), as forward takes them."""
        return self._heads(context, 1, 2)

    def _rows(self, x, offsets, cache, causal):
        """forward of rows (T, E) without padding."""
        if self.kernel != "softmax" or self.position_bias is not None:
            raise NotImplementedError("packed sequences and a cache in pages run on the 'softmax' kernel without a "
                                      "position bias")
        if x.dim() != 2:
            raise ValueError(f"packed rows must be (T, E), got {tuple(x.shape)}")
        q, k, v = (heads[0] for heads in self.split_heads(x[None]))                 # (H, T, Dh)
        if cache is None:
            heads = packed.packed_attention(q, k, v, offsets, scale=self.tau ** -2, causal=causal)
        else:
            pages, tables, lengths = cache
            pages.write(k, v, tables, lengths, offsets)
            heads = paged.paged_attention(q, pages, tables, lengths, offsets, scale=self.tau ** -2)
        return self.out_proj(heads.transpose(0, 1).flatten(1))

    def forward(self, x, keep=None, context=None, causal=False, start=0, offsets=None, cache=None):
        if offsets is not None or cache is not None:
            if keep is not None or context is not None or start != 0:
                raise ValueError("packed sequences and a cache in pages take no keep, context or start")
            return self._rows(x, offsets, cache, causal)
        if context is None:
            if start != 0:
                raise ValueError(f"start {start} without a context: the keys are x's own, whose first position is 0")
            q, k, v = self.split_heads(x)
            if self.position_bias is None and not causal:
                heads = attention(q, k, v, self.kernel, self.tau, keep, self.impl)  # (B, H, S, Dh)
                return self.out_proj(heads.transpose(1, 2).flatten(2))
        else:
            q, = self._heads(x, 0, 1)
            k, v = context if isinstance(context, (tuple, list)) else self.project_context(context)
        if self.kernel != "softmax":
            raise NotImplementedError(f"attention to a context, causal order and a position bias run on the 'softmax' kernel, "
                                      f"not on {self.kernel!r}")
        heads = _softmax_to(q, k, v, self.tau, keep, self.position_bias, causal, start)
        return self.out_proj(heads.transpose(1, 2).flatten(2))


def _softmax_to(q, k, v, tau, keep, position_bias, causal, start):
    """Softmax attention of q to k, v of another length: qlka.softmax on the GPU, torch's own on the CPU (no bias there)."""
    table = buckets = None
    if position_bias is not None:
        table, buckets = position_bias.weight, position_bias.buckets
    if q.is_cuda or position_bias is not None:
        return softmax.softmax_attention(q, k, v, scale=tau ** -2, keep=keep, table=table, buckets=buckets, causal=causal,
                                         start=start)
    mask = None if keep is None else keep.bool()[:, None, None, :]
    if causal:
        past = (torch.arange(k.shape[2])[None, :] <= torch.arange(q.shape[2])[:, None] + start)
        mask = past if mask is None else mask & past
    return F.scaled_dot_product_attention(q, k, v, attn_mask=mask, scale=tau ** -2)


# ---------------------------------------------------------------------------------------------------- nomic-bert
REGISTRY_NAME = "qlka"
_registered = False


def _hf_attention(module, query, key, value, attention_mask, scaling=None, dropout=0.0, **kwargs):
    """transformers attention function: (B, H, S, D) states of one layer -> ((B, S, H, D) output, None). The kernel
    is the one use_kernel_attention / KernelAttention attached to the layer's attention module."""
    kernel, tau, impl = module.qlka_kernel
    keep = None
    if attention_mask is not None:
        if attention_mask.dtype != torch.bool:
            raise TypeError("kernel attention expects the boolean key mask of the sdpa mask builder")
        keep = attention_mask[:, 0, 0, :]            # every query row of the bidirectional mask holds the key mask
    out = attention(query.contiguous(), key.contiguous(), value.contiguous(), kernel, tau, keep, impl)
    return out.transpose(1, 2), None


def register():
    """Register the "qlka" attention function (and the sdpa boolean-mask builder under the same name) with
    transformers. Idempotent."""
    global _registered
    if _registered:
        return REGISTRY_NAME
    from transformers import AttentionInterface
    from transformers.masking_utils import AttentionMaskInterface, sdpa_mask
    AttentionInterface.register(REGISTRY_NAME, _hf_attention)
    AttentionMaskInterface.register(REGISTRY_NAME, sdpa_mask)
    _registered = True
    return REGISTRY_NAME


def _tag(attn, kernel, tau, impl):
    if impl not in IMPLS:
        raise ValueError(f"impl must be one of {IMPLS}")
    attn.qlka_kernel = (kernel, _resolve_tau(kernel, tau), impl)
    attn.kernel, attn.tau, attn.impl = attn.qlka_kernel


def _encoder(model):
    """The NomicBertModel of a model: the model itself, or the auto_model of a SentenceTransformer's first module."""
    if hasattr(model, "layers"):
        return model
    return model[0].auto_model


def use_kernel_attention(model, kernel, tau=None, impl="efficient"):
    """Run every attention layer of a NomicBertModel (or a SentenceTransformer wrapping one) with `kernel`, in place;
    every parameter stays where it is. Returns the model."""
    name = register()
    enc = _encoder(model)
    for layer in enc.layers:
        _tag(layer.self_attn, kernel, tau, impl)
    enc.set_attn_implementation(name)
    return model


def KernelAttention(config, kernel="softmax", tau=None, impl="efficient"):
    """A NomicBertAttention for `config` (same parameters: q_proj, k_proj, v_proj, o_proj) that runs `kernel`; its
    config is a copy with the attention implementation set to the registered kernel attention."""
    from transformers.models.nomic_bert.modeling_nomic_bert import NomicBertAttention
    cfg = copy.copy(config)
    cfg._attn_implementation = register()
    attn = NomicBertAttention(cfg)
    _tag(attn, kernel, tau, impl)
    return attn
