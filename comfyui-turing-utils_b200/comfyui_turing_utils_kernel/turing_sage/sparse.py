"""Block-sparse Sage INT8 attention: each block of 128 queries attends to its own
list of 64-key blocks.

    select_key_blocks             lists from a cheap score of INT8 Q/K
    sparse_sageattn_prequantized  attention over given lists
    sparse_sageattn               quantize, choose, attend
    sparse_sageattn_from_prequantized
                                  choose and attend for codes of prequantize_sageattn
                                  or of the fused RMSNorm + RoPE prologue

Not causal, as the reference's sparse path; a block-causal order is a
block_policy of -1.  Forward only, as every INT8 attention here.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from .. import _sage_sparse as _sparse
from .core import PrequantizedSageAttention, _on_input_device, prequantize_sageattn


def _layout_id(tensor_layout: str) -> int:
    if tensor_layout not in {"HND", "NHD"}:
        raise ValueError(f"Unsupported tensor_layout: {tensor_layout}")
    return 0 if tensor_layout == "NHD" else 1


def _unit_rows(t: torch.Tensor) -> torch.Tensor:
    """t with contiguous channels, a copy only where they are not."""
    return t if t.dim() != 4 or t.stride(-1) == 1 else t.contiguous()


def select_key_blocks(q_int8: torch.Tensor, q_scale: torch.Tensor, k_int8: torch.Tensor,
                      k_scale: torch.Tensor, keep: int, *, tensor_layout: str = "HND",
                      key_lengths: Optional[torch.Tensor] = None,
                      block_policy: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The key blocks each query block attends to: int32 [B, Hq, ceil(Lq / 128),
    min(keep, ceil(Lk / 64))], ascending, -1 where fewer blocks can be chosen.

    The score of a query block and a key block is the product of their mean
    dequantized query and key; the `keep` highest are taken, ties to the lowest
    block, a NaN score last.  The mean query is held to 2^-40 of its largest
    channel, all else is exact up to three fp64 roundings; a query block with a scale
    that is not finite scores 0 everywhere, a key block with one comes last.  Positive sm_scale, K smoothing and
    the Hadamard rotation change no rank beyond INT8 rounding.

    q_int8 / k_int8 and scales: as the Sage quantizers return them (head_dim 64 or
    128, at most 1572864 keys).  key_lengths: int32 [B], keys from there on are
    padding.  block_policy: int8 [1 or query blocks, key blocks], -1 never
    chosen, 0 by score, 1 before any score (text tokens, a local window).
    """
    return _sparse.select_key_blocks(
        _unit_rows(q_int8), _unit_rows(k_int8), q_scale.contiguous(), k_scale.contiguous(),
        None if key_lengths is None else key_lengths.contiguous(),
        None if block_policy is None else block_policy.contiguous(), _layout_id(tensor_layout),
        keep)


def sparse_sageattn_prequantized(q_int8: torch.Tensor, q_scale: torch.Tensor,
                                 k_int8: torch.Tensor, k_scale: torch.Tensor, v: torch.Tensor,
                                 block_index: torch.Tensor, *, tensor_layout: str = "HND",
                                 sm_scale: Optional[float] = None,
                                 key_lengths: Optional[torch.Tensor] = None,
                                 return_lse: bool = False,
                                 output: Optional[torch.Tensor] = None,
                                 key_mean: Optional[torch.Tensor] = None):
    """Softmax attention of each query block over the key blocks its list names.

    q_int8, k_int8: head_dim 128 (pad smaller heads); v: float16 or bfloat16 of
    K's shape.  block_index: int32 [B, Hq, ceil(Lq / 128), keep] in any order;
    entries that name no block with visible keys are skipped, a block named twice
    counts twice.  key_lengths: int32 [B], keys from there on are not seen,
    whatever K and V hold there.  A row that sees no key is 0 (lse -inf).  lse:
    natural logarithm, float32 [B, Hq, Lq], of the scores of the codes; for codes of
    a smoothed K give key_mean, the [B, Hk, 128] mean taken off, and it is that of the
    scores against K itself.  output: written in place of a new
    tensor; it must not overlap the inputs.  sm_scale and the scales may have
    either sign.
    """
    if q_int8.ndim != 4:
        raise ValueError("prequantized Sage Q/K/V must be four-dimensional")
    scale = float(sm_scale) if sm_scale is not None else q_int8.size(-1) ** -0.5
    if not math.isfinite(scale):
        raise ValueError("sm_scale must be finite")
    output, lse = _sparse.sparse_attn(
        _unit_rows(q_int8), _unit_rows(k_int8), _unit_rows(v), output, q_scale.contiguous(),
        k_scale.contiguous(), block_index.contiguous(),
        None if key_lengths is None else key_lengths.contiguous(), _layout_id(tensor_layout),
        scale, return_lse, None if key_mean is None else key_mean.contiguous())
    return (output, lse) if return_lse else output


def sparse_sageattn_from_prequantized(quantized: PrequantizedSageAttention, keep: int, *,
                                      key_lengths: Optional[torch.Tensor] = None,
                                      block_policy: Optional[torch.Tensor] = None,
                                      return_lse: bool = False):
    """select_key_blocks, then the attention over its lists, for the codes of
    prequantize_sageattn or prequantize_sageattn_from_qk.  The lse counts the mean
    that smoothing took off K; for codes made with stabilize_k, whose anchor is not
    kept, it is refused."""
    if quantized.is_causal:
        raise ValueError("causal masking is supported only by dense attention")
    if quantized.sm_scale < 0.0:  # would turn the choice around
        raise ValueError("sm_scale must not be negative where key blocks are chosen")
    if return_lse and quantized.key_anchored:
        raise ValueError("return_lse needs codes made without stabilize_k")
    lists = select_key_blocks(
        quantized.query_int8, quantized.query_scale, quantized.key_int8, quantized.key_scale,
        keep, tensor_layout=quantized.tensor_layout, key_lengths=key_lengths,
        block_policy=block_policy)
    result = sparse_sageattn_prequantized(
        quantized.query_int8, quantized.query_scale, quantized.key_int8, quantized.key_scale,
        quantized.value, lists, tensor_layout=quantized.tensor_layout,
        sm_scale=quantized.sm_scale, key_lengths=key_lengths, return_lse=return_lse,
        key_mean=quantized.key_mean)
    output, lse = result if return_lse else (result, None)
    output = output[..., :quantized.original_head_dim]
    return (output, lse) if return_lse else output


@_on_input_device
def sparse_sageattn(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, keep: int, *,
                    tensor_layout: str = "HND", sm_scale: Optional[float] = None,
                    smooth_k: bool = False, key_lengths: Optional[torch.Tensor] = None,
                    block_policy: Optional[torch.Tensor] = None, return_lse: bool = False):
    """sageattn over the `keep` key blocks of 64 tokens that score highest for each
    block of 128 queries (head_dim up to 128, not causal).  Padding keys past
    key_lengths must be finite: they share a quantization block with real ones."""
    quantized = prequantize_sageattn.__wrapped__(q, k, v, tensor_layout=tensor_layout,
                                                 is_causal=False, sm_scale=sm_scale,
                                                 smooth_k=smooth_k)
    return sparse_sageattn_from_prequantized(quantized, keep, key_lengths=key_lengths,
                                             block_policy=block_policy, return_lse=return_lse)
