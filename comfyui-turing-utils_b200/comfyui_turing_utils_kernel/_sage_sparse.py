"""Bindings of the block-sparse Sage attention: the choice of key blocks and the
attention over them (tb_select_key_blocks, tb_sparse_attn).  Query blocks are
128 tokens, key blocks 64 tokens (one K scale)."""
from __future__ import annotations

import ctypes

import torch

from ._lib import call, device_major, dtype_code, layout_strides, on_device, raw_stream

QUERY_BLOCK = 128
KEY_BLOCK = 64


def _check(cond, msg):
    if not cond:
        raise RuntimeError(msg)


def _geometry(query, key, query_scale, key_scale, layout):
    """(device, B, Hq, Hk, Lq, Lk, D) after the checks shared by both entry points."""
    device = query.device
    _check(query.is_cuda, "query must be a CUDA tensor")
    _check(key.is_cuda and key.device == device, "key must be a CUDA tensor on the query's device")
    _check(query_scale.is_cuda and key_scale.is_cuda and query_scale.device == device
           and key_scale.device == device,
           "query_scale and key_scale must be CUDA tensors on the query's device")
    _check(query.dtype == torch.int8 and key.dtype == torch.int8, "query and key must be int8")
    _check(query.dim() == 4 and key.dim() == 4, "query and key must be 4D")
    if layout == 0:
        B, Lq, Hq, D = query.shape
        Bk, Lk, Hk, Dk = key.shape
    else:
        B, Hq, Lq, D = query.shape
        Bk, Hk, Lk, Dk = key.shape
    _check(Bk == B and Dk == D, "query and key shapes are incompatible")
    _check(B > 0 and Hq > 0 and Hk > 0 and Lq > 0 and Lk > 0,
           "empty Q/K sequences are not supported")
    _check(Hq % Hk == 0, "num_qo_heads must be divisible by num_kv_heads")
    _check(query_scale.dtype == torch.float32 and key_scale.dtype == torch.float32,
           "scales must be float32")
    _check(query_scale.shape == (B, Hq, (Lq + 63) // 64 * 4), "query_scale shape mismatch")
    _check(key_scale.shape == (B, Hk, (Lk + 63) // 64), "key_scale shape mismatch")
    _check(query.stride(3) == 1 and key.stride(3) == 1,
           "the last Q/K dimension must be contiguous")
    _check(query_scale.is_contiguous() and key_scale.is_contiguous(), "scales must be contiguous")
    return device, B, Hq, Hk, Lq, Lk, D


def _lengths_ptr(key_lengths, B, device):
    if key_lengths is None:
        return None
    _check(key_lengths.is_cuda and key_lengths.device == device
           and key_lengths.dtype == torch.int32 and key_lengths.shape == (B,)
           and key_lengths.is_contiguous(),
           "key_lengths must be a contiguous int32 [B] tensor on the query's device")
    return key_lengths.data_ptr()


def _require_sm100(device):
    _check(device_major(device) == 10,
           "block-sparse Sage attention requires an sm_100 (B200) device for this build")


def select_key_blocks(query, key, query_scale, key_scale, key_lengths, block_policy, layout, keep):
    device, B, Hq, Hk, Lq, Lk, D = _geometry(query, key, query_scale, key_scale, layout)
    _check(D in (64, 128), "the block choice takes head_dim 64 or 128")
    query_blocks, key_blocks = -(-Lq // QUERY_BLOCK), -(-Lk // KEY_BLOCK)
    _check(1 <= keep, "keep must be positive")
    keep = min(int(keep), key_blocks)
    lengths = _lengths_ptr(key_lengths, B, device)
    rows, policy = 0, None
    if block_policy is not None:
        _check(block_policy.is_cuda and block_policy.device == device
               and block_policy.dtype == torch.int8 and block_policy.dim() == 2
               and block_policy.size(0) in (1, query_blocks)
               and block_policy.size(1) == key_blocks and block_policy.is_contiguous(),
               "block_policy must be a contiguous int8 [1 or query blocks, key blocks] tensor on "
               "the query's device")
        rows, policy = block_policy.size(0), block_policy.data_ptr()
    strides = (ctypes.c_int64 * 6)(*layout_strides(query, layout), *layout_strides(key, layout))
    size = ctypes.c_int64(0)
    _require_sm100(device)
    with on_device(device):
        call("tb_select_key_blocks_workspace", B, Hq, Hk, Lq, Lk, D, ctypes.byref(size))
        workspace = torch.empty(size.value, dtype=torch.uint8, device=device)
        out = torch.empty((B, Hq, query_blocks, keep), dtype=torch.int32, device=device)
        call("tb_select_key_blocks", query.data_ptr(), key.data_ptr(), query_scale.data_ptr(),
             key_scale.data_ptr(), lengths, policy, rows, out.data_ptr(), workspace.data_ptr(),
             size.value, B, Hq, Hk, Lq, Lk, D, keep, strides, raw_stream(device))
    return out


def sparse_attn(query, key, value, output, query_scale, key_scale, block_index, key_lengths,
                layout, sm_scale, return_lse, key_mean=None):
    """Writes the attention into output (or a new tensor); returns (output, natural
    log-sum-exp or None), with the scores of key_mean added to the latter."""
    device, B, Hq, Hk, Lq, Lk, D = _geometry(query, key, query_scale, key_scale, layout)
    _check(D == 128, "the sparse attention kernel takes head_dim 128 (pad smaller heads)")
    _check(value.is_cuda and value.device == device and value.shape == key.shape
           and value.dtype in (torch.float16, torch.bfloat16) and value.stride(3) == 1,
           "value must be a float16 or bfloat16 tensor of the key's shape and device with "
           "contiguous channels")
    _check(block_index.is_cuda and block_index.device == device
           and block_index.dtype == torch.int32 and block_index.dim() == 4
           and block_index.shape[:3] == (B, Hq, -(-Lq // QUERY_BLOCK))
           and block_index.size(3) > 0 and block_index.is_contiguous(),
           "block_index must be a contiguous int32 [B, Hq, query blocks, keep] tensor on the "
           "query's device")
    lengths = _lengths_ptr(key_lengths, B, device)
    if output is not None:
        _check(output.is_cuda and output.device == device and output.shape == query.shape
               and output.dtype == value.dtype and output.stride(3) == 1,
               "output must match query's shape and value's dtype")
        _check(all(n == 1 or s > 0 for n, s in zip(output.shape, output.stride())),
               "output must have a place for every element")
    if key_mean is not None:
        _check(key_mean.is_cuda and key_mean.device == device and key_mean.shape == (B, Hk, D)
               and key_mean.dtype in (torch.float16, torch.bfloat16) and key_mean.is_contiguous(),
               "key_mean must be a contiguous float16 or bfloat16 [B, Hk, D] tensor on the "
               "query's device")
    keep = block_index.size(3)
    size = ctypes.c_int64(0)
    _require_sm100(device)
    with on_device(device):
        if output is None:
            output = torch.empty(query.shape, dtype=value.dtype, device=device)
        strides = (ctypes.c_int64 * 12)(
            *layout_strides(query, layout), *layout_strides(key, layout),
            *layout_strides(value, layout), *layout_strides(output, layout))
        call("tb_sparse_attn_workspace", B, Hq, Lq, keep, ctypes.byref(size))
        workspace = lse = None
        if size.value:
            workspace = torch.empty(size.value, dtype=torch.uint8, device=device)
        if return_lse:
            lse = torch.empty((B, Hq, Lq), dtype=torch.float32, device=device)
        call("tb_sparse_attn", query.data_ptr(), key.data_ptr(), value.data_ptr(),
             dtype_code(value), output.data_ptr(), query_scale.data_ptr(), key_scale.data_ptr(),
             block_index.data_ptr(), lengths, None if lse is None else lse.data_ptr(),
             None if workspace is None else workspace.data_ptr(), size.value, B, Hq, Hk, Lq, Lk,
             D, keep, strides, float(sm_scale), raw_stream(device))
        if lse is not None and key_mean is not None:
            call("tb_smoothed_lse", query.data_ptr(), query_scale.data_ptr(), key_mean.data_ptr(),
                 dtype_code(key_mean), lse.data_ptr(), B, Hq, Hk, Lq, D, strides, float(sm_scale),
                 raw_stream(device))
    return output, lse
