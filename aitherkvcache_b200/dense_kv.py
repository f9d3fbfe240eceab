"""Dense (fp16 / bf16) paged cache: append with the position rotation on the way, and paged attention.

For the layers of a model that stay uncompressed beside the packed ones - the same pages, block tables and slots, 16-bit
keys and values ``[num_blocks, block_size, kv_heads, head_dim]`` in any strides.  The reference leaves such layers to
vLLM's kernels; here they run in ``akv_rotary_kv_append``, ``akv_dense_paged_attn`` and ``akv_dense_prefill_attn``.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _lib
from .rotary import RotaryPositions


def _check_caches(k_cache: torch.Tensor, v_cache: torch.Tensor, kv_heads: int, head_dim: int) -> None:
    if (k_cache.dim() != 4 or k_cache.shape != v_cache.shape or k_cache.shape[2] != kv_heads or k_cache.shape[3] != head_dim
            or k_cache.stride(3) != 1 or v_cache.stride(3) != 1):
        raise ValueError(f"caches {tuple(k_cache.shape)} / {tuple(v_cache.shape)} must both be [blocks, block_size, {kv_heads}, "
                         f"{head_dim}] with a contiguous last dimension")
    if k_cache.dtype != v_cache.dtype:
        raise TypeError(f"caches must have one dtype, got {k_cache.dtype} and {v_cache.dtype}")


def rotary_kv_append(query: Optional[torch.Tensor], key: torch.Tensor, value: torch.Tensor, positions: torch.Tensor,
                     slot_mapping: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, rope: RotaryPositions,
                     query_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Rotate ``query`` and ``key`` [tokens, heads, head_dim] to ``positions`` and write the rotated keys and the values
    to slot ``slot_mapping[token]`` (= block * block_size + position) of the caches, in one launch.  Returns the rotated
    query in the caches' dtype (None for ``query=None``).

    Tokens with a negative slot, or one behind the cache, are skipped (padding).  The slots of one call must be distinct.
    ``query_out`` may be the query itself when their dtypes agree."""
    dev = _lib.require_cuda(query, key, value, positions, slot_mapping, k_cache, v_cache, query_out, rope.steps)
    p = _lib.RotaryAppendParams()
    r, query, key = rope._params(query, key, positions, False, dev)
    tokens, kv_heads, head_dim = key.shape
    _check_caches(k_cache, v_cache, kv_heads, head_dim)
    if value.shape != key.shape or value.dtype != key.dtype:
        raise ValueError(f"value {tuple(value.shape)} {value.dtype} must match key {tuple(key.shape)} {key.dtype}")
    if value.stride(2) != 1:
        value = value.contiguous()
    if slot_mapping.dim() != 1 or slot_mapping.shape[0] != tokens:
        raise ValueError(f"slot_mapping {tuple(slot_mapping.shape)} must be [{tokens}]")
    if slot_mapping.stride(0) != 1:
        slot_mapping = slot_mapping.contiguous()
    r.out_dtype = _lib.float_code(k_cache)
    if query is not None:
        query_out = RotaryPositions._out(query_out, query, k_cache.dtype, "query_out", dev)
        r.q_out, r.qo_stride_tok, r.qo_stride_head = query_out.data_ptr(), query_out.stride(0), query_out.stride(1)
    else:
        query_out = None
    p.rotary = r
    p.value, p.v_stride_tok, p.v_stride_head = value.data_ptr(), value.stride(0), value.stride(1)
    p.slot_mapping, p.slot_dtype = slot_mapping.data_ptr(), _lib.index_code(slot_mapping)
    p.k_cache, p.kc_stride_blk, p.kc_stride_pos, p.kc_stride_head = k_cache.data_ptr(), k_cache.stride(0), k_cache.stride(1), k_cache.stride(2)
    p.v_cache, p.vc_stride_blk, p.vc_stride_pos, p.vc_stride_head = v_cache.data_ptr(), v_cache.stride(0), v_cache.stride(1), v_cache.stride(2)
    p.block_size, p.num_blocks = k_cache.shape[1], k_cache.shape[0]
    if tokens and not (k_cache.shape[0] and k_cache.shape[1]):
        raise ValueError(f"caches {tuple(k_cache.shape)} hold no slot")
    _lib.call(dev, "akv_rotary_kv_append", ctypes.byref(p))
    return query_out
