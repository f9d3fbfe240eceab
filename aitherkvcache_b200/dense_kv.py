"""Dense (fp16 / bf16) paged cache: append with the position rotation on the way, and paged attention.

For the layers of a model that stay uncompressed beside the packed ones - the same pages, block tables and slots, 16-bit
keys and values ``[num_blocks, block_size, kv_heads, head_dim]`` in any strides.  The reference leaves such layers to
vLLM's kernels; here they run in ``akv_rotary_kv_append``, ``akv_dense_paged_attn`` and ``akv_dense_prefill_attn``.
"""
from __future__ import annotations

import ctypes
import math
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


class DensePagedAttention:
    """``DensePagedAttention(head_dim, query_heads, kv_heads).forward(query, k_cache, v_cache, block_tables, context_lens)``.

    The 16-bit counterpart of ``TQPagedAttention``: query and caches in one type (fp16 or bf16), head_dim 64, 128 or 256,
    any number of query heads per KV head, any block size, caches in any strides whose rows start on 16-byte boundaries.
    ``sliding_window``: keys a token sees, itself included (0: all).  ``scale`` defaults to 1/sqrt(head_dim).

    A row that sees no key is zero.  Block-table entries outside the pool are clamped to it, and what pages hold behind
    a sequence's end does not matter.  Scratch is allocated per call (stream-ordered, so calls on several streams and
    captured graphs share nothing)."""

    def __init__(self, head_dim: int, num_query_heads: int, num_kv_heads: int, scale: Optional[float] = None,
                 sliding_window: int = 0):
        if head_dim not in (64, 128, 256):
            raise ValueError(f"head_dim must be 64, 128 or 256, got {head_dim}")
        if num_kv_heads <= 0 or num_query_heads <= 0 or num_query_heads % num_kv_heads:
            raise ValueError(f"{num_query_heads} query heads are not a multiple of {num_kv_heads} KV heads")
        if sliding_window < 0:
            raise ValueError(f"sliding_window must not be negative, got {sliding_window}")
        self.head_dim, self.num_query_heads, self.num_kv_heads = head_dim, num_query_heads, num_kv_heads
        self.scale = 1.0 / math.sqrt(head_dim) if scale is None else float(scale)
        self.sliding_window = int(sliding_window)
        self._decode_bytes = _lib.lib().akv_dense_paged_attn_workspace_bytes(num_query_heads, num_kv_heads, head_dim)

    @staticmethod
    def _rows16(x: torch.Tensor) -> bool:
        """Whether every row of a 16-bit [a, b, head_dim] tensor starts on a 16-byte boundary."""
        return (x.stride(2) == 1 and x.stride(0) > 0 and x.stride(1) > 0
                and not (x.data_ptr() & 15 or (x.stride(0) | x.stride(1)) & 7))

    def _params(self, dev, query, k_cache, v_cache, block_tables, seq_lens, num_seqs, out):
        """Argument block of both entry points, and the output."""
        if query.dim() != 3 or query.shape[1] != self.num_query_heads or query.shape[2] != self.head_dim:
            raise ValueError(f"query {tuple(query.shape)} must be [tokens, {self.num_query_heads}, {self.head_dim}]")
        _check_caches(k_cache, v_cache, self.num_kv_heads, self.head_dim)
        if query.dtype not in (torch.float16, torch.bfloat16) or k_cache.dtype != query.dtype:
            raise TypeError(f"query and caches must be fp16 or bf16 alike, got {query.dtype} and {k_cache.dtype}")
        if block_tables.dim() != 2 or block_tables.shape[0] < num_seqs or seq_lens.dim() != 1 or seq_lens.shape[0] < num_seqs:
            raise ValueError(f"block_tables {tuple(block_tables.shape)} / lengths {tuple(seq_lens.shape)} do not cover "
                             f"{num_seqs} sequences")
        if not self._rows16(query):
            query = query.contiguous()
        if block_tables.stride(1) != 1:
            block_tables = block_tables.contiguous()
        if seq_lens.stride(0) != 1:
            seq_lens = seq_lens.contiguous()
        if out is None:
            out = torch.empty_like(query, memory_format=torch.contiguous_format)
        elif out.shape != query.shape or out.dtype != query.dtype or not self._rows16(out):
            raise ValueError(f"out {tuple(out.shape)} {out.dtype} must be {tuple(query.shape)} {query.dtype} with rows on 16-byte "
                             "boundaries")
        code = _lib._FLOAT_CODES[query.dtype]
        p = _lib.DenseAttnParams(
            query.data_ptr(), code, query.stride(0), query.stride(1),
            k_cache.data_ptr(), k_cache.stride(0), k_cache.stride(1), k_cache.stride(2),
            v_cache.data_ptr(), v_cache.stride(0), v_cache.stride(1), v_cache.stride(2),
            block_tables.data_ptr(), _lib.index_code(block_tables), block_tables.stride(0),
            seq_lens.data_ptr(), _lib.index_code(seq_lens), None, 0,
            num_seqs, query.shape[0], self.num_query_heads, self.num_kv_heads, self.head_dim,
            k_cache.shape[1], block_tables.shape[1], k_cache.shape[0], self.scale, self.sliding_window,
            out.data_ptr(), out.stride(0), out.stride(1))
        p.stream = _lib.stream_ptr(dev)
        return p, out, (query, block_tables, seq_lens)

    def forward(self, query: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                context_lens: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """One token per sequence: ``query`` [num_seqs, query_heads, head_dim], the last of each sequence's
        ``context_lens`` [num_seqs] tokens, over ``k_cache`` / ``v_cache`` [blocks, block_size, kv_heads, head_dim] through
        ``block_tables`` [num_seqs, max_blocks].  Returns ``out`` [num_seqs, query_heads, head_dim]."""
        dev = _lib.require_cuda(query, k_cache, v_cache, block_tables, context_lens, out)
        p, out, keep = self._params(dev, query, k_cache, v_cache, block_tables, context_lens, query.shape[0], out)
        ws = torch.empty(self._decode_bytes, dtype=torch.uint8, device=dev)
        p.workspace, p.workspace_bytes = ws.data_ptr(), self._decode_bytes
        _lib.call(dev, "akv_dense_paged_attn", ctypes.byref(p))
        return out

    def prefill(self, query: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                seq_lens: torch.Tensor, query_start_loc: torch.Tensor, out: Optional[torch.Tensor] = None,
                max_seq_len: Optional[int] = None) -> torch.Tensor:
        """Chunks of new tokens: rows ``query_start_loc[s] .. query_start_loc[s + 1]`` of ``query`` [tokens, query_heads,
        head_dim] are the last tokens of sequence s, whose keys and values (counted in ``seq_lens``) are in the cache
        already; each attends causally up to its own position.  Rows behind the last sequence are left as they are in
        ``out`` (zero when ``out`` is allocated here).  Lengths stay on the device: ``max_seq_len``, which
        ``TQPagedAttention.prefill`` sizes its scratch by, is accepted and not needed.

        Chunks run on the tensor cores for head_dim 64 and 128, at most 128 query heads per KV head and block sizes that
        are multiples of 8; other shapes attend token by token through ``forward``'s kernels."""
        dev = _lib.require_cuda(query, k_cache, v_cache, block_tables, seq_lens, query_start_loc, out)
        if query_start_loc.dim() != 1 or query_start_loc.shape[0] < 1:
            raise ValueError(f"query_start_loc {tuple(query_start_loc.shape)} must be [sequences + 1]")
        if query_start_loc.stride(0) != 1:
            query_start_loc = query_start_loc.contiguous()
        qs_code = _lib.index_code(query_start_loc)
        zero_tail = out is None
        p, out, keep = self._params(dev, query, k_cache, v_cache, block_tables, seq_lens, query_start_loc.shape[0] - 1, out)
        if not (self.head_dim <= 128 and self.num_query_heads <= 128 * self.num_kv_heads and k_cache.shape[1] % 8 == 0
                and block_tables.shape[1] > 0):
            if zero_tail:
                out.zero_()
            return self._prefill_by_rows(query, k_cache, v_cache, block_tables, seq_lens, query_start_loc, out)
        nbytes = _lib.lib().akv_dense_prefill_attn_workspace_bytes(p.num_kv_heads, p.head_dim, p.num_blocks, p.block_size, p.num_seqs,
                                                                   p.max_blocks_per_seq)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        p.workspace, p.workspace_bytes = ws.data_ptr(), nbytes
        p.query_start_loc, p.qs_dtype, p.zero_tail = query_start_loc.data_ptr(), qs_code, int(zero_tail)
        _lib.call(dev, "akv_dense_prefill_attn", ctypes.byref(p))
        return out

    ROWS = 2048      # tokens of one call of the single-token kernels

    def _prefill_by_rows(self, query, k_cache, v_cache, block_tables, seq_lens, query_start_loc, out):
        """Every token as a sequence of its own: its context length and its sequence's row of the block tables."""
        n = query.shape[0]
        if n == 0 or query_start_loc.shape[0] < 2:
            return out
        tok = torch.arange(n, device=query.device, dtype=torch.int64)
        ends = query_start_loc[1:].to(torch.int64).contiguous()
        seq = torch.bucketize(tok, ends, right=True)
        there = (seq < ends.shape[0])[:, None, None]
        seq = seq.clamp_(max=ends.shape[0] - 1)
        ctx = (seq_lens.to(torch.int64)[seq] - (ends[seq] - 1 - tok)).clamp_(min=0)
        for lo in range(0, n, self.ROWS):
            hi = min(n, lo + self.ROWS)
            rows = self.forward(query[lo:hi], k_cache, v_cache, block_tables[seq[lo:hi]], ctx[lo:hi])
            out[lo:hi].copy_(torch.where(there[lo:hi], rows, out[lo:hi]))
        return out
