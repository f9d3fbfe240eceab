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


_HALVES = {torch.float16: _lib.AKV_F16, torch.bfloat16: _lib.AKV_BF16}
_pack_append = _lib.packer(_lib.RotaryAppendParams)
_pack_attn = _lib.packer(_lib.DenseAttnParams)


def _check_caches(k_cache: torch.Tensor, v_cache: torch.Tensor, kv_heads: int, head_dim: int):
    """(shape, strides of the keys, strides of the values) of two caches that belong together."""
    shape, ks, vs = k_cache.shape, k_cache.stride(), v_cache.stride()
    if (len(shape) != 4 or shape != v_cache.shape or shape[2] != kv_heads or shape[3] != head_dim or ks[3] != 1 or vs[3] != 1):
        raise ValueError(f"caches {tuple(shape)} / {tuple(v_cache.shape)} must both be [blocks, block_size, {kv_heads}, "
                         f"{head_dim}] with a contiguous last dimension")
    if k_cache.dtype != v_cache.dtype:
        raise TypeError(f"caches must have one dtype, got {k_cache.dtype} and {v_cache.dtype}")
    return shape, ks, vs


def rotary_kv_append(query: Optional[torch.Tensor], key: torch.Tensor, value: torch.Tensor, positions: torch.Tensor,
                     slot_mapping: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, rope: RotaryPositions,
                     query_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Rotate ``query`` and ``key`` [tokens, heads, head_dim] to ``positions`` and write the rotated keys and the values
    to slot ``slot_mapping[token]`` (= block * block_size + position) of the caches, in one launch.  Returns the rotated
    query in the caches' dtype (None for ``query=None``).

    Tokens with a negative slot, or one behind the cache, are skipped (padding).  The slots of one call must be distinct.
    ``query_out`` may be the query itself when their dtypes agree."""
    index = _lib.cuda_index(key, query, value, positions, slot_mapping, k_cache, v_cache, query_out, rope.steps)
    tokens = key.shape[0]
    key = rope._heads(key, "key", tokens)
    shape, ks, vs = _check_caches(k_cache, v_cache, key.shape[1], key.shape[2])
    if value.shape != key.shape or value.dtype != key.dtype:
        raise ValueError(f"value {tuple(value.shape)} {value.dtype} must match key {tuple(key.shape)} {key.dtype}")
    st = value.stride()
    if st[2] != 1:
        value = value.contiguous()
        st = value.stride()
    if slot_mapping.dim() != 1 or slot_mapping.shape[0] != tokens:
        raise ValueError(f"slot_mapping {tuple(slot_mapping.shape)} must be [{tokens}]")
    if tokens and not (shape[0] and shape[1]):
        raise ValueError(f"caches {tuple(shape)} hold no slot")
    if slot_mapping.stride(0) != 1:
        slot_mapping = slot_mapping.contiguous()
    if query is not None:
        query = rope._heads(query, "query", tokens)
        if query.dtype != key.dtype:
            raise TypeError(f"query and key must have one dtype, got {query.dtype} and {key.dtype}")
        query_out = rope._out(query_out, query, k_cache.dtype, "query_out")
    else:
        query_out = None
    _lib.call(index, "akv_rotary_kv_append", _pack_append(
        *rope._values(query, key, positions, query_out, None, _lib.float_code(k_cache), 0, index),
        value.data_ptr(), st[0], st[1], slot_mapping.data_ptr(), _lib.index_code(slot_mapping),
        k_cache.data_ptr(), ks[0], ks[1], ks[2], v_cache.data_ptr(), vs[0], vs[1], vs[2], shape[1], shape[0]))
    return query_out


def kv_append(key: torch.Tensor, value: torch.Tensor, slot_mapping: torch.Tensor, k_cache: torch.Tensor,
              v_cache: torch.Tensor) -> None:
    """``rotary_kv_append`` of keys that carry their rotation already (or need none): ``key`` and ``value`` [tokens, heads,
    head_dim] go to their slots as they are, converted to the caches' dtype."""
    index = _lib.cuda_index(key, value, slot_mapping, k_cache, v_cache)
    if key.dim() != 3 or value.shape != key.shape or value.dtype != key.dtype:
        raise ValueError(f"key {tuple(key.shape)} {key.dtype} and value {tuple(value.shape)} {value.dtype} must be one [tokens, heads, "
                         "head_dim]")
    tokens, heads, head_dim = key.shape
    shape, ks, vs = _check_caches(k_cache, v_cache, heads, head_dim)
    key, value = (x if x.stride(2) == 1 else x.contiguous() for x in (key, value))
    if slot_mapping.dim() != 1 or slot_mapping.shape[0] != tokens:
        raise ValueError(f"slot_mapping {tuple(slot_mapping.shape)} must be [{tokens}]")
    if tokens and not (shape[0] and shape[1]):
        raise ValueError(f"caches {tuple(shape)} hold no slot")
    slot_mapping = slot_mapping.contiguous()
    tables = _lib.RotaryTables(head_dim, 0, 1, 0, None, None, 1.0)      # nothing is rotated
    k, v = key.stride(), value.stride()
    _lib.call(index, "akv_rotary_kv_append", _pack_append(
        ctypes.addressof(tables), 0, 0, 0, 0, tokens, _lib.float_code(key), _lib.float_code(k_cache), 0, 0, 0, 0, 0, 0, 0,
        key.data_ptr(), k[0], k[1], heads, 0, 0, 0, 0, _lib.raw_stream(index),
        value.data_ptr(), v[0], v[1], slot_mapping.data_ptr(), _lib.index_code(slot_mapping),
        k_cache.data_ptr(), ks[0], ks[1], ks[2], v_cache.data_ptr(), vs[0], vs[1], vs[2], shape[1], shape[0]))


class DensePagedAttention:
    """``DensePagedAttention(head_dim, query_heads, kv_heads).forward(query, k_cache, v_cache, block_tables, context_lens)``.

    The 16-bit counterpart of ``TQPagedAttention``: query and caches in one type (fp16 or bf16), head_dim 64, 128 or 256,
    any number of query heads per KV head, any block size, caches in any strides whose rows start on 16-byte boundaries.
    ``sliding_window``: keys a token sees, itself included (0: all).  ``scale`` defaults to 1/sqrt(head_dim).

    A row that sees no key is zero.  Block-table entries outside the pool are clamped to it, and what pages hold behind
    a sequence's end or before all windows does not matter.  ``out`` overlaps no input.  Scratch is allocated per call (stream-ordered, so calls on several streams and
    captured graphs share nothing)."""

    def __init__(self, head_dim: int, num_query_heads: int, num_kv_heads: int, scale: Optional[float] = None,
                 sliding_window: int = 0):
        if head_dim not in (64, 128, 256):
            raise ValueError(f"head_dim must be 64, 128 or 256, got {head_dim}")
        if num_kv_heads <= 0 or num_query_heads <= 0 or num_query_heads % num_kv_heads:
            raise ValueError(f"{num_query_heads} query heads are not a multiple of {num_kv_heads} KV heads")
        if scale is not None and not (0.0 < scale < math.inf):
            raise ValueError(f"scale must be positive and finite, got {scale}")
        if sliding_window < 0:
            raise ValueError(f"sliding_window must not be negative, got {sliding_window}")
        self.head_dim, self.num_query_heads, self.num_kv_heads = head_dim, num_query_heads, num_kv_heads
        self.scale = 1.0 / math.sqrt(head_dim) if scale is None else float(scale)
        self.sliding_window = min(int(sliding_window), 0x7fffffff)
        self._decode_bytes = _lib.lib().akv_dense_paged_attn_workspace_bytes(num_query_heads, num_kv_heads, head_dim)

    @staticmethod
    def _rows16(x: torch.Tensor) -> bool:
        """Whether every row of a 16-bit [a, b, head_dim] tensor starts on a 16-byte boundary (the stride of a dimension of
        one element is never used)."""
        n, s = x.shape, x.stride()
        a, b = s[0] if n[0] > 1 else 8, s[1] if n[1] > 1 else 8
        return s[2] == 1 and a > 0 and b > 0 and not (x.data_ptr() & 15 or (a | b) & 7)

    def _values(self, query, k_cache, v_cache, block_tables, seq_lens, starts, num_seqs, out):
        """(fields of ``akv_dense_attn_params`` up to the output, the output, tensors that must outlive the call)."""
        qshape = query.shape
        if len(qshape) != 3 or qshape[1] != self.num_query_heads or qshape[2] != self.head_dim:
            raise ValueError(f"query {tuple(qshape)} must be [tokens, {self.num_query_heads}, {self.head_dim}]")
        shape, ks, vs = _check_caches(k_cache, v_cache, self.num_kv_heads, self.head_dim)
        dtype = query.dtype
        if dtype not in _HALVES or k_cache.dtype != dtype:
            raise TypeError(f"query and caches must be fp16 or bf16 alike, got {dtype} and {k_cache.dtype}")
        tshape = block_tables.shape
        if len(tshape) != 2 or tshape[0] < num_seqs or seq_lens.dim() != 1 or seq_lens.shape[0] < num_seqs:
            raise ValueError(f"block_tables {tuple(tshape)} / lengths {tuple(seq_lens.shape)} do not cover {num_seqs} sequences")
        if not self._rows16(query):      # clone: contiguous() leaves a tensor at an odd offset where it is
            query = query.clone(memory_format=torch.contiguous_format)
        if block_tables.stride(1) != 1:
            block_tables = block_tables.contiguous()
        if seq_lens.stride(0) != 1:
            seq_lens = seq_lens.contiguous()
        if out is None:
            out = torch.empty_like(query)
        elif out.shape != qshape or out.dtype != dtype or not self._rows16(out):
            raise ValueError(f"out {tuple(out.shape)} {out.dtype} must be {tuple(qshape)} {dtype} with rows on 16-byte boundaries")
        qs, os = query.stride(), out.stride()
        return (query.data_ptr(), _HALVES[dtype], qs[0], qs[1], k_cache.data_ptr(), ks[0], ks[1], ks[2],
                v_cache.data_ptr(), vs[0], vs[1], vs[2], block_tables.data_ptr(), _lib.index_code(block_tables), block_tables.stride(0),
                seq_lens.data_ptr(), _lib.index_code(seq_lens), *starts, num_seqs, qshape[0], self.num_query_heads, self.num_kv_heads,
                self.head_dim, shape[1], tshape[1], shape[0], self.scale, self.sliding_window,
                out.data_ptr(), os[0], os[1]), out, (query, block_tables, seq_lens)

    def forward(self, query: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                context_lens: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """One token per sequence: ``query`` [num_seqs, query_heads, head_dim], the last of each sequence's
        ``context_lens`` [num_seqs] tokens, over ``k_cache`` / ``v_cache`` [blocks, block_size, kv_heads, head_dim] through
        ``block_tables`` [num_seqs, max_blocks].  Returns ``out`` [num_seqs, query_heads, head_dim]."""
        index = _lib.cuda_index(query, k_cache, v_cache, block_tables, context_lens, out)
        values, out, keep = self._values(query, k_cache, v_cache, block_tables, context_lens, (0, 0), query.shape[0], out)
        ws = out.new_empty((self._decode_bytes + 1) // 2)      # half the host time of torch.empty
        _lib.call(index, "akv_dense_paged_attn", _pack_attn(*values, 0, ws.data_ptr(), self._decode_bytes, _lib.raw_stream(index)))
        return out

    def prefill(self, query: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                seq_lens: torch.Tensor, query_start_loc: torch.Tensor, out: Optional[torch.Tensor] = None,
                max_seq_len: Optional[int] = None) -> torch.Tensor:
        """Chunks of new tokens: rows ``query_start_loc[s] .. query_start_loc[s + 1]`` of ``query`` [tokens, query_heads,
        head_dim] are the last tokens of sequence s, whose keys and values (counted in ``seq_lens``) are in the cache
        already; each attends causally up to its own position.  Rows before the first sequence and behind the last are left as
        they are in ``out`` (zero when ``out`` is allocated here).  A value that is not finite, of a key that some of a
        chunk's tokens see, may reach the chunk's earlier tokens too.  Lengths stay on the device: ``max_seq_len``, which
        ``TQPagedAttention.prefill`` sizes its scratch by, is accepted and not needed.

        Chunks run on the tensor cores for head_dim 64 and 128, at most 128 query heads per KV head and block sizes that
        are multiples of 8; other shapes attend token by token through ``forward``'s kernels."""
        index = _lib.cuda_index(query, k_cache, v_cache, block_tables, seq_lens, query_start_loc, out)
        if query_start_loc.dim() != 1 or query_start_loc.shape[0] < 1:
            raise ValueError(f"query_start_loc {tuple(query_start_loc.shape)} must be [sequences + 1]")
        if query_start_loc.stride(0) != 1:
            query_start_loc = query_start_loc.contiguous()
        num_seqs, zero_tail = query_start_loc.shape[0] - 1, out is None
        values, out, keep = self._values(query, k_cache, v_cache, block_tables, seq_lens,
                                         (query_start_loc.data_ptr(), _lib.index_code(query_start_loc)), num_seqs, out)
        blocks, block_size, width = k_cache.shape[0], k_cache.shape[1], block_tables.shape[1]
        if not (self.head_dim <= 128 and self.num_query_heads <= 128 * self.num_kv_heads and block_size % 8 == 0 and width > 0):
            if zero_tail:
                out.zero_()
            return self._prefill_by_rows(query, k_cache, v_cache, block_tables, seq_lens, query_start_loc, out)
        nbytes = _lib.lib().akv_dense_prefill_attn_call_bytes(query.shape[0], self.num_query_heads, self.num_kv_heads, self.head_dim,
                                                              blocks, block_size, num_seqs, width)
        ws = out.new_empty((nbytes + 1) // 2)
        _lib.call(index, "akv_dense_prefill_attn", _pack_attn(*values, int(zero_tail), ws.data_ptr(), nbytes, _lib.raw_stream(index)))
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
        there = ((seq < ends.shape[0]) & (tok >= query_start_loc[0]))[:, None, None]
        seq = seq.clamp_(max=ends.shape[0] - 1)
        lens = seq_lens.to(torch.int64).clamp(0, block_tables.shape[1] * k_cache.shape[1])
        ctx = (lens[seq] - (ends[seq] - 1 - tok)).clamp_(min=0)
        for lo in range(0, n, self.ROWS):
            hi = min(n, lo + self.ROWS)
            rows = self.forward(query[lo:hi], k_cache, v_cache, block_tables[seq[lo:hi]], ctx[lo:hi])
            out[lo:hi].copy_(torch.where(there[lo:hi], rows, out[lo:hi]))
        return out
