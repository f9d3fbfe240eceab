"""Rotary positions with one or several axes.

A vector's pair p turns by ``position[axis(p)] * frequency(p)``.  With one axis this is the usual rotary embedding; with
several (time, height, width of image and video tokens) each pair follows one of the token's positions.  The rotation
runs in ``akv_rotary``; ``rotary_kv_append`` (dense_kv.py) applies it while it writes keys and values to a paged cache.
The reference has no rotation of its own: its callers hand it rotated keys, and its spectral codec wants unrotated ones
(``inverse=True`` takes a rotation back).
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Sequence, Tuple

import torch

from . import _lib

MAX_AXES = 4
_pack = _lib.packer(_lib.RotaryParams)


def axis_of_pairs(pairs: int, sections: Optional[Sequence[int]], layout: str = "blocked") -> list:
    """Axis of every pair.  ``sections[a]`` pairs belong to axis a: "blocked" gives the first ``sections[0]`` pairs to axis
    0, the next ``sections[1]`` to axis 1 and so on; "cycled" lets the axes take turns until each has its share."""
    if layout not in ("blocked", "cycled"):
        raise ValueError(f"section_layout must be 'blocked' or 'cycled', got {layout!r}")
    if sections is None:
        return [0] * pairs
    left = [int(n) for n in sections]
    if not 1 <= len(left) <= MAX_AXES or min(left) < 0 or sum(left) != pairs:
        raise ValueError(f"sections {tuple(sections)} must be 1 to {MAX_AXES} counts that add up to {pairs} pairs")
    if layout == "blocked":
        return [a for a, n in enumerate(left) for _ in range(n)]
    axes, a = [], 0
    while len(axes) < pairs:
        if left[a % len(left)] > 0:
            left[a % len(left)] -= 1
            axes.append(a % len(left))
        a += 1
    return axes


class RotaryPositions:
    """``q, k = RotaryPositions(128, base=1e6).forward(query, key, positions)``.

    head_dim        elements of a vector; ``rotary_dim`` of them (default all, even) are rotated, the rest pass through
    base, inv_freq  frequency of pair p: ``base ** (-2 p / rotary_dim)``, or the ``rotary_dim / 2`` values given
    sections        pairs of every axis (``None``: one axis); ``section_layout``: see ``axis_of_pairs``
    pair_layout     "halves": pair p is elements (p, p + rotary_dim / 2); "adjacent": elements (2 p, 2 p + 1)
    scaling         factor of the rotated elements (the attention factor of scaled rotary embeddings)
    """

    def __init__(self, head_dim: int, rotary_dim: Optional[int] = None, base: float = 10000.0,
                 sections: Optional[Sequence[int]] = None, section_layout: str = "blocked", pair_layout: str = "halves",
                 inv_freq=None, scaling: float = 1.0, device: str = "cuda"):
        self.head_dim = int(head_dim)
        self.rotary_dim = self.head_dim if rotary_dim is None else int(rotary_dim)
        if self.head_dim <= 0 or not 0 < self.rotary_dim <= self.head_dim or self.rotary_dim % 2:
            raise ValueError(f"rotary_dim must be even and in (0, head_dim], got {self.rotary_dim} of {self.head_dim}")
        if pair_layout not in ("halves", "adjacent"):
            raise ValueError(f"pair_layout must be 'halves' or 'adjacent', got {pair_layout!r}")
        pairs = self.rotary_dim // 2
        axes = axis_of_pairs(pairs, sections, section_layout)
        self.num_axes = 1 if sections is None else len(sections)
        self.pair_layout, self.section_layout = pair_layout, section_layout
        self.sections = None if sections is None else tuple(int(n) for n in sections)
        self.scaling = float(scaling)
        if inv_freq is None:
            freq = [float(base) ** (-2.0 * p / self.rotary_dim) for p in range(pairs)]
        else:
            freq = [float(f) for f in (inv_freq.tolist() if isinstance(inv_freq, torch.Tensor) else inv_freq)]
            if len(freq) != pairs:
                raise ValueError(f"inv_freq must have {pairs} values, got {len(freq)}")
        if not all(math.isfinite(f) for f in freq) or not math.isfinite(self.scaling):
            raise ValueError("frequencies and scaling must be finite")
        # a frequency as a 64-bit fraction of a turn (radians / 2 pi * 2^64 modulo 2^64), kept as a signed 64-bit word
        turns = [int(f / (2.0 * math.pi) * 2.0 ** 64) % (1 << 64) for f in freq]
        self.inv_freq = torch.tensor(freq, dtype=torch.float64)
        self.steps = torch.tensor([t - (1 << 64) if t >= 1 << 63 else t for t in turns], dtype=torch.int64, device=device)
        self.axes = torch.tensor(axes, dtype=torch.int32, device=device)
        self._bind()

    def _bind(self) -> None:
        """The argument block that points at the tables."""
        self.device = self.steps.device
        self._tables = _lib.RotaryTables(self.head_dim, self.rotary_dim, self.num_axes, int(self.pair_layout == "adjacent"),
                                         self.steps.data_ptr(), self.axes.data_ptr(), self.scaling)
        self._tables_at = ctypes.addressof(self._tables)

    def __getstate__(self) -> dict:      # copies and pickles: addresses stay behind
        return {k: v for k, v in vars(self).items() if k not in ("_tables", "_tables_at")}

    def __setstate__(self, state: dict) -> None:
        vars(self).update(state)
        self._bind()

    def _positions(self, positions: torch.Tensor, tokens: int) -> Tuple[int, int]:
        """(stride over the axes, stride over the tokens) of [tokens] or [num_axes, tokens]."""
        shape = positions.shape
        if len(shape) == 1 and shape[0] == tokens:
            return 0, positions.stride(0)      # text: the same position on every axis
        if len(shape) == 2 and shape[0] == self.num_axes and shape[1] == tokens:
            return positions.stride()
        raise ValueError(f"positions {tuple(shape)} must be [{tokens}] or [{self.num_axes}, {tokens}]")

    def _heads(self, x: torch.Tensor, name: str, tokens: int) -> torch.Tensor:
        shape = x.shape
        if len(shape) != 3 or shape[2] != self.head_dim or shape[0] != tokens:
            raise ValueError(f"{name} {tuple(shape)} must be [{tokens}, heads, {self.head_dim}]")
        return x if x.stride(2) == 1 else x.contiguous()

    @staticmethod
    def _out(out, x, dtype, name):
        if out is None:
            return torch.empty_like(x) if x.dtype == dtype else torch.empty_like(x, dtype=dtype)
        if out.shape != x.shape or out.stride(2) != 1 or out.dtype != dtype:
            raise ValueError(f"{name} {tuple(out.shape)} {out.dtype} must be {tuple(x.shape)} {dtype} with a contiguous last "
                             "dimension")
        return out

    def _values(self, query, key, positions, query_out, key_out, out_dtype, inverse, index):
        """Fields of ``akv_rotary_params``: what the rotation and the append share.  Tensors are checked."""
        tokens = (query if query is not None else key).shape[0]
        pos_axis, pos_tok = self._positions(positions, tokens)
        none = (0, 0, 0, 0), (0, 0, 0)
        q, qo, k, ko = *none, *none
        if query is not None:
            st = query.stride()
            q, st = (query.data_ptr(), st[0], st[1], query.shape[1]), query_out.stride()
            qo = (query_out.data_ptr(), st[0], st[1])
        if key is not None:
            st = key.stride()
            k = (key.data_ptr(), st[0], st[1], key.shape[1])
            if key_out is not None:
                st = key_out.stride()
                ko = (key_out.data_ptr(), st[0], st[1])
        return (self._tables_at, positions.data_ptr(), _lib.index_code(positions), pos_axis, pos_tok, tokens,
                _lib.float_code(query if query is not None else key), out_dtype, *q, *qo, *k, *ko, inverse, _lib.raw_stream(index))

    def forward(self, query: Optional[torch.Tensor], key: Optional[torch.Tensor], positions: torch.Tensor,
                query_out: Optional[torch.Tensor] = None, key_out: Optional[torch.Tensor] = None,
                inverse: bool = False) -> Tuple[Optional[torch.Tensor], Optional[torch.Tensor]]:
        """``query`` [tokens, query_heads, head_dim] and ``key`` [tokens, kv_heads, head_dim] (either may be None, any
        strides with a contiguous last dimension) turned to ``positions``: [tokens] or [num_axes, tokens], int32 or int64.
        Returns (query, key) in their dtype.  ``query_out=query`` works in place.  ``inverse`` turns by the negative angles:
        the rotation taken back at scaling 1, and its gradient at any scaling."""
        if query is None and key is None:
            raise ValueError("query and key are both None")
        index = _lib.cuda_index(query, key, positions, query_out, key_out, self.steps)
        tokens = (query if query is not None else key).shape[0]
        if query is not None:
            query = self._heads(query, "query", tokens)
            query_out = self._out(query_out, query, query.dtype, "query_out")
        else:
            query_out = None
        if key is not None:
            key = self._heads(key, "key", tokens)
            if query is not None and key.dtype != query.dtype:
                raise TypeError(f"query and key must have one dtype, got {query.dtype} and {key.dtype}")
            key_out = self._out(key_out, key, key.dtype, "key_out")
        else:
            key_out = None
        code = _lib.float_code(query if query is not None else key)
        _lib.call(index, "akv_rotary", _pack(*self._values(query, key, positions, query_out, key_out, code, int(inverse), index)))
        return query_out, key_out

    __call__ = forward
