"""Rotary positions, the paged append and paged attention over 16-bit pages in 64 bits (torch, any device): loops over
sequences and heads, written from the definitions."""
from __future__ import annotations

import math

import torch


def rotate(x, positions, freq, axis, rotary_dim, adjacent, scaling=1.0, inverse=False):
    """x [tokens, heads, dim]; positions [axes, tokens]; freq / axis per pair.  Returns float64."""
    y = x.double().clone()
    for p, (f, a) in enumerate(zip(freq, axis)):
        i, j = (2 * p, 2 * p + 1) if adjacent else (p, rotary_dim // 2 + p)
        t = positions[a].double() * f * (-1.0 if inverse else 1.0)
        c, s = torch.cos(t)[:, None], torch.sin(t)[:, None]
        x0, x1 = x[..., i].double(), x[..., j].double()
        y[..., i] = scaling * (x0 * c - x1 * s)
        y[..., j] = scaling * (x1 * c + x0 * s)
    return y


def rotate_bound(x, y, rotary_dim, adjacent, out_dtype, scaling=1.0):
    """Largest error that the 32-bit rotation may have against ``rotate``, per element.

    The angle, as a fraction of half a turn in [-1, 1], is rounded to float32 once (2^-25 of half a turn, pi * 2^-25 rad)
    after cutting the 64-bit fraction to 32 bits (2^-32 turns); sincospif is good to 2 ulp (2^-23 of at most 1); the two
    products, the sum and the scaling of c and s round three times (3 * 2^-24 of |x0| + |x1|).  Then one rounding to the output's type (half a step; the smallest step
    of fp16 is 2^-24)."""
    per_pair = math.pi * 2.0 ** -25 + 2 * math.pi * 2.0 ** -32 + 2.0 ** -23 + 3 * 2.0 ** -24
    mag = x.double().abs()
    both = torch.zeros_like(mag)
    if rotary_dim:
        r = rotary_dim
        if adjacent:
            pair = mag[..., 0:r:2] + mag[..., 1:r:2]
            both[..., 0:r:2], both[..., 1:r:2] = pair, pair
        else:
            pair = mag[..., :r // 2] + mag[..., r // 2:r]
            both[..., :r // 2], both[..., r // 2:r] = pair, pair
    err = abs(scaling) * both * per_pair
    return err + (y.abs() + err) * (torch.finfo(out_dtype).eps / 2) + 2.0 ** -25


def attention(q, k_cache, v_cache, block_tables, seq_lens, starts, scale, window=0):
    """Chunk attention: token i of sequence s (rows starts[s] .. of q) sees keys j <= p, j > p - window (if window), with
    p = seq_lens[s] - new + i; a row that sees nothing is zero.  Rows behind the last sequence: zero.  Float64.

    Returns (out, bound): the largest error that float32 scores, sums and accumulators and 16-bit probabilities may have.
    A score is off by at most d = scale (D 2^-23 + 2^-22) sum|q k| (D accumulations of exact products, each off by a last
    place; scaling, and the subtraction of the reference), its weight by the factor e^d and 2^-21 of the
    exponential; the weight is rounded once to the type (half a step u, and for fp16 at most 2^-25 where it is
    subnormal; the largest weight is at least 1); numerator and denominator are float32 sums of n terms (n 2^-23).  With
    A = sum w|v| / sum w that is at most (2 d + 2 * 2^-21 + u + 2 n 2^-23) A + n 2^-25 max|v|, then u |out| for the result."""
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    bs, kvh, dim = k_cache.shape[1], k_cache.shape[2], q.shape[2]
    group = q.shape[1] // kvh
    u = torch.finfo(q.dtype).eps / 2
    for s in range(len(seq_lens)):
        lo, hi, total = int(starts[s]), int(starts[s + 1]), int(seq_lens[s])
        if hi <= lo or total <= 0:
            continue
        pages = block_tables[s, :-(-total // bs)].long()
        k = k_cache[pages].flatten(0, 1)[:total].double()
        v = v_cache[pages].flatten(0, 1)[:total].double()
        p = torch.arange(total - (hi - lo), total, device=q.device)[:, None]
        j = torch.arange(total, device=q.device)[None]
        seen = j <= p
        if window:
            seen &= j > p - window
        for h in range(q.shape[1]):
            qh, kh, vh = q[lo:hi, h].double(), k[:, h // group], v[:, h // group]
            sc = (scale * (qh @ kh.t())).masked_fill(~seen, -math.inf)
            top = sc.amax(1, keepdim=True)
            e = torch.exp(sc - torch.where(top == -math.inf, torch.zeros_like(top), top))
            tot = e.sum(1, keepdim=True)
            some = tot > 0
            w = torch.where(some, e / tot.clamp_min(1e-300), torch.zeros_like(e))
            o = w @ vh
            d = abs(scale) * (dim * 2.0 ** -23 + 2.0 ** -22) * (qh.abs() @ kh.abs().t()).masked_fill(~seen, 0).amax(1, keepdim=True)
            n = seen.sum(1, keepdim=True).double()
            vmax = vh.abs().max()
            err = (2 * d + 2.0 ** -20 + u + n * 2.0 ** -22) * (w @ vh.abs()) + n * 2.0 ** -25 * vmax
            out[lo:hi, h] = o
            bound[lo:hi, h] = torch.where(some, err + u * (o.abs() + err) + 2.0 ** -25, torch.zeros_like(err))
    return out, bound
