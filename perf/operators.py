"""Cases, plain forms and exact values of the dense paged cache's operators: rotary positions with one or several axes,
the append of keys and values with that rotation on the way, and attention over 16-bit pages for single tokens and for
chunks of new tokens.

``own`` false: elementary torch operations in 32 bits (angles in 64).  ``own`` true: the package's calls.
"""
import math
import random

import torch

own = False

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"fp16": 2, "bf16": 2, "fp32": 4}


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def _rotary(name, tokens, heads, kv_heads, dim, rotary_dim, dtype, sections, layout, pairs, inverse, far, base):
    return {"name": name, "kind": "rotary", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "rotary_dim": rotary_dim, "dtype": dtype, "sections": sections, "layout": layout, "pairs": pairs,
            "inverse": inverse, "far": far, "base": base}


def _append(name, tokens, heads, kv_heads, dim, dtype, sections, layout, block, padding, fused_qkv, far, base):
    return {"name": name, "kind": "append", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "rotary_dim": dim, "dtype": dtype, "sections": sections, "layout": layout, "pairs": "halves", "block": block,
            "padding": padding, "fused_qkv": fused_qkv, "far": far, "base": base}


def _attention(name, kind, seqs, heads, kv_heads, dim, dtype, block, window, past, new, lens_seed):
    """``past`` and ``new``: ranges "lo:hi" of the cached tokens before the call's and of the call's own per sequence."""
    return {"name": name, "kind": kind, "seqs": seqs, "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype,
            "block": block, "window": window, "past": past, "new": new, "lens_seed": lens_seed}


def listed():
    return [
        # the rotation of one decode step of 16 sequences: latency
        _rotary("rotary step", 16, 32, 8, 128, 128, "fp16", "", "blocked", "halves", False, 32768, 1e6),
        # a chunk of image / video tokens with time, height and width positions
        _rotary("rotary video chunk", 8192, 32, 8, 128, 128, "bf16", "16,24,24", "blocked", "halves", False, 100000, 1e6),
        # keys of an existing cache turned back to position zero for the spectral codec: partial rotation, neighbouring
        # pairs, odd counts, 32 bits, far positions
        _rotary("rotary inverse far", 4099, 9, 3, 96, 64, "fp32", "12,10,10", "cycled", "adjacent", True, 1000000, 1e4),
        # one decode step's append: 16 sequences, one token each
        _append("append step", 16, 32, 8, 128, "fp16", "", "blocked", 16, 0.0, False, 32768, 1e6),
        # the prefill write of 16 sequences with 2048 new tokens each
        _append("append prompts", 32768, 32, 8, 128, "fp16", "", "blocked", 16, 0.0, True, 32768, 1e6),
        # a padded multimodal batch out of a fused projection, small heads
        _append("append padded video", 5003, 14, 2, 64, "bf16", "12,10,10", "cycled", 32, 0.1, True, 100000, 1e6),
        # one short conversation: latency
        _attention("decode one short", "decode", 1, 32, 8, 128, "fp16", 16, 0, "499:499", "1:1", 1),
        # the batch of the headline benchmark, kept in 16 bits
        _attention("decode batch", "decode", 16, 32, 8, 128, "fp16", 16, 0, "4095:32767", "1:1", 1),
        # many sequences of a windowed layer with small heads
        _attention("decode windowed", "decode", 200, 64, 8, 64, "bf16", 16, 1024, "0:2500", "1:1", 2),
        # a chunk behind a long context
        _attention("chunk behind 30000", "chunk", 1, 32, 8, 128, "fp16", 16, 0, "30000:30000", "2048:2048", 1),
        # fresh prompts of a ragged batch
        _attention("ragged prompts", "chunk", 12, 32, 8, 128, "bf16", 16, 0, "0:0", "1:2000", 3),
        # a few drafted tokens per sequence to be verified, small heads, seven query heads per key head
        _attention("drafted tokens", "chunk", 32, 28, 4, 64, "bf16", 32, 0, "100:8000", "1:8", 4),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def _sections(rng, pairs):
    if rng.random() < 0.4:
        return ""
    third = pairs // 3
    h = rng.randint(max(1, third - 4), third)
    return "%d,%d,%d" % (pairs - 2 * h, h, h)


def draw(rng):
    kind = rng.choice(("rotary", "append", "decode", "decode", "chunk", "chunk"))
    kv = rng.choice((1, 2, 3, 4, 8))
    group = rng.choice((1, 2, 3, 4, 5, 7, 8))
    dim = rng.choice((64, 128))
    dtype = rng.choice(("fp16", "bf16"))
    block = rng.choice((16, 32, 64))
    if kind == "rotary":
        dim = rng.choice((64, 96, 128, 256))
        rd = rng.choice((dim, dim, dim // 2))
        c = _rotary("", _log(rng, 1, 8192), kv * group, kv, dim, rd, rng.choice(("fp16", "bf16", "fp32")), _sections(rng, rd // 2),
                    rng.choice(("blocked", "cycled")), rng.choice(("halves", "adjacent")), rng.random() < 0.3,
                    _log(rng, 1000, 1000000), rng.choice((1e4, 5e5, 1e6)))
    elif kind == "append":
        c = _append("", _log(rng, 1, 16384), kv * group, kv, dim, dtype, _sections(rng, dim // 2), rng.choice(("blocked", "cycled")),
                    block, rng.choice((0.0, 0.1)), rng.random() < 0.5, _log(rng, 1000, 1000000), rng.choice((1e4, 5e5, 1e6)))
    else:
        window = rng.choice((0, 0, 0, _log(rng, 100, 4000)))
        if kind == "decode":
            seqs = _log(rng, 1, 128)
            past = _log(rng, 1, 200000 // seqs)
            c = _attention("", kind, seqs, kv * group, kv, dim, dtype, block, window, "%d:%d" % (rng.randint(0, past), past), "1:1",
                           rng.randint(1, 10 ** 6))
        else:
            seqs = _log(rng, 1, 24)
            new = _log(rng, 1, 4000 // seqs)
            past = _log(rng, 1, 24000 // seqs)
            c = _attention("", kind, seqs, kv * group, kv, dim, dtype, block, window, "%d:%d" % (rng.randint(0, past), past),
                           "%d:%d" % (rng.randint(1, new), new), rng.randint(1, 10 ** 6))
    del c["name"]
    return c


def _lengths(case):
    """(new tokens, tokens with the new ones) of every sequence."""
    r = random.Random(case["lens_seed"])
    (p0, p1), (n0, n1) = ([int(x) for x in case[k].split(":")] for k in ("past", "new"))
    new = [r.randint(n0, n1) for _ in range(case["seqs"])]
    return new, [r.randint(p0, p1) + n for n in new]


def work(case):
    b = BYTES[case["dtype"]]
    if case["kind"] in ("rotary", "append"):
        axes = len(case["sections"].split(",")) if case["sections"] else 1
        n, turned = case["tokens"], case["tokens"] * (case["heads"] + case["kv_heads"])
        moved = turned + (n * case["kv_heads"] if case["kind"] == "append" else 0)
        return {"bytes": 2 * moved * case["dim"] * b + 8 * n * axes + (8 * n if case["kind"] == "append" else 0),
                "flops": 3 * turned * case["rotary_dim"]}
    new, total = _lengths(case)
    w, pairs, keys = case["window"], 0, 0
    for n, t in zip(new, total):
        if w:
            pairs += sum(min(w, t - n + 1 + i) for i in range(n))
            keys += min(t, n + w - 1)
        else:
            pairs += n * (t - n) + n * (n + 1) // 2
            keys += t
    return {"bytes": b * case["dim"] * (2 * keys * case["kv_heads"] + 2 * sum(new) * case["heads"]) + 4 * keys / case["block"],
            "flops": 4 * pairs * case["heads"] * case["dim"]}


# ---------------------------------------------------------------------------------------------------------------------
# states
# ---------------------------------------------------------------------------------------------------------------------
def _axes(case):
    """Number of axes and the axis of every pair."""
    pairs = case["rotary_dim"] // 2
    if not case["sections"]:
        return 1, [0] * pairs
    left = [int(x) for x in case["sections"].split(",")]
    if case["layout"] == "blocked":
        return len(left), [a for a, n in enumerate(left) for _ in range(n)]
    axes, a = [], 0
    while len(axes) < pairs:      # the axes take turns until each has its share
        if left[a % len(left)] > 0:
            left[a % len(left)] -= 1
            axes.append(a % len(left))
        a += 1
    return len(left), axes


def _positions(case, axes, g, dev):
    n = case["tokens"]
    if axes == 1:
        if n <= 64:      # a decode step: every token at a place of its own
            return torch.randint(0, case["far"], (n,), generator=g, device=dev)
        return torch.arange(n, device=dev) + torch.randint(0, max(1, case["far"] - n), (1,), generator=g, device=dev)
    start = torch.randint(0, case["far"], (1,), generator=g, device=dev)
    at = torch.arange(n, device=dev)
    return torch.stack([start + at // 576, start + at // 24 % 24, start + at % 24])[:axes].contiguous()


def _random(shape, dtype, g, dev):
    return torch.randn(shape, generator=g, device=dev, dtype=torch.float32).to(TYPES[dtype])


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dim, qh, kvh, dt = case["dim"], case["heads"], case["kv_heads"], case["dtype"]
    s = {"case": case}
    if case["kind"] in ("rotary", "append"):
        n = case["tokens"]
        axes, axis = _axes(case)
        s["positions"] = _positions(case, axes, g, dev)
        s["axis"] = torch.tensor(axis, device=dev)
        s["freq"] = case["base"] ** (-torch.arange(0, case["rotary_dim"], 2, dtype=torch.float64, device=dev) / case["rotary_dim"])
        if case.get("fused_qkv"):      # views of one projection's output
            qkv = _random((n, qh + 2 * kvh, dim), dt, g, dev)
            s["q"], s["k"], s["v"] = qkv[:, :qh], qkv[:, qh:qh + kvh], qkv[:, qh + kvh:]
        else:
            s["q"], s["k"] = _random((n, qh, dim), dt, g, dev), _random((n, kvh, dim), dt, g, dev)
            s["v"] = _random((n, kvh, dim), dt, g, dev) if case["kind"] == "append" else None
        if case["kind"] == "append":
            blocks = -(-n // case["block"]) + 3
            s["k_cache"] = _random((blocks, case["block"], kvh, dim), dt, g, dev)
            s["v_cache"] = _random((blocks, case["block"], kvh, dim), dt, g, dev)
            order = torch.randperm(blocks, generator=g, device=dev)      # blocks in any order, positions inside them in turn
            at = torch.arange(n, device=dev)
            slots = order[at // case["block"]] * case["block"] + at % case["block"]
            if case["padding"]:
                slots = torch.where(torch.rand(n, generator=g, device=dev) < case["padding"], -1, slots)
            s["slots"] = slots
        if own:
            from aitherkvcache_b200 import RotaryPositions
            sections = tuple(int(x) for x in case["sections"].split(",")) if case["sections"] else None
            s["rope"] = RotaryPositions(dim, rotary_dim=case["rotary_dim"], base=case["base"], sections=sections,
                                        section_layout=case["layout"], pair_layout=case["pairs"], device="cuda")
        return s
    new, total = _lengths(case)
    bs, seqs = case["block"], case["seqs"]
    need = [-(-t // bs) for t in total]
    blocks = sum(need) + 2
    order = torch.randperm(blocks, generator=g, device=dev).to(torch.int32)
    width, used, at = max(need), [], 0
    for c in need:
        used += [min(at + i, at + c - 1) for i in range(width)]      # the row's rest repeats its last block
        at += c
    s["block_tables"] = order[torch.tensor(used, device=dev)].view(seqs, width).contiguous()
    s["lens"] = torch.tensor(total, dtype=torch.int32, device=dev)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    s["starts"] = torch.tensor(starts, dtype=torch.int32, device=dev)
    s["max_new"], s["max_len"] = max(new), max(total)      # known on the host, as a scheduler knows them
    s["q"] = _random((starts[-1], qh, dim), dt, g, dev)
    s["k_cache"] = _random((blocks, bs, kvh, dim), dt, g, dev)
    s["v_cache"] = _random((blocks, bs, kvh, dim), dt, g, dev)
    if own:
        from aitherkvcache_b200 import DensePagedAttention
        s["attn"] = DensePagedAttention(dim, qh, kvh, sliding_window=case["window"])
    return s


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def _turn(x, cos, sin, case):
    """x [tokens, heads, dim] turned by the angles of cos / sin [tokens, rotary_dim / 2], in 32 bits."""
    r = case["rotary_dim"]
    f = x.float()
    c, s = cos[:, None], sin[:, None]
    if case["pairs"] == "halves":
        a, b = f[..., :r // 2], f[..., r // 2:r]
        y = torch.cat([a * c - b * s, b * c + a * s], dim=-1)
    else:
        a, b = f[..., 0:r:2], f[..., 1:r:2]
        y = torch.stack([a * c - b * s, b * c + a * s], dim=-1).flatten(-2)
    return torch.cat([y, f[..., r:]], dim=-1).to(x.dtype)


def _cos_sin(s, case):
    p = s["positions"] if s["positions"].dim() == 2 else s["positions"][None]
    angle = p[s["axis"]].t().double() * s["freq"]
    if case.get("inverse"):
        angle = -angle
    return angle.cos().float(), angle.sin().float()


def _plain_attention(s, case):
    q, lens, starts, bt = s["q"], s["lens"].long(), s["starts"].long(), s["block_tables"].long()
    seqs, mq, length = lens.numel(), s["max_new"], s["max_len"]
    kvh, dim = case["kv_heads"], case["dim"]
    group = case["heads"] // kvh
    new = starts[1:] - starts[:-1]
    i = torch.arange(mq, device=q.device)
    rows = (starts[:-1, None] + i).clamp(max=q.shape[0] - 1)
    qp = q[rows].float().view(seqs, mq, kvh, group, dim).permute(0, 2, 1, 3, 4).reshape(seqs, kvh, mq * group, dim)
    j = torch.arange(length, device=q.device)
    inside = (j[None] < lens[:, None])[:, None, :, None]
    k = s["k_cache"][bt].flatten(1, 2)[:, :length].float().transpose(1, 2)
    v = s["v_cache"][bt].flatten(1, 2)[:, :length].float().transpose(1, 2)
    v = torch.where(inside, v, 0.0)
    scores = torch.matmul(qp, k.transpose(-1, -2)).view(seqs, kvh, mq, group, length) * (1.0 / math.sqrt(dim))
    at = (lens - new)[:, None] + i      # position of every query token
    seen = (j <= at[..., None]) & (i < new[:, None])[..., None]
    if case["window"]:
        seen &= j > at[..., None] - case["window"]
    scores = scores.masked_fill(~seen[:, None, :, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top.isinf(), 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(seqs, kvh, mq * group, length), v).view(seqs, kvh, mq, group, dim)
    o = torch.where(total > 0, o / total, 0.0).permute(0, 2, 1, 3, 4).reshape(seqs, mq, case["heads"], dim)
    t = torch.arange(q.shape[0], device=q.device)
    seq = torch.bucketize(t, starts[1:], right=True)
    return o[seq, t - starts[seq]].to(q.dtype)


def run(s):
    case = s["case"]
    if own:
        if case["kind"] == "rotary":
            return s["rope"].forward(s["q"], s["k"], s["positions"], inverse=case["inverse"])
        if case["kind"] == "append":
            from aitherkvcache_b200 import rotary_kv_append
            q = rotary_kv_append(s["q"], s["k"], s["v"], s["positions"], s["slots"], s["k_cache"], s["v_cache"], s["rope"])
            return q, s["k_cache"], s["v_cache"]
        if case["kind"] == "decode":
            return s["attn"].forward(s["q"], s["k_cache"], s["v_cache"], s["block_tables"], s["lens"])
        return s["attn"].prefill(s["q"], s["k_cache"], s["v_cache"], s["block_tables"], s["lens"], s["starts"],
                                 max_seq_len=s["max_len"])
    if case["kind"] == "rotary":
        cos, sin = _cos_sin(s, case)
        return _turn(s["q"], cos, sin, case), _turn(s["k"], cos, sin, case)
    if case["kind"] == "append":
        cos, sin = _cos_sin(s, case)
        there = (s["slots"] >= 0).nonzero()[:, 0]
        slots = s["slots"][there]
        s["k_cache"].view(-1, case["kv_heads"], case["dim"])[slots] = _turn(s["k"], cos, sin, case)[there]
        s["v_cache"].view(-1, case["kv_heads"], case["dim"])[slots] = s["v"][there]
        return _turn(s["q"], cos, sin, case), s["k_cache"], s["v_cache"]
    return _plain_attention(s, case)


# ---------------------------------------------------------------------------------------------------------------------
# exact values
# ---------------------------------------------------------------------------------------------------------------------
def _exact_turn(x, s, case):
    """Every pair as a complex number times e^(i angle)."""
    r = case["rotary_dim"]
    where = s["positions"].double().reshape(-1, x.shape[0])
    theta = torch.stack([where[a] * f for a, f in zip(s["axis"].tolist(), s["freq"].tolist())], dim=1)
    unit = torch.polar(torch.ones_like(theta), -theta if case.get("inverse") else theta)[:, None]
    y = x.double().clone()
    if case["pairs"] == "halves":
        z = torch.complex(y[..., :r // 2], y[..., r // 2:r]) * unit
        y[..., :r // 2], y[..., r // 2:r] = z.real, z.imag
    else:
        z = torch.view_as_complex(y[..., :r].unflatten(-1, (r // 2, 2)).contiguous()) * unit
        y[..., :r] = torch.view_as_real(z).flatten(-2)
    return y


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rotary":
        return _exact_turn(s["q"], s, case), _exact_turn(s["k"], s, case)
    if case["kind"] == "append":
        out = [_exact_turn(s["q"], s, case)]
        slots = s["slots"].cpu()
        keep = [t for t, x in enumerate(slots.tolist()) if x >= 0]
        at = slots[keep].to(s["q"].device)
        for cache, x in ((s["k_cache"], _exact_turn(s["k"], s, case)), (s["v_cache"], s["v"].double())):
            c = cache.double()
            c[at // case["block"], at % case["block"]] = x[keep]
            out.append(c)
        return tuple(out)
    starts, lens = s["starts"].tolist(), s["lens"].tolist()
    kvh, dim, bs = case["kv_heads"], case["dim"], case["block"]
    group = case["heads"] // kvh
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    for n, total in enumerate(lens):
        pages = s["block_tables"][n, :-(-total // bs)].long()
        k = s["k_cache"][pages].reshape(-1, kvh, dim)[:total].double()
        v = s["v_cache"][pages].reshape(-1, kvh, dim)[:total].double()
        lo, hi = starts[n], starts[n + 1]
        q = s["q"][lo:hi].double()
        place = torch.arange(total - (hi - lo), total, device=q.device)[:, None]
        key = torch.arange(total, device=q.device)[None]
        hidden = key > place
        if case["window"]:
            hidden |= key <= place - case["window"]
        for h in range(case["heads"]):
            score = (q[:, h] @ k[:, h // group].t()) / math.sqrt(dim)
            out[lo:hi, h] = torch.softmax(score.masked_fill(hidden, -math.inf), dim=-1) @ v[:, h // group]
    return out
