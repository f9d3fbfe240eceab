"""The dense cache's operators as a serving loop uses them, and behind the vLLM backend's methods, against attention over
the whole sequence in 64 bits."""
import math
import types

import pytest
import torch

from oracle import dense as od

pytestmark = pytest.mark.gpu


def _rotated(x, pos, rope):
    p = pos if pos.dim() == 2 else pos[None].expand(rope.num_axes, -1)
    return od.rotate(x, p, rope.inv_freq.tolist(), rope.axes.tolist(), rope.rotary_dim, rope.pair_layout == "adjacent", rope.scaling)


def _pages(n_seqs, per_seq, bs, H, D, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    nb = n_seqs * per_seq + 3
    kv = torch.full((nb, 2, bs, H, D), math.nan, dtype=dtype, device="cuda")      # nothing may read what was not written
    return kv, torch.randperm(nb, generator=g)[:n_seqs * per_seq].view(n_seqs, per_seq).int().cuda()


def _slots(bt, bs, seq, first, n):
    at = torch.arange(first, first + n, device="cuda")
    return bt[seq].long()[at // bs] * bs + at % bs


def _expect(q, k, v, lens, new, window, scale):
    """Rows of the last `new` tokens of every sequence from whole rotated q, k, v (lists of float64): output and bound.

    The caches hold k and the attention sees q rounded to the type (relative error u each, so a score is off by 2 u
    sum|q k| and a weight by that factor), v is as it was; the attention's own bound (oracle.dense.attention) is 2 d + u and
    below: 3 u in all for the weights' relative error of the rounding, and u for the result."""
    outs, bounds = [], []
    u = torch.finfo(torch.bfloat16).eps / 2
    for qs, ks, vs, L, n in zip(q, k, v, lens, new):
        group = qs.shape[1] // ks.shape[1]
        kk, vv = (x.repeat_interleave(group, 1) for x in (ks, vs))
        s = torch.einsum("qhd,khd->hqk", qs[L - n:L], kk[:L]) * scale
        mag = torch.einsum("qhd,khd->hqk", qs[L - n:L].abs(), kk[:L].abs()) * scale
        p, j = torch.arange(L - n, L, device="cuda")[:, None], torch.arange(L, device="cuda")[None]
        hide = j > p
        if window:
            hide |= j <= p - window
        w = torch.softmax(s.masked_fill(hide, -math.inf), -1)
        o = torch.einsum("hqk,khd->qhd", w, vv[:L])
        a = torch.einsum("hqk,khd->qhd", w, vv[:L].abs())
        d = (2 * u + 2.0 ** -14) * mag.masked_fill(hide, 0).amax(-1).transpose(0, 1)[..., None]
        outs.append(o)
        bounds.append((torch.expm1(2 * d) + 2 * u) * a + u * o.abs() + 1e-6)
    return torch.cat(outs), torch.cat(bounds)


@pytest.mark.parametrize("H,QH,D,bs,window", [(2, 8, 128, 16, 0), (4, 4, 64, 32, 100)])
def test_prompt_chunks_then_single_tokens(H, QH, D, bs, window):
    """Two prompts in two chunks each, then three single-token steps: append with rotation, attention, every time."""
    from aitherkvcache_b200 import DensePagedAttention, RotaryPositions, rotary_kv_append
    dtype, total = torch.bfloat16, [333, 150]
    rope = RotaryPositions(D, base=1e4, sections=(D // 8, D // 4, D // 8))
    attn = DensePagedAttention(D, QH, H, sliding_window=window)
    g = torch.Generator().manual_seed(0)
    q, k, v = ([torch.randn(n + 3, h, D, generator=g).to(dtype).cuda() for n in total] for h in (QH, H, H))
    pos = [torch.randint(0, 5000, (3, n + 3), generator=g).cuda() for n in total]
    qr, kr = ([_rotated(x, p, rope) for x, p in zip(xs, pos)] for xs in (q, k))
    kv, bt = _pages(2, -(-340 // bs), bs, H, D, dtype, 1)
    done = [0, 0]
    for step in range(5):
        new = [[200, 100], [133, 50], [1, 1], [1, 1], [1, 1]][step]
        cut = [slice(d, d + n) for d, n in zip(done, new)]
        args = [torch.cat([x[c] for x, c in zip(xs, cut)]) for xs in (q, k, v)]
        slots = torch.cat([_slots(bt, bs, s, d, n) for s, (d, n) in enumerate(zip(done, new))])
        qo = rotary_kv_append(*args, torch.cat([p[:, c] for p, c in zip(pos, cut)], 1), slots, kv[:, 0], kv[:, 1], rope)
        done = [d + n for d, n in zip(done, new)]
        lens = torch.tensor(done, dtype=torch.int32, device="cuda")
        starts = torch.tensor([0, new[0], sum(new)], dtype=torch.int32, device="cuda")
        if max(new) > 1:
            out = attn.prefill(qo, kv[:, 0], kv[:, 1], bt, lens, starts)
        else:
            out = attn.forward(qo, kv[:, 0], kv[:, 1], bt, lens)
            chunk = attn.prefill(qo, kv[:, 0], kv[:, 1], bt, lens, starts)
        want, bound = _expect(qr, kr, [x.double() for x in v], done, new, window, 1 / math.sqrt(D))
        assert bool(((out.double() - want).abs() <= bound).all())
        if max(new) == 1:
            assert bool(((chunk.double() - want).abs() <= bound).all())


def _impl(QH, H, D, window=None):
    from aitherkvcache_b200.vllm.backend import TurboQuantImplBase
    impl = TurboQuantImplBase()
    impl._tq_setup(QH, D, 1 / math.sqrt(D), H, "auto")
    impl.sliding_window = window
    return impl


@pytest.mark.parametrize("window,as_vllm", [(0, None), (64, (63, 0)), (64, 64), (0, (-1, -1))])
def test_backend_over_a_16_bit_cache(window, as_vllm):
    """The impl's cache update and forward on a bf16 cache: prompts, a mixed batch (a chunk, single tokens), single tokens."""
    QH, H, D, bs, dtype = 8, 2, 128, 16, torch.bfloat16
    from aitherkvcache_b200 import RotaryPositions
    impl, rope = _impl(QH, H, D, as_vllm), RotaryPositions(D, base=1e4)
    layer = types.SimpleNamespace(layer_name="dense")
    g = torch.Generator().manual_seed(3)
    total = [220, 90, 31]
    q, k, v = ([torch.randn(n, h, D, generator=g).to(dtype).cuda() for n in total] for h in (QH, H, H))
    pos = [torch.arange(n).cuda() for n in total]
    qr, kr = ([_rotated(x, p, rope) for x, p in zip(xs, pos)] for xs in (q, k))
    kv, bt = _pages(3, 15, bs, H, D, dtype, 2)
    done = [0, 0, 0]
    for new in ([100, 88, 29], [60, 1, 1], [1, 1, 1]):
        cut = [slice(d, d + n) for d, n in zip(done, new)]
        qn, kn, vn = (torch.cat([x[c] for x, c in zip(xs, cut)]) for xs in (q, k, v))
        slots = torch.cat([_slots(bt, bs, s, d, n) for s, (d, n) in enumerate(zip(done, new))])
        p = torch.cat([x[c] for x, c in zip(pos, cut)])
        qo = impl.rope_and_kv_cache_update(layer, qn, kn, vn, p, rope, kv, slots)
        done = [d + n for d, n in zip(done, new)]
        starts = [0, new[0], new[0] + new[1], sum(new)]
        md = types.SimpleNamespace(num_actual_tokens=sum(new), max_query_len=max(new), block_table=bt, max_seq_len=max(done),
                                   seq_lens=torch.tensor(done, dtype=torch.int32, device="cuda"),
                                   query_start_loc=torch.tensor(starts, dtype=torch.int32, device="cuda"))
        out = torch.zeros(sum(new) + 5, QH * D, dtype=dtype, device="cuda")      # a padded batch
        pad = torch.cat([qo, torch.zeros(5, QH, D, dtype=dtype, device="cuda")])
        impl.forward(layer, pad.flatten(1), None, None, kv, md, output=out)
        want, bound = _expect(qr, kr, [x.double() for x in v], done, new, window, 1 / math.sqrt(D))
        got = out[:sum(new)].view(-1, QH, D).double()
        assert bool(((got - want).abs() <= bound).all())
        assert bool((out[sum(new):] == 0).all())


def test_backend_update_of_rotated_keys_and_of_packed_caches():
    """do_kv_cache_update on a 16-bit cache stores as is; on a packed cache the rotating update equals rotation then update."""
    QH, H, D, bs = 8, 2, 128, 16
    from aitherkvcache_b200 import RotaryPositions
    impl, rope = _impl(QH, H, D), RotaryPositions(D, base=1e4)
    layer = types.SimpleNamespace(layer_name="packed")
    g = torch.Generator().manual_seed(4)
    q, k, v = (torch.randn(37, h, D, generator=g).half().cuda() for h in (QH, H, H))
    slots, pos = torch.randperm(64, generator=g)[:37].cuda(), torch.arange(1000, 1037).cuda()
    slots[5] = -1
    kv = torch.zeros(4, 2, bs, H, D, dtype=torch.float16, device="cuda")
    impl.do_kv_cache_update(layer, k, v, kv, slots)
    keep = slots >= 0
    for side, x in ((0, k), (1, v)):
        flat = kv[:, side].reshape(-1, H, D)
        assert torch.equal(flat[slots[keep]], x[keep]) and int((flat != 0).flatten(1).any(1).sum()) == 36
    a, b = (torch.zeros(4, 2, bs, H, D, dtype=torch.uint8, device="cuda") for _ in range(2))
    qa = impl.rope_and_kv_cache_update(layer, q, k, v, pos, rope, a, slots)
    qb, kb = rope.forward(q, k, pos)
    impl.do_kv_cache_update(layer, kb, v, b, slots)
    assert torch.equal(qa, qb) and torch.equal(a, b) and int((a != 0).sum()) > 0


def test_calls_on_two_streams_at_once():
    """The same objects used on two streams at the same time: no scratch is shared."""
    from aitherkvcache_b200 import DensePagedAttention, RotaryPositions, rotary_kv_append
    H, QH, D, bs = 8, 32, 128, 16
    attn, rope = DensePagedAttention(D, QH, H), RotaryPositions(D)
    g = torch.Generator().manual_seed(5)
    work = []
    for i in range(2):
        kv = torch.randn(300, 2, bs, H, D, generator=g).half().cuda()
        bt = torch.randperm(300, generator=g)[:292].view(4, 73).int().cuda()
        lens = torch.tensor([1100 + i, 700, 30, 5], dtype=torch.int32).cuda()
        starts = torch.tensor([0, 300, 340, 350, 352], dtype=torch.int32).cuda()
        work.append((torch.randn(352, QH, D, generator=g).half().cuda(), kv, bt, lens, starts))
    run = lambda q, kv, bt, lens, starts: (attn.prefill(q, kv[:, 0], kv[:, 1], bt, lens, starts),  # noqa: E731
                                           attn.forward(q[:4], kv[:, 0], kv[:, 1], bt, lens),
                                           rope.forward(q, None, torch.arange(352, device="cuda"))[0])
    want = [run(*w) for w in work]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(run(*work[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for res in got[i]:
            assert all(torch.equal(x, y) for x, y in zip(res, want[i]))


@pytest.mark.parametrize("src,dst", [(torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16)])
@pytest.mark.parametrize("heads,D,bs", [(2, 128, 16), (3, 64, 5), (1, 40, 1)])
def test_kv_append(src, dst, heads, D, bs):
    """Keys as they are: slices of a fused projection, a transposed one, padding, and what lies around the slots."""
    from aitherkvcache_b200 import kv_append
    g = torch.Generator().manual_seed(D + bs)
    for n in (0, 1, 77):
        blocks = 2 * n // bs + 2
        slots = torch.randperm(blocks * bs, generator=g)[:n]
        if n > 3:
            slots[1], slots[2] = -1, blocks * bs
        qkv = torch.randn(n, heads * 4, D, generator=g).to(src).cuda()
        caches = torch.randn(blocks, 2, bs, heads, D, generator=g).to(dst).cuda()
        want = caches.clone()
        key, value = qkv[:, heads:2 * heads], qkv[:, 2 * heads:3 * heads]
        for t, s in enumerate(slots.tolist()):
            if 0 <= s < blocks * bs:
                want[s // bs, 0, s % bs], want[s // bs, 1, s % bs] = key[t].to(dst), value[t].to(dst)
        for form in (lambda x: x, lambda x: x.transpose(1, 2).contiguous().transpose(1, 2)):
            got = caches.clone()
            kv_append(form(key), form(value), slots.cuda(), got[:, 0], got[:, 1])
            assert torch.equal(got, want)
            got = caches.clone()
            kv_append(key, form(value), slots.int().cuda(), got[:, 0], got[:, 1])
            assert torch.equal(got, want)


@pytest.mark.parametrize("kind", ["dense", "packed"])
@pytest.mark.parametrize("pad", [1, 30])
def test_backend_rotating_update_of_a_padded_batch(kind, pad):
    """Query, key, value and positions padded behind the slots' length: what has a slot is stored as without the padding,
    nothing else is touched, and every query row is turned."""
    QH, H, D, bs, n = 8, 2, 128, 16, 37
    from aitherkvcache_b200 import RotaryPositions
    impl, rope = _impl(QH, H, D), RotaryPositions(D, base=1e4)
    layer = types.SimpleNamespace(layer_name="padded")
    g = torch.Generator().manual_seed(pad)
    q, k, v = (torch.randn(n + pad, h, D, generator=g).half().cuda() for h in (QH, H, H))
    slots, pos = torch.randperm(64, generator=g)[:n].cuda(), torch.arange(n + pad).cuda()
    dtype = torch.float16 if kind == "dense" else torch.uint8
    a, b = (torch.zeros(4, 2, bs, H, D, dtype=dtype, device="cuda") for _ in range(2))
    qa = impl.rope_and_kv_cache_update(layer, q, k, v, pos, rope, a, slots)
    qb = impl.rope_and_kv_cache_update(layer, q[:n], k[:n], v[:n], pos[:n], rope, b, slots)
    assert torch.equal(a, b) and int((a != 0).sum()) > 0
    assert torch.equal(qa[:n], qb) and torch.equal(qa, rope.forward(q, None, pos)[0])
    graph = torch.cuda.CUDAGraph()
    out = torch.empty_like(q)
    a.zero_()
    with torch.cuda.graph(graph):
        impl.rope_and_kv_cache_update(layer, q, k, v, pos, rope, a, slots, out)
    graph.replay()
    assert torch.equal(a, b) and torch.equal(out, qa)


def test_compressed_and_exempt_layers_side_by_side():
    """A layer with a compressed cache dtype and one that is exempt from it, in one process, with the same block tables and
    slots and pages of one shape: each gives what it gives alone."""
    from aitherkvcache_b200.vllm.backend import TurboQuantImplBase
    QH, H, D, bs, dtype = 8, 2, 128, 16, torch.bfloat16
    g = torch.Generator().manual_seed(7)
    packed, exempt = TurboQuantImplBase(), TurboQuantImplBase()
    packed._tq_setup(QH, D, 1 / math.sqrt(D), H, "tq-t4nc")
    exempt._tq_setup(QH, D, 1 / math.sqrt(D), H, "auto")
    layers = [types.SimpleNamespace(layer_name=n) for n in ("side.0", "side.1")]
    new = [[48, 32], [1, 1], [5, 1]]
    _, bt = _pages(2, 4, bs, H, D, dtype, 3)
    x = [[torch.randn(2, 64, h, D, generator=g).to(dtype).cuda() for h in (QH, H, H)] for _ in layers]      # per layer: q, k, v by sequence

    def serve(which):
        caches = [torch.zeros(11, 2, bs, H, D, dtype=torch.uint8, device="cuda"), torch.zeros(11, 2, bs, H, D, dtype=dtype, device="cuda")]
        done, outs = [0, 0], {i: [] for i in which}
        for step in new:
            cut = [slice(d, d + n) for d, n in zip(done, step)]
            slots = torch.cat([_slots(bt, bs, s, d, n) for s, (d, n) in enumerate(zip(done, step))])
            done = [d + n for d, n in zip(done, step)]
            md = types.SimpleNamespace(num_actual_tokens=sum(step), max_query_len=max(step), block_table=bt, max_seq_len=max(done),
                                       seq_lens=torch.tensor(done, dtype=torch.int32, device="cuda"),
                                       query_start_loc=torch.tensor([0, step[0], sum(step)], dtype=torch.int32, device="cuda"))
            for i in which:
                q, k, v = (torch.cat([t[s, c] for s, c in enumerate(cut)]) for t in x[i])
                impl = (packed, exempt)[i]
                impl.do_kv_cache_update(layers[i], k, v, caches[i], slots)
                outs[i].append(impl.forward(layers[i], q.flatten(1), None, None, caches[i], md, output=torch.zeros(sum(step), QH * D, dtype=dtype, device="cuda")))
        return caches, outs

    both, both_outs = serve((0, 1))
    for i in (0, 1):
        alone, outs = serve((i,))
        assert torch.equal(alone[i], both[i]) and all(torch.equal(a, b) for a, b in zip(outs[i], both_outs[i]))
    q, k, v = ([t[s].double() for s in range(2)] for t in x[1])
    want, bound = _expect(q, k, v, [48, 32], [48, 32], 0, 1 / math.sqrt(D))
    assert bool(((both_outs[1][0].view(-1, QH, D).double() - want).abs() <= bound).all())
