"""Rotary positions and the append with rotation against the definition in 64 bits (oracle/dense.py)."""
import pytest
import torch

from oracle import dense as od

pytestmark = pytest.mark.gpu


def _rope(D, R=None, **kw):
    from aitherkvcache_b200 import RotaryPositions
    return RotaryPositions(D, rotary_dim=R, **kw)


def _positions(axes, n, far, seed, dtype=torch.int64):
    g = torch.Generator().manual_seed(seed)
    p = torch.randint(-far // 4, far, (axes, n), generator=g)
    if n:
        p[:, 0] = 0
        p[:, -1] = far
    return p.to(dtype).cuda()


def _check(got, x, pos, rope, inverse=False):
    pos = pos if pos.dim() == 2 else pos[None].expand(rope.num_axes, -1)
    adj = rope.pair_layout == "adjacent"
    want = od.rotate(x, pos, rope.inv_freq.tolist(), rope.axes.tolist(), rope.rotary_dim, adj, rope.scaling, inverse)
    bound = od.rotate_bound(x, want, rope.rotary_dim, adj, got.dtype, rope.scaling)
    assert got.shape == x.shape
    assert bool(((got.double() - want).abs() <= bound).all()), float(((got.double() - want).abs() - bound).max())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D,R,sections,layout,pairs", [
    (128, 128, None, "blocked", "halves"),
    (128, 128, (16, 24, 24), "blocked", "halves"),
    (128, 64, (12, 10, 10), "cycled", "adjacent"),
    (64, 64, (8, 12, 12), "cycled", "halves"),
    (256, 256, None, "blocked", "adjacent"),
    (96, 48, (10, 14), "blocked", "halves"),      # 24 pairs: units of eight
    (80, 36, None, "blocked", "halves"),          # not whole units: the element kernel
    (72, 72, (9, 9, 9, 9), "cycled", "adjacent"),
    (2, 2, None, "blocked", "halves"),
])
@pytest.mark.parametrize("n,qh,kh", [(1, 1, 1), (37, 5, 3), (700, 32, 8)])
def test_rotation(dtype, D, R, sections, layout, pairs, n, qh, kh):
    rope = _rope(D, R, base=1e4, sections=sections, section_layout=layout, pair_layout=pairs)
    g = torch.Generator().manual_seed(n + D)
    q = torch.randn(n, qh, D, generator=g).to(dtype).cuda()
    k = torch.randn(n, kh, D, generator=g).to(dtype).cuda()
    pos = _positions(rope.num_axes, n, 1 << 20, n)
    for inverse in (False, True):
        qo, ko = rope.forward(q, k, pos, inverse=inverse)
        _check(qo, q, pos, rope, inverse)
        _check(ko, k, pos, rope, inverse)


def test_one_position_for_all_axes_int32_scaling_and_given_frequencies():
    freq = [2.5, -0.75, 1e-9, 6.4] + [0.01] * 28      # above half a turn per position, negative, tiny
    rope = _rope(64, sections=(8, 12, 12), inv_freq=torch.tensor(freq, dtype=torch.float64), scaling=1.25)
    x = torch.randn(50, 4, 64, generator=torch.Generator().manual_seed(0)).cuda()
    pos = torch.randint(0, 1 << 24, (50,), generator=torch.Generator().manual_seed(1), dtype=torch.int32).cuda()
    out, none = rope.forward(x, None, pos)
    assert none is None
    _check(out, x, pos, rope)
    none, out2 = rope(None, x, pos)
    assert none is None and torch.equal(out, out2)


def test_strided_views_misaligned_rows_and_in_place():
    rope = _rope(128, base=1e6)
    g = torch.Generator().manual_seed(3)
    qkv = torch.randn(33, (8 + 2 + 2) * 128 + 4, generator=g).half().cuda()
    pos = _positions(1, 33, 100000, 5)[0]
    for first in (0, 4):      # 16-byte rows, then 8-byte ones
        q = qkv[:, first:first + 8 * 128].unflatten(1, (8, 128))
        k = qkv[:, first + 8 * 128:first + 10 * 128].unflatten(1, (2, 128))
        before = qkv.clone()
        qo, ko = rope.forward(q, k, pos)
        assert torch.equal(before, qkv)
        _check(qo, q, pos, rope)
        _check(ko, k, pos, rope)
        rope.forward(q, k, pos, query_out=q, key_out=k)      # in place
        assert torch.equal(q, qo) and torch.equal(k, ko)
        rest = qkv.clone()
        rest[:, first:first + 10 * 128] = before[:, first:first + 10 * 128]
        assert torch.equal(rest, before)      # nothing else was touched
    wide = torch.randn(33, 128, 6, generator=g).half().cuda().transpose(1, 2)      # last dimension not contiguous
    _check(rope.forward(wide, None, pos)[0], wide, pos, rope)
    one = torch.randn(33, 1, 128, generator=g).half().cuda().expand(33, 5, 128)      # broadcast heads
    _check(rope.forward(one, None, pos)[0], one, pos, rope)


def test_inverse_is_the_transpose_and_takes_the_rotation_back():
    """<g, R x> = <R^T g, x> and differences of the rotation (it is linear) against the inverse applied to g."""
    rope = _rope(64, sections=(8, 12, 12), base=1e4)
    gen = torch.Generator().manual_seed(7)
    x, g = (torch.randn(20, 3, 64, generator=gen).cuda() for _ in range(2))
    pos = _positions(3, 20, 5000, 9)
    y, _ = rope.forward(x, None, pos)
    back, _ = rope.forward(y, None, pos, inverse=True)
    assert torch.allclose(back, x, rtol=0, atol=4e-6)      # two rotations of |x| < 5: 2 * 5 * 4e-7
    grad, _ = rope.forward(g, None, pos, inverse=True)
    a, b = (g.double() * y.double()).sum(), (grad.double() * x.double()).sum()
    assert abs(float(a - b)) <= 4e-7 * 2 * float((g.abs().sum() * 5))
    for at in ((0, 0, 3), (19, 2, 40), (7, 1, 63)):
        step = torch.zeros_like(x)
        step[at] = 1.0
        moved, _ = rope.forward(x + step, None, pos)
        diff = (g.double() * (moved.double() - y.double())).sum()
        # every |difference| carries the bound of two rotations on the two elements of one pair
        assert abs(float(diff) - float(grad[at])) <= 2 * 2 * 4e-7 * 12 * float(g.abs().max())


def test_empty_calls_and_other_streams():
    rope = _rope(128)
    q = torch.randn(0, 4, 128).half().cuda()
    qo, ko = rope.forward(q, q, torch.zeros(0, dtype=torch.int64, device="cuda"))
    assert qo.shape == (0, 4, 128) and ko.shape == (0, 4, 128)
    x = torch.randn(64, 4, 128).half().cuda()
    pos = torch.arange(64).cuda()
    want, _ = rope.forward(x, None, pos)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got, _ = rope.forward(x, None, pos)
    s.synchronize()
    assert torch.equal(got, want)


def _append_ref(key, value, pos, slots, kc, vc, rope):
    """Caches after the append, float64, and the bound of the keys."""
    adj = rope.pair_layout == "adjacent"
    p = pos if pos.dim() == 2 else pos[None].expand(rope.num_axes, -1)
    k = od.rotate(key, p, rope.inv_freq.tolist(), rope.axes.tolist(), rope.rotary_dim, adj, rope.scaling)
    kb = od.rotate_bound(key, k, rope.rotary_dim, adj, kc.dtype, rope.scaling)
    ks, vs, bound = kc.double().clone(), vc.double().clone(), torch.zeros_like(kc, dtype=torch.float64)
    bs = kc.shape[1]
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < kc.shape[0] * bs:
            ks[s // bs, s % bs], vs[s // bs, s % bs], bound[s // bs, s % bs] = k[t], value[t].to(vc.dtype).double(), kb[t]
    return ks, vs, bound


@pytest.mark.parametrize("n,qh,kh,D,bs,sections,pairs", [
    (1, 4, 1, 64, 16, None, "halves"), (16, 32, 8, 128, 16, None, "halves"), (301, 7, 7, 128, 24, (16, 24, 24), "halves"),
    (2050, 32, 8, 128, 16, None, "halves"), (130, 6, 2, 256, 1, (40, 44, 44), "adjacent"), (45, 3, 3, 40, 5, None, "adjacent"),
])
@pytest.mark.parametrize("src,dst", [(torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16),
                                     (torch.float32, torch.bfloat16), (torch.bfloat16, torch.float16), (torch.float16, torch.float32)])
def test_append(n, qh, kh, D, bs, sections, pairs, src, dst):
    from aitherkvcache_b200 import rotary_kv_append
    rope = _rope(D, base=1e6, sections=sections, pair_layout=pairs)
    g = torch.Generator().manual_seed(n)
    qkv = torch.randn(n, qh + 2 * kh, D, generator=g).to(src).cuda()
    q, k, v = qkv[:, :qh], qkv[:, qh:qh + kh], qkv[:, qh + kh:]
    nb = -(-n // bs) + 4
    both = torch.randn(nb, 2, bs, kh, D, generator=g).to(dst).cuda()      # keys and values of a block side by side
    kc, vc = both[:, 0], both[:, 1]
    slots = torch.randperm(nb * bs, generator=g)[:n].cuda()
    if n > 1:
        slots[::7] = -1
        slots[3 % n] = nb * bs + 3      # behind the cache
    pos = _positions(rope.num_axes, n, 200000, n)
    pos = pos[0] if sections is None else pos
    want_k, want_v, bound = _append_ref(k, v, pos, slots, kc, vc, rope)
    out = rotary_kv_append(q, k, v, pos, slots.int() if n % 2 else slots, kc, vc, rope)
    assert out.dtype == dst and out.shape == q.shape
    _check(out, q, pos, rope)
    assert torch.equal(vc.double(), want_v)
    assert bool(((kc.double() - want_k).abs() <= bound).all())
    # without a query: the same cache
    again = both.clone()
    assert rotary_kv_append(None, k, v, pos, slots, again[:, 0], again[:, 1], rope) is None
    assert torch.equal(again, both)


def test_append_into_a_cache_past_32_bit_offsets():
    from aitherkvcache_b200 import rotary_kv_append
    rope = _rope(128)
    nb = (1 << 31) // (16 * 8 * 128) + 40      # over 2^31 elements: 4.3 GB
    kc, vc = (torch.zeros(nb, 16, 8, 128, dtype=torch.float16, device="cuda") for _ in range(2))
    g = torch.Generator().manual_seed(0)
    k, v = (torch.randn(3, 8, 128, generator=g).half().cuda() for _ in range(2))
    pos = torch.tensor([5, 6, 7]).cuda()
    slots = torch.tensor([nb * 16 - 1, 0, (nb - 5) * 16 + 3]).cuda()
    rotary_kv_append(None, k, v, pos, slots, kc, vc, rope)
    kr, _ = rope.forward(k, None, pos)
    for cache, rows in ((kc, kr), (vc, v)):
        flat = cache.view(-1, 8, 128)
        assert torch.equal(flat[slots], rows)
        for part in (flat[:64], flat[-128:]):
            assert int((part != 0).flatten(1).any(1).sum()) == (1 if part.data_ptr() == flat.data_ptr() else 2)


def test_append_replays_from_a_graph_with_new_inputs():
    from aitherkvcache_b200 import rotary_kv_append
    rope = _rope(128, base=1e6)
    n, qh, kh = 16, 32, 8
    g = torch.Generator().manual_seed(2)
    make = lambda h: torch.randn(n, h, 128, generator=g).half().cuda()  # noqa: E731
    q, k, v, qo = make(qh), make(kh), make(kh), torch.empty(n, qh, 128, dtype=torch.float16, device="cuda")
    kc, vc = (torch.zeros(20, 16, kh, 128, dtype=torch.float16, device="cuda") for _ in range(2))
    pos, slots = torch.arange(n).cuda(), torch.arange(n).cuda() * 16
    run = lambda: rotary_kv_append(q, k, v, pos, slots, kc, vc, rope, query_out=qo)  # noqa: E731
    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for seed in range(2):
        q.copy_(make(qh)), k.copy_(make(kh)), v.copy_(make(kh))
        pos.add_(seed + 1000), slots.add_(1)
        graph.replay()
        k2, v2 = kc.clone(), vc.clone()
        out = rotary_kv_append(q, k, v, pos, slots, k2, v2, rope)
        assert torch.equal(out, qo) and torch.equal(k2, kc) and torch.equal(v2, vc)
        _check(qo, q, pos, rope)


def test_copies_of_rotary_positions():
    """A deep copy on the device rotates alike after the original and its tables are gone."""
    import copy
    from aitherkvcache_b200 import RotaryPositions
    rope = RotaryPositions(64, base=1e5, sections=(16, 8, 8))
    q = torch.randn(50, 3, 64, device="cuda")
    pos = torch.randint(0, 10 ** 6, (3, 50), device="cuda")
    want = rope.forward(q, None, pos)[0]
    twin = copy.deepcopy(rope)
    rope.steps.fill_(0)      # what the copy must not look at
    rope.axes.fill_(0)
    del rope
    assert torch.equal(twin.forward(q, None, pos)[0], want)
