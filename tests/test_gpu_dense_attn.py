"""Attention over the dense paged cache against the definition in 64 bits (oracle/dense.py)."""
import math

import pytest
import torch

from oracle import dense as od

pytestmark = pytest.mark.gpu


def make(lens, new, qh, kvh, D, bs, dtype, seed=0, scale_q=1.0, stale=None, extra=2, tail=0):
    """Random query, paged caches in a permuted pool (one tensor holds the keys and values of a block) and tables.
    ``stale``: value of every slot behind a sequence's end and of the unused blocks."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // bs) for n in lens]
    nb = sum(need) + extra
    kv = torch.randn(nb, 2, bs, kvh, D, generator=g).to(dtype)
    perm = torch.randperm(nb, generator=g)
    width = max(need + [1])
    bt = torch.zeros(len(lens), width, dtype=torch.int32)
    at = 0
    used = torch.zeros(nb, bs, dtype=torch.bool)
    for s, (n, c) in enumerate(zip(lens, need)):
        bt[s, :c] = perm[at:at + c]
        for i in range(c):
            used[perm[at + i], :max(0, min(bs, n - i * bs))] = True
        at += c
    if stale is not None:
        kv.transpose(1, 2)[~used] = stale
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    q = (torch.randn(starts[-1] + tail, qh, D, generator=g) * scale_q).to(dtype)
    kv = kv.cuda()
    return (q.cuda(), kv[:, 0], kv[:, 1], bt.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(),
            torch.tensor(starts, dtype=torch.int32).cuda())


def check(out, q, kc, vc, bt, lens, starts, window=0, scale=None, rows=None):
    want, bound = od.attention(q, kc, vc, bt, lens.tolist(), starts.tolist(), scale or 1.0 / math.sqrt(q.shape[2]), window)
    rows = slice(0, int(starts[-1])) if rows is None else rows
    off = (out[rows].double() - want[rows]).abs() - bound[rows]
    assert bool((off <= 0).all()), (float(off.max()), float(want.abs().max()))


def attn(qh, kvh, D, **kw):
    from aitherkvcache_b200 import DensePagedAttention
    return DensePagedAttention(D, qh, kvh, **kw)


LENS = [[1], [17, 0, 300], [1, 2, 15, 16, 17, 31, 32, 33, 511, 0, 1200], [5000, 3]]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("qh,kvh,D", [(32, 8, 128), (8, 8, 64), (7, 1, 128), (16, 1, 64), (40, 2, 128), (6, 2, 256), (12, 1, 256), (33, 3, 64)])
@pytest.mark.parametrize("lens", LENS, ids=lambda x: str(len(x)))
def test_single_tokens(dtype, qh, kvh, D, lens):
    q, kc, vc, bt, cl, starts = make(lens, [1] * len(lens), qh, kvh, D, 16, dtype, seed=len(lens), scale_q=2.0, stale=math.nan)
    out = attn(qh, kvh, D).forward(q, kc, vc, bt, cl)
    check(out, q, kc, vc, bt, cl, starts)


@pytest.mark.parametrize("bs", [1, 5, 8, 24, 48, 256])
@pytest.mark.parametrize("window", [0, 1, 16, 100])
def test_single_tokens_blocks_and_windows(bs, window):
    lens = [1, 40, 129, 700, 0]
    q, kc, vc, bt, cl, starts = make(lens, [1] * 5, 8, 2, 128, bs, torch.float16, seed=bs, stale=math.inf)
    out = attn(8, 2, 128, sliding_window=window).forward(q, kc, vc, bt.long(), cl.long())
    check(out, q, kc, vc, bt, cl, starts, window)


def test_single_tokens_many_sequences():
    g = torch.Generator().manual_seed(1)
    lens = torch.randint(0, 90, (4500,), generator=g).tolist()      # more than one launch takes
    q, kc, vc, bt, cl, starts = make(lens, [1] * len(lens), 2, 1, 64, 16, torch.bfloat16, stale=math.nan)
    out = attn(2, 1, 64).forward(q, kc, vc, bt, cl)
    check(out, q, kc, vc, bt, cl, starts)


def test_single_tokens_large_scores_and_growing_maxima():
    """Scores of hundreds that grow along the keys: the reference moves at every step."""
    q, kc, vc, bt, cl, starts = make([900], [1], 4, 1, 128, 16, torch.float16, seed=3)
    kc.mul_(0.02)
    q.fill_(1.0)
    ramp = torch.arange(900, device="cuda").half() / 64      # q.k grows by 2 per key
    for i in range(57):
        n = min(16, 900 - 16 * i)
        kc[bt[0, i].long(), :n] += ramp[16 * i:16 * i + n, None, None]
    out = attn(4, 1, 128, scale=1.0).forward(q, kc, vc, bt, cl)
    check(out, q, kc, vc, bt, cl, starts, scale=1.0)


def test_single_tokens_strides_padding_and_bad_tables():
    lens = [70, 33, 100]
    q, kc, vc, bt, cl, starts = make(lens, [1] * 3, 8, 2, 128, 16, torch.float16, seed=5)
    a = attn(8, 2, 128)
    want = a.forward(q, kc, vc, bt, cl)
    # heads first inside a block, query rows inside a wider projection, output rows likewise
    kh, vh = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (kc, vc))
    wide = torch.randn(3, 12, 128, device="cuda").half()
    wide[:, 2:10] = q
    out = torch.full((3, 9, 128), 7.0, dtype=torch.float16, device="cuda")
    res = a.forward(wide[:, 2:10], kh, vh, bt, cl, out=out[:, :8])
    assert res.data_ptr() == out.data_ptr() and torch.equal(out[:, :8], want) and bool((out[:, 8] == 7.0).all())
    # rows that start anywhere are copied first
    odd = torch.randn(3, 8 * 128 + 1, device="cuda").half()
    odd[:, 1:] = q.flatten(1)
    assert torch.equal(a.forward(odd[:, 1:].unflatten(1, (8, 128)), kc, vc, bt, cl), want)
    # tables wider than needed with entries outside the pool behind the sequence, lengths clamped to the table
    wide_bt = torch.full((5, 20), -9, dtype=torch.int64, device="cuda")
    wide_bt[:, 10:] = 1 << 40
    wide_bt[:3, :bt.shape[1]] = bt
    for s, n in enumerate(lens):
        wide_bt[s, -(-n // 16):] = 1 << 40
    assert torch.equal(a.forward(q, kc, vc, wide_bt, torch.cat([cl, cl[:1]])), want)
    clamped = a.forward(q, kc, vc, bt, torch.tensor([10 ** 9, -5, 100], dtype=torch.int32, device="cuda"))
    full = a.forward(q, kc, vc, bt, torch.tensor([bt.shape[1] * 16, 0, 100], dtype=torch.int32, device="cuda"))
    assert torch.equal(clamped, full) and bool((clamped[1] == 0).all())


def test_single_tokens_nan_reaches_the_rows_that_see_it():
    q, kc, vc, bt, cl, starts = make([40, 40], [1, 1], 8, 2, 64, 16, torch.bfloat16, seed=8)
    q[0, 3, 5] = math.nan      # one head of one sequence
    out = attn(8, 2, 64).forward(q, kc, vc, bt, cl)
    assert bool(out[0, 3].isnan().all())
    out[0, 3] = 0
    assert bool(out.isfinite().all())


def test_single_tokens_past_32_bit_offsets():
    nb = (1 << 31) // (16 * 8 * 128) + 64      # over 2^31 elements per cache
    kc, vc = (torch.zeros(nb, 16, 8, 128, dtype=torch.float16, device="cuda") for _ in range(2))
    g = torch.Generator().manual_seed(0)
    bt = torch.tensor([[nb - 1, 0, nb - 40], [3, nb - 2, 5]], dtype=torch.int32)
    for b in bt.flatten().tolist():
        kc[b] = torch.randn(16, 8, 128, generator=g).half().cuda()
        vc[b] = torch.randn(16, 8, 128, generator=g).half().cuda()
    q = torch.randn(2, 32, 128, generator=g).half().cuda()
    cl = torch.tensor([48, 41], dtype=torch.int32).cuda()
    out = attn(32, 8, 128).forward(q, kc, vc, bt.cuda(), cl)
    check(out, q, kc, vc, bt.cuda(), cl, torch.tensor([0, 1, 2]))


def test_single_tokens_graph_replay_and_streams():
    lens = [700, 20, 4000]
    q, kc, vc, bt, cl, starts = make(lens, [1] * 3, 32, 8, 128, 16, torch.float16, seed=9)
    a = attn(32, 8, 128)
    out = torch.empty_like(q)
    a.forward(q, kc, vc, bt, cl, out=out)
    graphs = []
    for _ in range(2):      # two graphs of one object
        o = torch.empty_like(q)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            a.forward(q, kc, vc, bt, cl, out=o)
        graphs.append((graph, o, torch.cuda.Stream()))
    for step in range(3):
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(step)).half())
        cl.add_(-1)
        want = a.forward(q, kc, vc, bt, cl)
        for graph, o, s in graphs:      # replayed at the same time
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                graph.replay()
        for graph, o, s in graphs:
            s.synchronize()
            assert torch.equal(o, want)
    check(want, q, kc, vc, bt, cl, starts)


# ---------------------------------------------------------------------------------------------------------------------
# chunks of new tokens
# ---------------------------------------------------------------------------------------------------------------------
CHUNKS = {      # (tokens with the chunk's, the chunk's)
    "one": ([1], [1]),
    "prompt": ([130], [130]),
    "tiles": ([127, 128, 129, 256, 257], [127, 128, 129, 256, 257]),
    "behind": ([1000, 40, 513], [3, 40, 70]),
    "mixed": ([700, 0, 5, 90, 33, 1500], [1, 1, 5, 0, 33, 200]),
    "long": ([5000], [300]),
}


def run_chunks(lens, new, qh, kvh, D, bs, dtype, window=0, seed=0, tail=0, **kw):
    q, kc, vc, bt, cl, starts = make(lens, new, qh, kvh, D, bs, dtype, seed=seed, stale=math.nan, tail=tail, **kw)
    out = attn(qh, kvh, D, sliding_window=window).prefill(q, kc, vc, bt, cl, starts)
    from aitherkvcache_b200 import _lib
    assert _lib.device_status()["attn_window"] == 0
    check(out, q, kc, vc, bt, cl, starts, window)
    return out


@pytest.mark.parametrize("chunks", CHUNKS)
@pytest.mark.parametrize("qh,kvh,D", [(8, 2, 128), (8, 1, 64), (3, 3, 128), (14, 2, 64), (20, 4, 128), (64, 1, 64)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_chunks(dtype, qh, kvh, D, chunks):
    lens, new = CHUNKS[chunks]
    run_chunks(lens, new, qh, kvh, D, 16, dtype, seed=len(lens), scale_q=2.0)


@pytest.mark.parametrize("bs", [8, 24, 32, 128, 384])
@pytest.mark.parametrize("window", [0, 1, 100, 128, 1000])
def test_chunks_blocks_and_windows(bs, window):
    run_chunks([900, 77, 2000, 1], [300, 77, 9, 1], 8, 2, 128, bs, torch.float16, window, seed=bs)


@pytest.mark.parametrize("qh,kvh,D,bs", [(4, 2, 256, 16), (4, 2, 128, 5), (129, 1, 64, 16)])
def test_chunks_that_attend_token_by_token(qh, kvh, D, bs):
    out = run_chunks([300, 20, 0], [40, 20, 2], qh, kvh, D, bs, torch.bfloat16, 30, tail=3)
    assert bool((out[-3:] == 0).all())


def test_chunks_more_query_tokens_than_cached_tokens():
    """The first tokens of a chunk longer than its sequence see nothing and come out as zeros."""
    q, kc, vc, bt, cl, starts = make([50, 60], [50, 60], 8, 2, 128, 16, torch.float16, seed=4)
    cl[0] = 20
    out = attn(8, 2, 128).prefill(q, kc, vc, bt, cl, starts)
    assert bool((out[:30] == 0).all())
    check(out, q, kc, vc, bt, cl, starts)


def test_chunks_rows_behind_the_last_sequence():
    lens, new = [200, 40], [33, 40]
    q, kc, vc, bt, cl, starts = make(lens, new, 8, 2, 64, 16, torch.float16, seed=6, tail=700)
    a = attn(8, 2, 64)
    want = a.prefill(q, kc, vc, bt, cl, starts)
    assert bool((want[73:] == 0).all())
    check(want, q, kc, vc, bt, cl, starts)
    out = torch.full((773, 10, 64), 5.0, dtype=torch.float16, device="cuda")
    res = a.prefill(q, kc, vc, bt.long(), cl.long(), starts.long(), out=out[:, :8], max_seq_len=200)
    assert res.data_ptr() == out.data_ptr() and torch.equal(out[:73, :8], want[:73])
    assert bool((out[73:] == 5.0).all()) and bool((out[:, 8:] == 5.0).all())


def test_chunks_large_scores_and_growing_maxima():
    q, kc, vc, bt, cl, starts = make([900], [200], 4, 1, 128, 16, torch.bfloat16, seed=3)
    kc.mul_(0.02)
    q.fill_(1.0)
    ramp = (torch.arange(912, device="cuda") / 64).to(torch.bfloat16).view(57, 16)
    kc[bt[0, :57].long()] += ramp[:, :, None, None]
    out = attn(4, 1, 128, scale=1.0).prefill(q, kc, vc, bt, cl, starts)
    check(out, q, kc, vc, bt, cl, starts, scale=1.0)


def test_chunks_strides_and_bad_tables():
    lens, new = [300, 100], [50, 100]
    q, kc, vc, bt, cl, starts = make(lens, new, 8, 2, 128, 16, torch.float16, seed=5)
    a = attn(8, 2, 128)
    want = a.prefill(q, kc, vc, bt, cl, starts)
    kh, vh = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (kc, vc))      # heads first inside a block
    wide = torch.randn(150, 12, 128, device="cuda").half()
    wide[:, 2:10] = q
    assert torch.equal(a.prefill(wide[:, 2:10], kh, vh, bt, cl, starts), want)
    odd = torch.randn(150, 8 * 128 + 1, device="cuda").half()
    odd[:, 1:] = q.flatten(1)
    assert torch.equal(a.prefill(odd[:, 1:].unflatten(1, (8, 128)), kc, vc, bt, cl, starts), want)
    far = torch.full((2, 40), 1 << 40, dtype=torch.int64, device="cuda")
    for s, n in enumerate(lens):
        far[s, :-(-n // 16)] = bt[s, :-(-n // 16)]
    far[0, 30:] = -7
    assert torch.equal(a.prefill(q, kc, vc, far, cl, starts), want)
    one = attn(8, 2, 128).prefill(q, kc, vc, bt, torch.tensor([10 ** 9, 100], dtype=torch.int32, device="cuda"), starts)
    full = attn(8, 2, 128).prefill(q, kc, vc, bt, torch.tensor([bt.shape[1] * 16, 100], dtype=torch.int32, device="cuda"), starts)
    assert torch.equal(one, full)


def test_chunks_nan_of_a_query_or_key_reaches_the_rows_that_see_it():
    q, kc, vc, bt, cl, starts = make([300], [300], 4, 2, 128, 16, torch.float16, seed=8)
    q[7, 1, 5] = math.nan
    out = attn(4, 2, 128).prefill(q, kc, vc, bt, cl, starts)
    assert bool(out[7, 1].isnan().all()) and int(out.isnan().any(-1).sum()) == 1
    q[7, 1, 5] = 0
    kc[bt[0, 6].long(), 4, 0, 9] = math.nan      # key 100 of KV head 0: query heads 0 and 1 from token 100 on
    out = attn(4, 2, 128).prefill(q, kc, vc, bt, cl, starts)
    assert bool(out[100:, :2].isnan().all()) and bool(out[:100].isfinite().all()) and bool(out[:, 2:].isfinite().all())


def test_chunks_many_sequences_and_repeatability():
    g = torch.Generator().manual_seed(2)
    new = torch.randint(0, 4, (2300,), generator=g).tolist()      # more than one launch takes
    lens = [n + int(x) for n, x in zip(new, torch.randint(0, 300, (2300,), generator=g))]
    q, kc, vc, bt, cl, starts = make(lens, new, 2, 1, 64, 16, torch.bfloat16, seed=1, stale=math.nan)
    a = attn(2, 1, 64)
    out = a.prefill(q, kc, vc, bt, cl, starts)
    check(out, q, kc, vc, bt, cl, starts)
    for _ in range(3):
        assert torch.equal(a.prefill(q, kc, vc, bt, cl, starts), out)


def test_chunks_many_short_pieces_repeatedly():
    """Row tiles of one to four key tiles, one or two halves of rows each: every end of a piece has its own wait, which no
    delay of a warp may carry past its barrier."""
    from aitherkvcache_b200 import _lib
    g = torch.Generator().manual_seed(3)
    new = torch.randint(0, 9, (380,), generator=g).tolist()
    new[::7] = [100] * len(new[::7])
    lens = [n + int(x) for n, x in zip(new, torch.randint(0, 500, (380,), generator=g))]
    for D, bs in ((64, 16), (128, 32)):
        q, kc, vc, bt, cl, starts = make(lens, new, 4, 2, D, bs, torch.float16, seed=3, stale=math.nan)
        a = attn(4, 2, D)
        out = a.prefill(q, kc, vc, bt, cl, starts)
        check(out, q, kc, vc, bt, cl, starts)
        for _ in range(200):
            assert torch.equal(a.prefill(q, kc, vc, bt, cl, starts), out)
    assert _lib.device_status()["attn_window"] == 0


@pytest.mark.parametrize("D,bs", [(64, 32), (128, 16), (128, 8), (64, 256)])
@pytest.mark.parametrize("window", [0, 3, 130, 1000])
def test_chunks_of_few_rows(D, bs, window):
    """Few rows per sequence: the two halves take alternate key tiles of the same rows.  Ends just behind a key tile's edge
    leave rows that see nothing of the last tile, windows leave rows that see nothing of the others."""
    lens = [1, 128, 129, 130, 131, 133, 256, 257, 259, 384, 385, 390, 1030, 3333, 12000, 5]
    new = [1, 1, 1, 4, 7, 9, 2, 3, 9, 1, 8, 8, 9, 5, 3, 5]
    run_chunks(lens, new, 14, 2, D, bs, torch.bfloat16, window=window, seed=bs + window, scale_q=2.0)


@pytest.mark.parametrize("D,bs", [(64, 16), (128, 32), (256, 16)])
@pytest.mark.parametrize("new", [1, 3, 150])
def test_chunks_pages_that_have_left_the_window(D, bs, new):
    """A cache of sliding windows gives its pages back: what lies before the first window of a chunk may be anything."""
    lens, window = [999, 130, 400, 700], 100
    q, kc, vc, bt, cl, starts = make(lens, [new if n >= new else n for n in lens], 8, 2, D, bs, torch.bfloat16, seed=new, stale=math.nan)
    want, bound = od.attention(q, kc, vc, bt, cl.tolist(), starts.tolist(), 1 / math.sqrt(D), window)
    for s, n in enumerate(lens):
        first = n - (new if n >= new else n) + 1 - window           # the first key that a row sees
        for j in range(max(first, 0)):
            kc[bt[s, j // bs], j % bs] = vc[bt[s, j // bs], j % bs] = math.nan if j % 2 else math.inf
    out = attn(8, 2, D, sliding_window=window).prefill(q, kc, vc, bt, cl, starts)
    assert bool(((out.double() - want).abs() <= bound).all())
    if new == 1:
        out = attn(8, 2, D, sliding_window=window).forward(q, kc, vc, bt, cl)
        assert bool(((out.double() - want).abs() <= bound).all())


def test_no_blocks_and_no_tokens():
    """Block tables without columns, sequences without tokens, calls without rows."""
    for D in (64, 128, 256):
        kc, vc = (torch.full((3, 16, 2, D), math.nan, dtype=torch.float16, device="cuda") for _ in range(2))
        q = torch.randn(4, 4, D, device="cuda").half()
        a = attn(4, 2, D)
        none, zeros = torch.zeros(4, 0, dtype=torch.int32, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
        lens = torch.tensor([5, 0, 1, 9], dtype=torch.int32, device="cuda")      # clamped to what the table addresses
        starts = torch.tensor([0, 1, 1, 3, 4], dtype=torch.int32, device="cuda")
        assert bool((a.forward(q, kc, vc, none, lens) == 0).all())
        assert bool((a.prefill(q, kc, vc, none, lens, starts) == 0).all())
        table = torch.zeros(4, 1, dtype=torch.int32, device="cuda")
        assert bool((a.forward(q, kc, vc, table, zeros) == 0).all())
        assert bool((a.prefill(q, kc, vc, table, zeros, starts) == 0).all())
        assert a.forward(q[:0], kc, vc, table, zeros).shape == (0, 4, D)
        assert a.prefill(q[:0], kc, vc, table, zeros, zeros[:1]).shape == (0, 4, D)
        assert bool((a.prefill(q, kc, vc, table, zeros, zeros[:1]) == 0).all())
        out = torch.ones_like(q)
        a.prefill(q, kc, vc, table, zeros, starts[:3], out=out)
        assert bool((out[:1] == 0).all()) and bool((out[1:] == 1).all())


def test_chunks_of_many_keys():
    """Keys and values of 245 MB under few row tiles each."""
    run_chunks([20000, 300, 25000, 14700], [70, 300, 130, 1], 16, 8, 128, 16, torch.float16, seed=12)


def test_chunks_of_many_row_tiles_in_rounds():
    """Keys and values of 146 MB that eight row tiles and more read: three rounds, which begin between the KV heads of a
    sequence, among sequences that do not count towards them."""
    run_chunks([30000, 300, 40000, 900], [130, 20, 150, 3], 64, 4, 128, 16, torch.float16, seed=13)


def test_chunks_past_32_bit_offsets():
    nb = (1 << 31) // (16 * 8 * 128) + 64
    kc, vc = (torch.zeros(nb, 16, 8, 128, dtype=torch.float16, device="cuda") for _ in range(2))
    g = torch.Generator().manual_seed(0)
    bt = torch.tensor([[nb - 1, 0, nb - 40], [3, nb - 2, 5]], dtype=torch.int32)
    for b in bt.flatten().tolist():
        kc[b] = torch.randn(16, 8, 128, generator=g).half().cuda()
        vc[b] = torch.randn(16, 8, 128, generator=g).half().cuda()
    q = torch.randn(50, 16, 128, generator=g).half().cuda()
    cl, starts = torch.tensor([48, 41], dtype=torch.int32).cuda(), torch.tensor([0, 30, 50], dtype=torch.int32).cuda()
    out = attn(16, 8, 128).prefill(q, kc, vc, bt.cuda(), cl, starts)
    check(out, q, kc, vc, bt.cuda(), cl, starts)


def test_chunks_graph_replay_and_streams():
    lens, new = [700, 20, 1800], [100, 20, 130]
    q, kc, vc, bt, cl, starts = make(lens, new, 32, 8, 128, 16, torch.float16, seed=9)
    a = attn(32, 8, 128)
    a.prefill(q, kc, vc, bt, cl, starts)
    graphs = []
    for _ in range(2):
        o = torch.empty_like(q)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            a.prefill(q, kc, vc, bt, cl, starts, out=o)
        graphs.append((graph, o, torch.cuda.Stream()))
    for step in range(3):
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(step)).half())
        cl.add_(-3)
        want = a.prefill(q, kc, vc, bt, cl, starts)
        for graph, o, s in graphs:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                graph.replay()
        for graph, o, s in graphs:
            s.synchronize()
            assert torch.equal(o, want)
    check(want, q, kc, vc, bt, cl, starts)


def test_chunks_a_wait_that_runs_out_is_reported():
    """Test hook: CTA 0 withholds the scores of key tile 1; its waits run out, the status word says so, nothing hangs, and
    the next call is whole again."""
    from aitherkvcache_b200 import _lib
    q, kc, vc, bt, cl, starts = make([600], [300], 8, 2, 128, 16, torch.float16, seed=1)
    a = attn(8, 2, 128)
    want = a.prefill(q, kc, vc, bt, cl, starts)
    assert _lib.device_status(reset=True)["attn_window"] == 0
    _lib.check(_lib.lib().akv_debug_tc_withhold(3, 1), "hook")
    try:
        a.prefill(q, kc, vc, bt, cl, starts)
        assert _lib.device_status(reset=True)["attn_window"] == 2
    finally:
        _lib.check(_lib.lib().akv_debug_tc_withhold(3, -1), "hook")
    assert torch.equal(a.prefill(q, kc, vc, bt, cl, starts), want)
    assert _lib.device_status()["attn_window"] == 0


@pytest.mark.parametrize("lens,new,qh,kvh,D", [([20000], [5], 8, 1, 128), ([17000, 3, 9001], [70, 3, 40], 16, 2, 64), ([12345], [100], 32, 8, 128),
                                               ([8300], [1], 1, 1, 64), ([9000, 8200], [64, 130], 4, 1, 128)])
def test_chunks_cut_into_many_parts(lens, new, qh, kvh, D):
    """Few row tiles of long sequences: every one is cut into many parts, which several groups of threads join."""
    out = run_chunks(lens, new, qh, kvh, D, 16, torch.bfloat16, seed=sum(lens), scale_q=2.0)
    assert torch.equal(run_chunks(lens, new, qh, kvh, D, 16, torch.bfloat16, seed=sum(lens), scale_q=2.0), out)


@pytest.mark.parametrize("D,bs", [(128, 16), (256, 16), (64, 5)])
def test_chunks_longer_than_their_table(D, bs):
    """Lengths are clamped to what a row of the table addresses, in every path."""
    q, kc, vc, bt, cl, starts = make([3 * bs, 4 * bs], [9, 12], 4, 2, D, bs, torch.float16, seed=5, stale=math.nan)
    a = attn(4, 2, D)
    want = a.prefill(q, kc, vc, bt, torch.full_like(cl, 4 * bs), starts)
    assert torch.equal(a.prefill(q, kc, vc, bt, torch.tensor([4 * bs + 1, 1 << 40], device="cuda"), starts), want)
    assert bool((a.prefill(q, kc, vc, bt, torch.full_like(cl, -3), starts) == 0).all())


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 40, 2 ** 31 - 200, 1500])
def test_windows_that_no_sequence_fills(window):
    lens, new = [1400, 300, 1290, 1500], [300, 300, 200, 1]
    q, kc, vc, bt, cl, starts = make(lens, new, 8, 2, 128, 16, torch.float16, seed=6, stale=math.nan)
    wide, none = attn(8, 2, 128, sliding_window=window), attn(8, 2, 128)
    assert torch.equal(wide.prefill(q, kc, vc, bt, cl, starts), none.prefill(q, kc, vc, bt, cl, starts))
    assert torch.equal(wide.forward(q[:4], kc, vc, bt, cl), none.forward(q[:4], kc, vc, bt, cl))


@pytest.mark.parametrize("D,bs", [(64, 16), (128, 16), (256, 16), (128, 5)])
@pytest.mark.parametrize("n", [1, 4, 3000])
def test_no_sequences_in_memory_that_held_something_else(D, bs, n):
    """Rows of a call without sequences are behind the last one: zeros, whatever the block that the allocator hands out held."""
    q = torch.randn(n, 4, D, device="cuda").half()
    kc, vc = (torch.randn(3, bs, 2, D, device="cuda").half() for _ in range(2))
    table, none = torch.zeros(0, 2, dtype=torch.int32, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda")
    a = attn(4, 2, D)
    for starts in (torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int64, device="cuda")):
        used = torch.full_like(q, math.nan)
        del used
        assert bool((a.prefill(q, kc, vc, table, none, starts) == 0).all())
        out = torch.full((n, 6, D), 5.0, dtype=torch.float16, device="cuda")
        a.prefill(q, kc, vc, table, none, starts, out=out[:, 1:5])
        assert bool((out == 5.0).all())


@pytest.mark.parametrize("D,bs,first,seqs", [(64, 16, 3, 2), (128, 16, 700, 2), (256, 16, 5, 2), (128, 5, 5, 2), (64, 16, 40, 400), (128, 16, 9, 1)])
def test_chunks_rows_before_the_first_sequence(D, bs, first, seqs):
    """query_start_loc of a batch's later sequences: the rows of those before belong to no sequence of the call."""
    lens, new = [first + 50] + [70 + i % 5 for i in range(seqs)], [first] + [33 - i % 30 for i in range(seqs)]
    q, kc, vc, bt, cl, starts = make(lens, new, 4, 2, D, bs, torch.float16, seed=D + first, tail=6)
    a = attn(4, 2, D)
    want = a.prefill(q, kc, vc, bt, cl, starts)
    used = torch.full_like(q, math.nan)
    del used
    out = a.prefill(q, kc, vc, bt[1:], cl[1:], starts[1:])
    assert bool((out[:first] == 0).all()) and bool((out[-6:] == 0).all())
    want[:first] = 0
    _, bound = od.attention(q, kc, vc, bt, cl.tolist(), starts.tolist(), 1 / math.sqrt(D), 0)
    # both are within the bound of the same values (their cuts may differ)
    assert bool(((out.double() - want.double()).abs() <= 2 * bound)[first:-6].all())
    out = torch.full((q.shape[0], 6, D), 5.0, dtype=torch.float16, device="cuda")
    a.prefill(q, kc, vc, bt[1:], cl[1:], starts[1:], out=out[:, 1:5])
    assert bool((out[:first] == 5.0).all()) and bool((out[-6:] == 5.0).all()) and bool((out[:, 0] == 5.0).all())
    assert bool(((out[:, 1:5].double() - want.double()).abs() <= 2 * bound)[first:-6].all())


@pytest.mark.parametrize("D,bs", [(64, 16), (128, 16), (256, 16), (128, 5)])
@pytest.mark.parametrize("n", [1, 3])
def test_queries_that_start_anywhere(D, bs, n):
    """A contiguous query off the 16-byte boundaries, one token of an odd pitch and heads of one element's stride: the same
    bits as from a query of its own, in both forms."""
    H = 2
    lens, new = [70] + [33] * (n - 1), [1] * n
    for QH in (8, 2):
        q, kc, vc, bt, cl, starts = make(lens, new, QH, H, D, bs, torch.float16, seed=D + n)
        a = attn(QH, H, D)
        want, chunk = a.forward(q, kc, vc, bt, cl), a.prefill(q, kc, vc, bt, cl, starts)
        wide = torch.randn(n * (QH * D + 3) + 16, device="cuda").half()
        for pitch, offset in ((QH * D, 1), (QH * D, 4), (QH * D + 3, 0), (QH * D + 3, 5)):
            at = wide.as_strided((n, QH, D), (pitch, D, 1), offset)
            at.copy_(q)
            assert torch.equal(a.forward(at, kc, vc, bt, cl), want)
            assert torch.equal(a.prefill(at, kc, vc, bt, cl, starts), chunk)
    # one query head and one KV head, whose strides say nothing; in the output too
    q, kc, vc, bt, cl, starts = make(lens, new, 1, 1, D, bs, torch.float16, seed=D)
    a = attn(1, 1, D)
    want, chunk = a.forward(q, kc, vc, bt, cl), a.prefill(q, kc, vc, bt, cl, starts)
    q1, k1, v1 = q.as_strided(q.shape, (D, 1, 1)), *(x.as_strided(x.shape, (x.stride(0), x.stride(1), 7, 1)) for x in (kc, vc))
    out = torch.full((n, D), 5.0, dtype=torch.float16, device="cuda")
    assert torch.equal(a.forward(q1, k1, v1, bt, cl, out=out.as_strided((n, 1, D), (D, 3, 1))), want) and torch.equal(out, want[:, 0])
    out.fill_(5.0)
    assert torch.equal(a.prefill(q1, k1, v1, bt, cl, starts, out=out.as_strided((n, 1, D), (D, 3, 1))), chunk) and torch.equal(out, chunk[:, 0])
    assert torch.equal(a.forward(q1, k1, v1, bt, cl), want) and torch.equal(a.prefill(q1, k1, v1, bt, cl, starts), chunk)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,QH", [(64, 4), (64, 16), (128, 8), (256, 2)])
@pytest.mark.parametrize("at", [0, 20000, 39990])
def test_many_small_weights_beside_a_large_one(dtype, D, QH, at):
    """One key takes nearly all of the weight, 40000 others e^-18 = 2^-26 of it each, and only theirs have values: what they
    add up to must not be lost, although each is below the smallest step of fp16 (2^-24).

    Bound, relative to the result: a weight is rounded to the type: u, and for fp16 half a step 2^-25 of 2^-26 times the
    factor 2^7 that weights carry there, 2^-6; the exponential 2^-21 and the score (its error is 64 to 256 additions of zeros, one product and the
    reference's subtraction, 2^-22 of 26: 2^-17); float32 sums of n terms above and below, 2 n 2^-23; u of the result."""
    n, new, bs = 40000, 150, 16
    blocks = n // bs
    kc, vc = torch.zeros(blocks, bs, 1, D, dtype=dtype, device="cuda"), torch.ones(blocks, bs, 1, D, dtype=dtype, device="cuda")
    kc[:, :, 0, 3] = -18.0
    kc[at // bs, at % bs, 0, 3] = 0.0
    vc[at // bs, at % bs] = 0.0
    bt = torch.arange(blocks, dtype=torch.int32, device="cuda").view(1, -1)
    q = torch.zeros(new, QH, D, dtype=dtype, device="cuda")
    q[:, :, 3] = 1.0
    a, u = attn(QH, 1, D, scale=1.0), torch.finfo(dtype).eps / 2
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")

    def near(out, keys):
        seen = (keys > at).double()      # rows that do not see the large key: all ones
        rest = (keys - seen) * math.exp(-18.0)
        want = torch.where(seen > 0, rest / (1 + rest), torch.ones_like(rest))[:, None, None]
        bound = want * (2 * u + 2.0 ** -6 + 2.0 ** -21 + 2.0 ** -16 + 2 * n * 2.0 ** -23) + 2.0 ** -25
        assert bool(((out.double() - want).abs() <= bound).all()), (out.flatten()[:3].tolist(), want.flatten()[:3].tolist())

    full = torch.full((1,), n, dtype=torch.float64, device="cuda")
    near(a.forward(q[:1], kc, vc, bt, lens), full)
    for m in (1, 3, new):
        starts = torch.tensor([0, m], dtype=torch.int32, device="cuda")
        near(a.prefill(q[:m], kc, vc, bt, lens, starts), full - m + 1 + torch.arange(m, device="cuda"))


def test_scratch_of_few_tokens_over_a_large_pool():
    """One drafted token over a pool of 300 MB takes the scratch of one round; more tokens may take four."""
    nb = 4600
    kc, vc = (torch.randn(nb, 16, 8, 128, device="cuda").half() for _ in range(2))
    bt = torch.randperm(nb, generator=torch.Generator().manual_seed(0))[:4500].view(1, -1).int().cuda()
    a, cl = attn(32, 8, 128), torch.tensor([72000], dtype=torch.int32, device="cuda")
    for n, most in ((1, 45 << 20), (448, 45 << 20), (449, 170 << 20)):
        q = torch.randn(n, 32, 128, device="cuda").half()
        starts = torch.tensor([0, n], dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        out = a.prefill(q, kc, vc, bt, cl, starts)
        assert torch.cuda.max_memory_allocated() - before - out.numel() * 2 <= most
        if n == 1:
            check(out, q, kc, vc, bt, cl, starts)
