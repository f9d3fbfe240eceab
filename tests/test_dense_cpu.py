"""Host side of the dense paged cache's operators: tables, argument checks, struct layouts (no GPU)."""
import ctypes
import math
import os
import re
import subprocess

import pytest
import torch

from conftest import ROOT


def test_axis_of_pairs():
    from aitherkvcache_b200.rotary import axis_of_pairs
    assert axis_of_pairs(4, None) == [0, 0, 0, 0]
    assert axis_of_pairs(6, (1, 2, 3)) == [0, 1, 1, 2, 2, 2]
    assert axis_of_pairs(8, (4, 2, 2), "cycled") == [0, 1, 2, 0, 1, 2, 0, 0]
    assert axis_of_pairs(6, (1, 3, 2), "cycled") == [0, 1, 2, 1, 2, 1]
    for bad in ((3, 2), (1, 1, 1, 1, 2), (7, -1), ()):
        with pytest.raises(ValueError):
            axis_of_pairs(6, bad)
    with pytest.raises(ValueError):
        axis_of_pairs(6, None, "other")


def test_steps_are_the_angles():
    """pos * step modulo 2^64 is pos * frequency modulo a full turn: float64 angles agree to their own rounding."""
    from aitherkvcache_b200 import RotaryPositions
    freq = [1.0, 0.5, 3.9, -2.0, 1e-7, 7.1, 100.0, 1e-3]
    rope = RotaryPositions(16, inv_freq=freq, device="cpu")
    for p in (0, 1, -1, 12345, -99999, (1 << 24) + 1):
        for f, step in zip(freq, rope.steps.tolist()):
            turn = ((p * step) % (1 << 64)) / 2.0 ** 64
            t = p * f
            # the step is cut (2^-64 turns) after a float64 rounding of f / 2 pi (2^-52 of it)
            tol = 2 * math.pi * (abs(p) * 2.0 ** -64 + abs(t) * 2.0 ** -51) + 1e-12
            assert abs(math.cos(2 * math.pi * turn) - math.cos(t)) <= tol
            assert abs(math.sin(2 * math.pi * turn) - math.sin(t)) <= tol


def test_rotary_refuses():
    from aitherkvcache_b200 import RotaryPositions
    for kw in (dict(rotary_dim=7), dict(rotary_dim=18), dict(rotary_dim=0), dict(pair_layout="x"), dict(inv_freq=[1.0]),
               dict(sections=(4, 3)), dict(section_layout="x"), dict(scaling=float("nan")), dict(inv_freq=[float("inf")] * 8)):
        with pytest.raises(ValueError):
            RotaryPositions(16, device="cpu", **kw)
    rope = RotaryPositions(16, device="cpu", sections=(4, 4))
    x = torch.zeros(3, 2, 16)
    with pytest.raises(RuntimeError, match="CUDA"):
        rope.forward(x, None, torch.zeros(3, dtype=torch.int64))
    with pytest.raises(ValueError):
        rope.forward(None, None, torch.zeros(3, dtype=torch.int64))
    for bad in (torch.zeros(2), torch.zeros(3, 3), torch.zeros(2, 2)):
        with pytest.raises(ValueError):
            rope._positions(bad, 3)
    with pytest.raises(ValueError):
        rope._heads(torch.zeros(3, 2, 15), "query", 3)
    with pytest.raises(ValueError):
        rope._heads(torch.zeros(3, 16), "query", 3)
    with pytest.raises(ValueError):
        RotaryPositions._out(torch.zeros(3, 2, 16).half(), x, torch.float32, "query_out")


def test_rotary_entry_points_refuse():
    """Argument blocks that the C entry points turn into errors before any launch."""
    from aitherkvcache_b200 import _lib
    L = _lib.lib()
    good = dict(head_dim=16, rotary_dim=16, num_axes=1, adjacent=0, steps=64, axes=64, scaling=1.0)

    def params(tables, **kw):
        p = _lib.RotaryParams()
        p.tables = ctypes.pointer(_lib.RotaryTables(**tables))
        p.positions, p.num_tokens, p.query, p.q_out, p.num_q_heads = 64, 1, 64, 64, 1
        for k, v in kw.items():
            setattr(p, k, v)
        return p

    assert L.akv_rotary(None) == _lib.AKV_ERR_ARG
    for t in (dict(good, rotary_dim=15), dict(good, rotary_dim=18), dict(good, head_dim=0), dict(good, num_axes=5),
              dict(good, num_axes=0), dict(good, steps=None), dict(good, num_axes=2, axes=None)):
        assert L.akv_rotary(ctypes.byref(params(t))) == _lib.AKV_ERR_ARG, t
    for kw in (dict(num_tokens=-1), dict(in_dtype=3), dict(out_dtype=-1), dict(pos_dtype=2), dict(positions=None), dict(query=None),
               dict(q_out=None), dict(num_kv_heads=2), dict(num_q_heads=-1), dict(num_kv_heads=2, key=64)):
        assert L.akv_rotary(ctypes.byref(params(good, **kw))) == _lib.AKV_ERR_ARG, kw
    assert L.akv_rotary(ctypes.byref(params(good, num_tokens=0))) == 0
    assert L.akv_rotary_kv_append(None) == _lib.AKV_ERR_ARG

    def append(**kw):
        a = _lib.RotaryAppendParams()
        a.rotary = params(good, num_kv_heads=1, key=64)
        a.value = a.slot_mapping = a.k_cache = a.v_cache = 64
        a.block_size, a.num_blocks = 16, 4
        for k, v in kw.items():
            setattr(a, k, v)
        return L.akv_rotary_kv_append(ctypes.byref(a))

    for kw in (dict(block_size=0), dict(num_blocks=-1), dict(slot_dtype=7), dict(slot_mapping=None), dict(value=None),
               dict(k_cache=None), dict(v_cache=None)):
        assert append(**kw) == _lib.AKV_ERR_ARG, kw


def test_append_refuses():
    from aitherkvcache_b200 import dense_kv
    a = torch.zeros(4, 16, 2, 32)
    dense_kv._check_caches(a, a, 2, 32)
    for k, v in ((a, a[:3]), (a[:, :, :1], a[:, :, :1]), (a[..., :16], a[..., :16]), (a.transpose(2, 3), a.transpose(2, 3)), (a[0], a[0])):
        with pytest.raises(ValueError):
            dense_kv._check_caches(k, v, 2, 32)
    with pytest.raises(TypeError):
        dense_kv._check_caches(a, a.half(), 2, 32)


def test_dense_structures_match_the_header_layout(tmp_path):
    """The parameter structs of the dense cache against their ctypes mirrors: sizeof and every offset, from gcc."""
    from aitherkvcache_b200 import _lib
    pairs = {"akv_rotary_tables": _lib.RotaryTables, "akv_rotary_params": _lib.RotaryParams,
             "akv_rotary_append_params": _lib.RotaryAppendParams}
    if hasattr(_lib, "DenseAttnParams"):
        pairs["akv_dense_attn_params"] = _lib.DenseAttnParams
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "akv_b200.h"', "int main(void) {"]
    for cname, st in pairs.items():
        lines.append('printf("%s %%zu", sizeof(%s));' % (cname, cname))
        lines += ['printf(" %%zu", offsetof(%s, %s));' % (cname, f) for f, _ in st._fields_]
        lines.append('printf("\\n");')
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["return 0;", "}"]))
    subprocess.run(["gcc", "-std=c99", "-I", os.path.join(ROOT, "include"), "-o", str(exe), str(src)], check=True)
    header = open(os.path.join(ROOT, "include", "akv_b200.h")).read()
    for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.strip().splitlines():
        cname, size, *offs = line.split()
        st = pairs[cname]
        assert ctypes.sizeof(st) == int(size), cname
        assert [getattr(st, f).offset for f, _ in st._fields_] == [int(o) for o in offs], cname
        body = re.sub(r"/\*.*?\*/", "", re.search(r"typedef struct %s \{(.*?)\} %s;" % (cname, cname), header, re.S).group(1), flags=re.S)
        names = [re.findall(r"[A-Za-z_]\w*", part)[-1] for decl in body.split(";") if decl.strip() for part in decl.split(",")]
        assert names == [f for f, _ in st._fields_], cname


def test_attention_refuses():
    from aitherkvcache_b200 import DensePagedAttention
    for args, kw in (((96, 8, 2), {}), ((128, 7, 2), {}), ((128, 0, 1), {}), ((128, 4, 0), {}), ((128, 4, 2), dict(sliding_window=-1)),
                     ((128, 4, 2), dict(scale=0.0)), ((128, 4, 2), dict(scale=-1.0)), ((128, 4, 2), dict(scale=math.inf)),
                     ((128, 4, 2), dict(scale=math.nan))):
        with pytest.raises(ValueError):
            DensePagedAttention(*args, **kw)
    a = DensePagedAttention(64, 4, 2)
    q, c = torch.zeros(3, 4, 64).half(), torch.zeros(5, 16, 2, 64).half()
    bt, n, st = torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    for call in (lambda: a.forward(q, c, c, bt, n), lambda: a.prefill(q, c, c, bt, n, st)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    good = (q, c, c, bt, n, (0, 0), 3, None)
    a._values(*good)
    for at, bad in ((0, q[:, :3]), (0, q[0]), (1, c[:, :, :1]), (2, c[:4]), (3, bt[:2]), (3, bt[0]), (4, n[:2]), (4, bt), (7, q[:2]), (7, q.transpose(1, 2))):
        with pytest.raises(ValueError):
            a._values(*good[:at], bad, *good[at + 1:])
    for at, bad in ((0, q.float()), (0, q.bfloat16()), (3, bt.short()), (4, n.float())):
        with pytest.raises(TypeError):
            a._values(*good[:at], bad, *good[at + 1:])


def test_attention_entry_points_refuse():
    """Argument blocks that the C entry points turn into errors before any launch."""
    from aitherkvcache_b200 import _lib
    L = _lib.lib()

    def call(name, **kw):
        p = _lib.DenseAttnParams()
        for f in ("query", "k_cache", "v_cache", "block_tables", "seq_lens", "query_start_loc", "out", "workspace"):
            setattr(p, f, 256)
        p.q_stride_tok = p.out_stride_tok = p.k_stride_pos = p.v_stride_pos = 256
        p.q_stride_head = p.out_stride_head = p.k_stride_head = p.v_stride_head = 128
        p.k_stride_blk = p.v_stride_blk = 4096
        p.num_seqs, p.num_tokens, p.num_q_heads, p.num_kv_heads, p.head_dim, p.block_size = 2, 4, 2, 2, 128, 16
        p.max_blocks_per_seq, p.num_blocks, p.scale = 3, 9, 1.0
        for k, v in kw.items():
            setattr(p, k, v)
        return getattr(L, name)(ctypes.byref(p))

    for name in ("akv_dense_paged_attn", "akv_dense_prefill_attn"):
        assert getattr(L, name)(None) == _lib.AKV_ERR_ARG
        assert call(name) == _lib.AKV_ERR_WORKSPACE      # everything but the workspace is right
        for kw in (dict(num_seqs=-1), dict(num_q_heads=3), dict(num_kv_heads=0), dict(block_size=0), dict(num_blocks=-1), dict(window=-1),
                   dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(bt_dtype=2),
                   dict(sl_dtype=3), dict(qs_dtype=-1), dict(query=None), dict(out=None), dict(seq_lens=None), dict(block_tables=None),
                   dict(k_cache=None), dict(v_cache=None), dict(num_blocks=0), dict(query=264), dict(out=264), dict(k_cache=264),
                   dict(k_stride_pos=260), dict(v_stride_head=4), dict(q_stride_tok=258), dict(out_stride_head=1)):
            assert call(name, **kw) == _lib.AKV_ERR_ARG, (name, kw)
        for kw in (dict(head_dim=96), dict(dtype=_lib.AKV_F32), dict(max_blocks_per_seq=1 << 28)):
            assert call(name, **kw) == _lib.AKV_ERR_UNSUPPORTED, (name, kw)
        assert call(name, num_seqs=0) == 0
    assert call("akv_dense_paged_attn", num_tokens=1) == _lib.AKV_ERR_ARG
    assert call("akv_dense_prefill_attn", query_start_loc=None) == _lib.AKV_ERR_ARG
    for kw in (dict(head_dim=256), dict(block_size=12), dict(num_q_heads=258), dict(max_blocks_per_seq=0)):
        assert call("akv_dense_prefill_attn", **kw) == _lib.AKV_ERR_UNSUPPORTED, kw
    assert L.akv_dense_prefill_attn_workspace_bytes(8, 128, 10, 16, 1, 10) > 0
    small, large = (L.akv_dense_prefill_attn_workspace_bytes(8, 128, n, 16, 4, 1 << 20) for n in (100, 1 << 20))
    assert large == 4 * small or large > 3.9 * small      # up to four rounds


def test_chunk_entry_point_without_sequences():
    """Rows of a call without sequences are zeroed (zero_tail): their output and the start must be there."""
    from aitherkvcache_b200 import _lib
    L = _lib.lib()
    p = _lib.DenseAttnParams()
    p.num_tokens, p.num_q_heads, p.num_kv_heads, p.head_dim, p.block_size, p.max_blocks_per_seq, p.num_blocks, p.scale = 4, 2, 2, 128, 16, 3, 9, 1.0
    assert L.akv_dense_prefill_attn(ctypes.byref(p)) == 0      # nothing asked for
    p.zero_tail = 1
    assert L.akv_dense_prefill_attn(ctypes.byref(p)) == _lib.AKV_ERR_ARG
    p.out = 256
    assert L.akv_dense_prefill_attn(ctypes.byref(p)) == _lib.AKV_ERR_ARG
    p.num_tokens = 0
    assert L.akv_dense_prefill_attn(ctypes.byref(p)) == 0


def test_backend_window_of_uncompressed_layers():
    from aitherkvcache_b200.vllm.backend import TurboQuantImplBase
    impl = TurboQuantImplBase()
    impl._tq_setup(8, 128, 0.1, 2, "auto")
    cache = torch.zeros(1, dtype=torch.bfloat16)
    for value, window in ((None, 0), ((-1, -1), 0), ((127, 0), 128), (64, 64), ((0, 0), 1)):
        impl.sliding_window = value
        attn = impl._dense_attention(cache)
        assert (attn.sliding_window, attn.scale, attn.head_dim, attn.num_kv_heads) == (window, 0.1, 128, 2)


class _Enum:
    value = "encoder_only"


@pytest.mark.parametrize("name,value", [("logits_soft_cap", 30.0), ("alibi_slopes", [0.5] * 8), ("sinks", torch.zeros(8)),
                                        ("attn_type", "encoder"), ("attn_type", _Enum()), ("chunk_lookback", 1)])
def test_backend_refuses_what_uncompressed_layers_do_not_compute(name, value):
    """Scale and sliding window are all that the 16-bit path applies: an impl that asks for more is refused by name, in
    every method that meets the cache, before anything is written or launched."""
    from aitherkvcache_b200.vllm.backend import TurboQuantImplBase
    cache = torch.zeros(3, 2, 16, 2, 128, dtype=torch.bfloat16)
    q, k, n = torch.zeros(4, 8, 128, dtype=torch.bfloat16), torch.zeros(4, 2, 128, dtype=torch.bfloat16), torch.zeros(4, dtype=torch.int64)
    impl = TurboQuantImplBase()
    impl._tq_setup(8, 128, 0.1, 2, "auto")
    setattr(impl, name, value)
    for run in (lambda: impl.do_kv_cache_update(None, k, k, cache, n), lambda: impl.rope_and_kv_cache_update(None, q, k, k, n, None, cache, n),
                lambda: impl._attend(None, q, q, cache, n[:, None], n), lambda: impl._prefill(None, q, q, cache, None)):
        with pytest.raises(NotImplementedError, match=name):
            run()


def test_backend_takes_uncompressed_layers_without_them():
    """What vLLM's impls hold where none of these is asked for."""
    from aitherkvcache_b200.vllm.backend import TurboQuantImplBase
    cache, k, n = torch.zeros(3, 2, 16, 2, 128, dtype=torch.bfloat16), torch.zeros(4, 2, 128, dtype=torch.bfloat16), torch.zeros(4, dtype=torch.int64)
    for cap, kind in ((None, "decoder"), (0, "decoder"), (0.0, None)):
        impl = TurboQuantImplBase()
        impl._tq_setup(8, 128, 0.1, 2, "auto")
        impl.logits_soft_cap, impl.alibi_slopes, impl.sinks, impl.attn_type, impl.chunk_lookback = cap, None, None, kind, -1
        with pytest.raises(RuntimeError, match="CUDA tensors only"):      # as far as a host without a GPU gets
            impl.do_kv_cache_update(None, k, k, cache, n)


def test_backend_under_vllm_reads_its_impl(monkeypatch):
    """The attributes are those that vLLM's own constructor sets."""
    pytest.importorskip("vllm")
    from aitherkvcache_b200.vllm.backend import TurboQuantBackend
    for name in ("AITHER_TQ_MODE", "AITHER_TQ_BITS"):
        monkeypatch.delenv(name, raising=False)
    make = lambda **kw: TurboQuantBackend.get_impl_cls()(num_heads=8, head_size=128, scale=0.1, num_kv_heads=2, sliding_window=None,  # noqa: E731
                                                         kv_cache_dtype="auto", **{"alibi_slopes": None, **kw})
    cache = torch.zeros(3, 2, 16, 2, 128, dtype=torch.bfloat16)
    assert make()._dense(cache) and not make()._dense(cache.view(torch.uint8))
    for kw in (dict(logits_soft_cap=50.0), dict(alibi_slopes=[0.5] * 8), dict(sinks=torch.zeros(8))):
        with pytest.raises(NotImplementedError, match=next(iter(kw))):
            make(**kw)._dense(cache)
        assert not make(**kw)._dense(cache.view(torch.uint8))


@pytest.mark.parametrize("name", ["tq-t4nc", "tq-t3nc", "tq-t2nc", "tq-t35nc", "tq-t25nc"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_backend_refuses_16_bit_caches_of_layers_with_a_compressed_dtype(name, dtype):
    """A layer that was set up with a compressed cache dtype is not stored uncompressed without a word."""
    from aitherkvcache_b200.vllm.backend import TurboQuantImplBase
    cache, n = torch.zeros(3, 2, 16, 2, 128, dtype=dtype), torch.zeros(4, dtype=torch.int64)
    q, k = torch.zeros(4, 8, 128, dtype=dtype), torch.zeros(4, 2, 128, dtype=dtype)
    impl = TurboQuantImplBase()
    impl._tq_setup(8, 128, 0.1, 2, name)
    for run in (lambda: impl.do_kv_cache_update(None, k, k, cache, n), lambda: impl.rope_and_kv_cache_update(None, q, k, k, n, None, cache, n),
                lambda: impl._attend(None, q, q, cache, n[:, None], n), lambda: impl._prefill(None, q, q, cache, None)):
        with pytest.raises(TypeError, match=name):
            run()


@pytest.mark.parametrize("env,value,words", [("AITHER_TQ_MODE", "tq35", 1), ("AITHER_TQ_BITS", "3", 1), (None, "", 0)])
def test_backend_says_once_that_a_layer_stays_uncompressed(monkeypatch, caplog, env, value, words):
    """Where the environment names a codec and the layer's dtype does not, a 16-bit cache is taken and said so, once."""
    from aitherkvcache_b200.vllm import backend
    for name in ("AITHER_TQ_MODE", "AITHER_TQ_BITS"):
        monkeypatch.delenv(name, raising=False)
    if env:
        monkeypatch.setenv(env, value)
    monkeypatch.setattr(backend._LayerState, "told", set())
    impl = backend.TurboQuantImplBase()
    impl._tq_setup(8, 128, 0.1, 2, "auto")
    with caplog.at_level("WARNING"):
        for _ in range(3):
            assert impl._dense(torch.zeros(3, 2, 16, 2, 128, dtype=torch.bfloat16))
            assert not impl._dense(torch.zeros(3, 2, 16, 2, 128, dtype=torch.uint8))
    assert sum("uncompressed" in r.getMessage() for r in caplog.records) == words


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_backend_rotating_update_of_a_padded_batch(monkeypatch, index):
    """Tokens behind the slots' length are padding: turned, and without a slot.  Other batches go through as they are."""
    from aitherkvcache_b200 import dense_kv
    from aitherkvcache_b200.vllm.backend import TurboQuantImplBase
    seen = []
    monkeypatch.setattr(dense_kv, "rotary_kv_append", lambda *a: seen.append(a) or "query")
    impl = TurboQuantImplBase()
    impl._tq_setup(8, 128, 0.1, 2, "auto")
    cache = torch.zeros(3, 2, 16, 2, 128, dtype=torch.bfloat16)
    q, k, v, pos = torch.zeros(9, 8, 128), torch.zeros(9, 2, 128), torch.zeros(9, 2, 128), torch.zeros(3, 9, dtype=torch.int64)
    for n in (6, 9, 0):
        slots = torch.arange(n, dtype=index)
        assert impl.rope_and_kv_cache_update(None, q, k, v, pos, "rope", cache, slots, "out") == "query"
        got = seen.pop()
        assert got[0] is q and got[1] is k and got[2] is v and got[3] is pos and got[7:] == ("rope", "out")
        assert got[4].dtype == index and got[4].tolist() == list(range(n)) + [-1] * (9 - n)
        assert n < 9 or got[4] is slots


def test_rows_on_16_byte_boundaries():
    """Which query rows are readable as they are: strides of dimensions with one element say nothing."""
    from aitherkvcache_b200 import DensePagedAttention
    flat = torch.zeros(4096, dtype=torch.float16)
    assert flat.data_ptr() % 16 == 0
    rows16 = DensePagedAttention._rows16
    for shape, strides, offset, good in (((3, 4, 64), (256, 64, 1), 0, True), ((3, 4, 64), (264, 64, 1), 8, True), ((3, 4, 64), (260, 64, 1), 0, False),
                                         ((3, 4, 64), (256, 64, 1), 1, False), ((3, 4, 64), (256, 64, 1), 4, False), ((1, 4, 64), (257, 64, 1), 0, True),
                                         ((1, 4, 64), (257, 64, 1), 1, False), ((1, 4, 64), (0, 64, 1), 0, True), ((3, 1, 64), (64, 1, 1), 0, True),
                                         ((3, 1, 64), (65, 1, 1), 0, False), ((1, 1, 64), (3, 5, 1), 0, True), ((3, 4, 64), (0, 64, 1), 0, False),
                                         ((3, 4, 64), (64, 0, 1), 0, False), ((1, 4, 64), (0, 65, 1), 0, False), ((3, 4, 32), (256, 64, 2), 0, False)):
        assert rows16(flat.as_strided(shape, strides, offset)) is good, (shape, strides, offset)


def test_attention_entry_points_ignore_strides_of_single_elements():
    """A dimension of one element may have any stride: only the workspace is missing."""
    from aitherkvcache_b200 import _lib
    L = _lib.lib()
    for name in ("akv_dense_paged_attn", "akv_dense_prefill_attn"):
        p = _lib.DenseAttnParams()
        for f in ("query", "k_cache", "v_cache", "block_tables", "seq_lens", "query_start_loc", "out", "workspace"):
            setattr(p, f, 256)
        p.num_seqs = p.num_tokens = p.num_q_heads = p.num_kv_heads = p.num_blocks = p.max_blocks_per_seq = 1
        p.head_dim, p.block_size, p.scale, p.k_stride_pos, p.v_stride_pos = 128, 16, 1.0, 128, 128
        p.q_stride_tok, p.q_stride_head, p.out_stride_tok, p.out_stride_head = 257, 1, 3, 129
        p.k_stride_blk, p.k_stride_head, p.v_stride_blk, p.v_stride_head = 33, 1, 77, 5
        assert getattr(L, name)(ctypes.byref(p)) == _lib.AKV_ERR_WORKSPACE
        for kw in (dict(num_tokens=2), dict(num_blocks=2)):
            for f, v in kw.items():
                setattr(p, f, v)
            assert getattr(L, name)(ctypes.byref(p)) == _lib.AKV_ERR_ARG, kw
            for f in kw:
                setattr(p, f, 1)
        for heads in (dict(num_q_heads=2, q_stride_head=128), dict(num_q_heads=2, out_stride_head=128, q_stride_head=1)):
            for f, v in heads.items():
                setattr(p, f, v)
            assert getattr(L, name)(ctypes.byref(p)) == _lib.AKV_ERR_ARG, heads
            p.num_q_heads = 1


@pytest.mark.parametrize("how", ["copy", "deepcopy", "pickle", "module"])
def test_rotary_positions_are_copied(how):
    """A copy has an argument block of its own that points at its own tables, and outlives the original."""
    import copy
    import gc
    import pickle
    from aitherkvcache_b200 import RotaryPositions
    rope = RotaryPositions(32, rotary_dim=16, base=5e5, sections=(4, 3, 1), section_layout="cycled", pair_layout="adjacent", scaling=1.5, device="cpu")
    if how == "module":
        layer = torch.nn.Module()
        layer.rope = rope
        twin = copy.deepcopy(layer).rope
    else:
        twin = {"copy": copy.copy, "deepcopy": copy.deepcopy, "pickle": lambda x: pickle.loads(pickle.dumps(x))}[how](rope)
    plain = {k: v for k, v in vars(rope).items() if not k.startswith("_")}
    assert set(plain) == {k for k in vars(twin) if not k.startswith("_")}
    for k, v in plain.items():
        assert torch.equal(v, getattr(twin, k)) if isinstance(v, torch.Tensor) else v == getattr(twin, k)
    if how != "copy":
        assert twin.steps.data_ptr() != rope.steps.data_ptr() and twin.axes.data_ptr() != rope.axes.data_ptr()
    assert twin._tables_at != rope._tables_at
    del rope
    gc.collect()
    t = ctypes.cast(twin._tables_at, ctypes.POINTER(type(twin._tables))).contents
    assert (t.head_dim, t.rotary_dim, t.num_axes, t.adjacent, t.scaling) == (32, 16, 3, 1, 1.5)
    assert (t.steps, t.axes) == (twin.steps.data_ptr(), twin.axes.data_ptr())


def test_chunk_workspace_goes_by_the_call():
    """Rounds are for sequences of eight row tiles of 256 rows: calls with fewer tokens need one round's workspace, whatever the
    pool; the bound without tokens covers every call."""
    from aitherkvcache_b200 import _lib
    L = _lib.lib()
    for heads, kv, D in ((32, 8, 128), (8, 8, 64), (28, 4, 64), (128, 1, 128)):
        need = lambda n: L.akv_dense_prefill_attn_call_bytes(n, heads, kv, D, 1 << 20, 16, 4, 1 << 20)  # noqa: E731
        few = 7 * 2 * (128 // (heads // kv))
        bound = L.akv_dense_prefill_attn_workspace_bytes(kv, D, 1 << 20, 16, 4, 1 << 20)
        assert need(0) == need(1) == need(few) and need(few + 1) == need(1 << 30) == bound
        assert 3.9 * need(1) < bound <= 4 * need(1)
    for bad in ((-1, 8, 8, 64, 9, 16, 4, 9), (1, 4, 8, 64, 9, 16, 4, 9), (1, 8, 0, 64, 9, 16, 4, 9), (1, 8, 8, 64, 9, 0, 4, 9), (1, 8, 8, 64, -1, 16, 4, 9)):
        assert L.akv_dense_prefill_attn_call_bytes(*bad) == 0
