"""The device check in front of the lean calls, on the host: nothing is launched, so stand-ins for tensors do."""
import pytest
import torch


class On:
    """What the check looks at of a tensor on CUDA device ``index`` (-1: in host memory)."""

    def __init__(self, index):
        self.index, self.is_cuda = index, index >= 0
        self.device = torch.device("cuda", index) if index >= 0 else torch.device("cpu")

    def get_device(self):
        return self.index


@pytest.mark.parametrize("where", [(-1,), (-1, -1), (-1, 0, 0), (0, -1), (0, 0, -1), (None, -1, 0), (-1, None, 1), (1, None, -1)])
def test_host_tensors_are_refused_in_every_place(where):
    from aitherkvcache_b200 import _lib
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        _lib.cuda_index(*(None if i is None else On(i) for i in where))


@pytest.mark.parametrize("where", [(0, 1), (1, 0), (None, 2, 2, 0)])
def test_two_devices_are_refused(where):
    from aitherkvcache_b200 import _lib
    with pytest.raises(RuntimeError, match="different devices"):
        _lib.cuda_index(*(None if i is None else On(i) for i in where))


def test_no_tensor_is_refused():
    from aitherkvcache_b200 import _lib
    for none in ((), (None,), (None, None)):
        with pytest.raises(RuntimeError):
            _lib.cuda_index(*none)


@pytest.mark.parametrize("where,index", [((0,), 0), ((3, 3), 3), ((None, 2, None, 2), 2)])
def test_index_of_the_one_device(where, index):
    from aitherkvcache_b200 import _lib
    assert _lib.cuda_index(*(None if i is None else On(i) for i in where)) == index


def test_host_tensors_never_reach_a_call(monkeypatch):
    """Every lean operator refuses host tensors before it asks for a stream, scratch or its entry point."""
    from aitherkvcache_b200 import DensePagedAttention, RotaryPositions, _lib, kv_append, rotary_kv_append

    def reached(*a, **k):
        raise AssertionError("a host tensor got past the check")
    monkeypatch.setattr(_lib, "call", reached)
    monkeypatch.setattr(_lib, "raw_stream", reached)
    rope, attn = RotaryPositions(64, device="cpu"), DensePagedAttention(64, 4, 2)
    x, k = torch.zeros(3, 4, 64).half(), torch.zeros(3, 2, 64).half()
    cache, pos, table = torch.zeros(5, 16, 2, 64).half(), torch.zeros(3, dtype=torch.int64), torch.zeros(3, 2, dtype=torch.int32)
    for run in (lambda: rope.forward(x, k, pos), lambda: rope.forward(None, k, pos), lambda: kv_append(k, k, pos, cache, cache),
                lambda: rotary_kv_append(x, k, k, pos, pos, cache, cache, rope), lambda: rotary_kv_append(None, k, k, pos, pos, cache, cache, rope),
                lambda: attn.forward(x, cache, cache, table, pos), lambda: attn.prefill(x, cache, cache, table, pos, torch.zeros(4, dtype=torch.int32))):
        with pytest.raises(RuntimeError, match="CUDA tensors only"):
            run()
