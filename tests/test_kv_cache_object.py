"""A KVCache is tied to the tensors it was made from: its attributes cannot be set to others (the calls use addresses taken
at its creation), and copies and pickles take the copied tensors' addresses.  The extension that looks at the tensors
accepts CUDA tensors only, so a stand-in takes its place here; the GPU test below uses the real one."""
import copy
import pickle

import pytest
import torch


class _StandIn:
    @staticmethod
    def cache_fields(k, v, k_scale, v_scale, sinks):
        return (b"%d %d" % (k.data_ptr(), v.data_ptr()), k.dtype, 0, k.shape[0], k.shape[1], k.shape[3],
                k.shape[2] - sinks, 0)


def _check(cache, field):
    import cudasep

    for name in ("k", "v", "k_scale", "v_scale", "sinks", "ring", "dtype", "dev", "desc"):
        with pytest.raises(AttributeError):
            setattr(cache, name, cache.k.clone())
    for make in (copy.deepcopy, lambda c: pickle.loads(pickle.dumps(c))):
        other = make(cache)
        assert isinstance(other, cudasep.KVCache) and torch.equal(other.k, cache.k) and other.sinks == cache.sinks
        assert other.k.data_ptr() != cache.k.data_ptr() and field(other) == (other.k.data_ptr(), other.v.data_ptr())
    same = copy.copy(cache)
    assert same.k is cache.k and field(same) == field(cache) == (cache.k.data_ptr(), cache.v.data_ptr())


def test_a_cache_is_tied_to_its_tensors(monkeypatch):
    import cudasep

    monkeypatch.setattr(cudasep, "_CALLS", _StandIn)
    cache = cudasep.KVCache(torch.randn(2, 3, 8, 64), torch.randn(2, 3, 8, 64), sinks=2)
    _check(cache, lambda c: tuple(int(x) for x in c.desc.split()))


@pytest.mark.gpu
def test_a_cache_on_the_gpu_is_tied_to_its_tensors():
    import struct

    import cudasep

    for bits in (0, 4):
        cache = cudasep.KVCache.empty(2, 3, 8, 64, torch.float16, sinks=2, bits=bits)
        _check(cache, lambda c: struct.unpack_from("@PP", c.desc))
