"""The streaming operators' `stream` argument: a torch stream, its handle, the default stream's handle 0.  What a call
allocates for itself belongs to that stream, so that later work of other streams cannot be given the memory while the call
still runs."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch_cuda():
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch


def _owner(torch, t):
    """Handle of the stream that the allocator keeps t's memory for."""
    for seg in torch.cuda.memory_snapshot():
        if seg["address"] <= t.data_ptr() < seg["address"] + seg["total_size"]:
            return seg["stream"]
    raise AssertionError("not the allocator's memory")


def _ways(torch):
    side = torch.cuda.Stream()
    return [(side, side.cuda_stream), (side.cuda_stream, side.cuda_stream), (0, 0), (torch.cuda.default_stream(), 0)]


def _split(torch):
    """A call that needs a workspace, and what it gives."""
    import cudasep

    q = torch.randn((1, 1, 2, 64), device="cuda").half()
    cache = cudasep.KVCache.empty(1, 1, 20000, 64, torch.float16)
    cache.k.normal_(), cache.v.normal_()
    length = torch.full((1,), 20000, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    return lambda **kw: cudasep.op_cache_attention(q, cache, length, **kw)


def test_a_workspace_belongs_to_the_stream_of_its_call(torch_cuda):
    torch = torch_cuda
    import cudasep

    call = _split(torch)
    want = call()
    torch.cuda.synchronize()
    for stream, handle in _ways(torch):
        w = cudasep._workspace(1 << 20, torch.device("cuda", 0), stream)
        assert _owner(torch, w) == handle
        other = torch.cuda.Stream()
        with torch.cuda.stream(other):  # another stream is the current one
            got = call(stream=stream)
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_the_split_call_needs_a_workspace(torch_cuda):
    """(else the test above shows nothing)"""
    torch = torch_cuda
    import ctypes

    import cudasep

    cache = cudasep.KVCache.empty(1, 1, 20000, 64, torch.float16)
    n = ctypes.c_int64()
    assert cudasep.lib().mbr_op_cache_attention_workspace(cache.desc, 1, 2, -1, 0, ctypes.byref(n)) == 0
    assert n.value > 0


def test_outputs_belong_to_the_stream_of_their_call(torch_cuda):
    torch = torch_cuda
    import cudasep

    q = torch.randn((2, 5, 2, 64), device="cuda").half()
    cache = cudasep.KVCache.empty(2, 2, 16, 64, torch.float16)
    pos = torch.zeros(2, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    calls = [lambda s: cudasep.op_qk_norm_rope(q, q, stream=s),
             lambda s: (cudasep.op_window_attention(q, q, q, stream=s),),
             lambda s: cudasep.op_cache_append(cache, q, q, pos, stream=s) or cudasep.op_cache_read(cache, pos, 5, stream=s),
             lambda s: (cudasep.op_cache_attention(q, cache, pos + 5, stream=s),)]
    for call in calls:
        want = call(None)
        torch.cuda.synchronize()
        for stream, handle in _ways(torch):
            other = torch.cuda.Stream()
            with torch.cuda.stream(other):
                got = call(stream)
            torch.cuda.synchronize()
            assert [_owner(torch, t) for t in got] == [handle] * len(got)
            assert all(torch.equal(a, b) for a, b in zip(got, want))
            with torch.cuda.stream(other):
                assert all(_owner(torch, t) == other.cuda_stream for t in call(None))
            torch.cuda.synchronize()
