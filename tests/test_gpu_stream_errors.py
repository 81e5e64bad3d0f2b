"""What a kernel-side wait that ran out means for later calls: the error word of its stream, and nobody else's, is reported
once.  The words are written here by the host; no wait runs out."""
import ctypes

import pytest

pytestmark = pytest.mark.gpu

TIMEOUT, MISALIGNED = 1, 2  # what the kernels write


@pytest.fixture(scope="module")
def torch_cuda():
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch


def _word(stream):
    import cudasep

    p = ctypes.POINTER(ctypes.c_int)()
    assert cudasep.lib().mbr_op_stream_error_word(stream.cuda_stream, ctypes.byref(p)) == 0
    return p


def _calls(torch, dtype):
    """A call of each attention kernel."""
    import cudasep

    q = torch.randn((1, 200, 2, 64), device="cuda").to(dtype)
    cache = cudasep.KVCache.empty(1, 2, 9000, 64, dtype)
    cache.k.normal_(), cache.v.normal_()
    length = torch.full((1,), 9000, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    return [lambda **kw: cudasep.op_window_attention(q, q, q, right=0, **kw),
            lambda **kw: cudasep.op_window_attention(q[:, :3], q, q, right=0, **kw),
            lambda **kw: cudasep.op_cache_attention(q[:, :1], cache, length, **kw)]


@pytest.mark.parametrize("dtype", ["float32", "float16"])
def test_an_error_belongs_to_its_stream(torch_cuda, dtype):
    torch = torch_cuda
    import cudasep

    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    wa, wb = _word(a), _word(b)
    assert ctypes.addressof(wa.contents) != ctypes.addressof(wb.contents)
    for call in _calls(torch, getattr(torch, dtype)):
        with torch.cuda.stream(a):
            want = call()
        a.synchronize()
        wa[0] = TIMEOUT
        with torch.cuda.stream(b):
            got = call()  # not its error
        b.synchronize()
        assert torch.equal(got, want) and wa[0] == TIMEOUT and wb[0] == 0
        with torch.cuda.stream(a):
            with pytest.raises(cudasep.MBRError) as e:
                call()
            assert e.value.code == 6 and wa[0] == 0
            got = call()
        cudasep.op_stream_check(a)
        assert torch.equal(got, want)


def test_a_check_reports_once_and_tells_the_codes_apart(torch_cuda):
    torch = torch_cuda
    import cudasep

    for stream in (torch.cuda.Stream(), torch.cuda.default_stream()):
        w = _word(stream)
        cudasep.op_stream_check(stream)
        for code, status in ((TIMEOUT, 6), (MISALIGNED, 2)):
            w[0] = code
            with pytest.raises(cudasep.MBRError) as e:
                cudasep.op_stream_check(stream)
            assert e.value.code == status and w[0] == 0
            cudasep.op_stream_check(stream)


def test_graph_replays_are_checked(torch_cuda):
    """Replays report to the word of the captured stream, and run again once it is cleared."""
    torch = torch_cuda
    import cudasep

    calls = _calls(torch, torch.bfloat16)
    want = [c() for c in calls]
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        outs = [c() for c in calls]
    w = _word(side)
    for _ in range(2):
        w[0] = TIMEOUT
        graph.replay()
        torch.cuda.synchronize()
        with pytest.raises(cudasep.MBRError):
            cudasep.op_stream_check(side)
        for t in outs:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        cudasep.op_stream_check(side)
        assert all(torch.equal(x, y) for x, y in zip(outs, want))
