"""The few-token attention split over several CTAs and joined by a second kernel through the workspace: every type of cache
and view, more than one row tile, ragged and empty sequences, captured, on several streams and from several threads.  Each
test asserts that its call is split (its workspace query is not zero)."""
import ctypes
import threading

import pytest

from test_gpu_stream_ops import CACHES, _cache_case, _dt, _randn, _window_case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch_cuda():
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch


def _cache_bytes(cache, tokens, H, left=-1, right=0):
    import cudasep

    n = ctypes.c_int64()
    assert cudasep.lib().mbr_op_cache_attention_workspace(cache.desc, tokens, H, left, right, ctypes.byref(n)) == 0
    return n.value


def _window_bytes(S, N, M, H, G, D, left, right, sinks, dtype):
    import cudasep

    n = ctypes.c_int64()
    code = {"fp16": cudasep.FP16, "bf16": cudasep.BF16}[dtype]
    assert cudasep.lib().mbr_op_window_attention_workspace(S, N, M, H, G, D, left, right, sinks, code, ctypes.byref(n)) == 0
    return n.value


SPLIT_CACHES = [c for c in CACHES if c[0] != "fp32"]  # fp32 caches have no such form


@pytest.mark.parametrize("dtype,bits", SPLIT_CACHES)
@pytest.mark.parametrize("S,N,H,G,D,sinks,ring,lengths,left", [
    (1, 1, 2, 1, 64, 4, 12000, [12004], -1),
    (1, 1, 1, 1, 32, 4, 12000, [20001], -1),            # the ring starts over
    (2, 6, 4, 2, 64, 0, 12000, [11999, 3], -1),         # 12 rows; a sequence with fewer tokens than rows
    (2, 5, 8, 2, 64, 3, 13000, [13500, 0], -1),         # two row tiles; an empty sequence
    (1, 10, 4, 2, 128, 17, 9000, [9100], 7000),
    (1, 10, 4, 2, 96, 17, 9000, [9017], -1),
    (1, 2, 2, 2, 96, 0, 9000, [8999], -1),
])
def test_split_cache_attention(torch_cuda, dtype, bits, S, N, H, G, D, sinks, ring, lengths, left):
    torch = torch_cuda
    import cudasep

    cache = cudasep.KVCache.empty(S, G, sinks + ring, D, _dt(torch, dtype), sinks=sinks, bits=bits)
    assert _cache_bytes(cache, N, H, left) > 0
    del cache
    _cache_case(torch, dtype, bits, S, N, H, G, D, sinks, ring, lengths, left)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("S,N,M,H,G,D,left,right,sinks,q_len,kv_len", [
    (1, 3, 9000, 4, 2, 64, -1, 0, 0, None, None),
    (3, 3, 8001, 4, 2, 64, -1, 0, 0, [3, 0, 2], [8001, 8001, 77]),
    (3, 3, 8001, 2, 1, 64, -1, 0, 0, [3, 1, 3], [0, 8000, 2]),
    (2, 12, 8001, 1, 1, 128, -1, 0, 5, None, None),
    (2, 20, 8001, 2, 2, 64, -1, 2, 5, [20, 7], [8001, 4000]),  # two row tiles
    (1, 5, 8001, 4, 1, 40, -1, 0, 0, None, None),
    (1, 1, 8001, 1, 1, 32, 6000, 0, 3, None, None),
])
def test_split_window_attention(torch_cuda, dtype, S, N, M, H, G, D, left, right, sinks, q_len, kv_len):
    assert _window_bytes(S, N, M, H, G, D, left, right, sinks, dtype) > 0
    _window_case(torch_cuda, dtype, S, N, M, H, G, D, left, right, sinks, q_len, kv_len)


def _cases(torch, dtype, bits, seed, n=2):
    """Calls that are split, with their outputs: n caches and a view."""
    import cudasep

    dt, calls = _dt(torch, dtype), []
    for i in range(n):
        cache = cudasep.KVCache.empty(2, 2, 12000, 64, dt, sinks=3, bits=bits)
        assert _cache_bytes(cache, 2, 4) > 0
        k = _randn(torch, (2, 12000, 2, 64), dt, seed + 4 * i).cuda()
        cudasep.op_cache_append(cache, k, k.flip(1), torch.zeros(2, dtype=torch.int32, device="cuda"))
        length = torch.tensor([12000, 9000 + i], dtype=torch.int32, device="cuda")
        q = _randn(torch, (2, 2, 4, 64), dt, seed + 4 * i + 1).cuda()
        calls.append(lambda out, q=q, cache=cache, length=length, **kw: cudasep.op_cache_attention(q, cache, length, out=out, **kw))
    assert _window_bytes(2, 2, 12000, 4, 2, 64, -1, 0, 0, dtype) > 0
    calls.append(lambda out, q=q, k=k, **kw: cudasep.op_window_attention(q, k, k, right=0, out=out, **kw))
    outs = [torch.empty((2, 2, 4, 64), dtype=dt, device="cuda") for _ in calls]
    torch.cuda.synchronize()
    return calls, outs


@pytest.mark.parametrize("dtype,bits", SPLIT_CACHES)
def test_split_calls_captured_and_on_other_streams(torch_cuda, dtype, bits):
    torch = torch_cuda
    calls, outs = _cases(torch, dtype, bits, 100)
    want = [call(out).clone() for call, out in zip(calls, outs)]
    assert all(torch.isfinite(w.float()).all() and w.abs().sum() > 0 for w in want)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for stream in (side, side.cuda_stream, 0):
        for call, out in zip(calls, outs):
            out.zero_()
            torch.cuda.synchronize()
            call(out, stream=stream)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for call, out in zip(calls, outs):
            call(out)
            call(out)  # the workspace's memory is used again by the calls behind
    for _ in range(5):
        for out in outs:
            out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_split_calls_from_two_threads(torch_cuda):
    """Two threads, a stream and caches each: the same bits as alone, however they overlap."""
    torch = torch_cuda
    work = [_cases(torch, "fp16", 0, 200), _cases(torch, "bf16", 4, 300)]
    want = [[call(out).clone() for call, out in zip(*w)] for w in work]
    torch.cuda.synchronize()
    bad = []

    def run(w, expect):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(40):
                    got = [call(None) for call in w[0]]
                    if not all(torch.equal(a, b) for a, b in zip(got, expect)):
                        bad.append("other bits")
        except Exception as e:
            bad.append(repr(e))

    threads = [threading.Thread(target=run, args=(w, e)) for w, e in zip(work, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_fp32_cache_with_more_rows_than_the_grid(torch_cuda):
    """A CTA takes more than one row."""
    _cache_case(torch_cuda, "fp32", 0, 60, 20, 8, 2, 8, 1, 14, [20, 0, 3, 41] * 15, 9)
