"""Windowed attention of few rows on both sides of the rule that chooses the few-token form or the tile form."""
import pytest

import stream_ref as ref
from test_gpu_stream_ops import _dt, _randn, _within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch_cuda():
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("S,N,M,H,G,D", [
    (40, 1, 90, 4, 4, 128),   # few rows in the tile form: heads past 64, more key heads than SMs
    (80, 4, 300, 8, 2, 96),
    (40, 25, 90, 4, 4, 64),   # more CTAs of 16 rows than SMs
    (30, 30, 200, 2, 2, 64),  # and fewer
])
@pytest.mark.parametrize("aligned", [True, False])
def test_few_rows_in_either_form(torch_cuda, dtype, S, N, M, H, G, D, aligned):
    """Also with an output that the tile form does not take."""
    torch = torch_cuda
    import cudasep

    dt = _dt(torch, dtype)
    q, k, v = _randn(torch, (S, N, H, D), dt, 1), _randn(torch, (S, M, G, D), dt, 2), _randn(torch, (S, M, G, D), dt, 3)
    out = torch.empty((S, N, H, D + 1 - aligned), dtype=dt, device="cuda")[..., :D]
    got = cudasep.op_window_attention(q.cuda(), k.cuda(), v.cuda(), left=50, right=0, sinks=2, out=out)
    see = ref.visible(range(M - N, M), M, 50, 0, 2)
    for s in (0, S // 2, S - 1):
        _within(got[s], *ref.attention(q[s], k[s], v[s], see, D ** -0.5, None), "few rows")
