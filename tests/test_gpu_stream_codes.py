"""4-bit caches at the edges of their definition: steps below fp32's normal range."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch_cuda():
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch


@pytest.mark.parametrize("aligned", [True, False])
def test_steps_below_the_normal_range(torch_cuda, aligned):
    """bf16 groups whose step is subnormal: codes are rint((x - m) / s) + 8 of the definition in 64 bits (no tie is near:
    x - m and s are small multiples of 2^-133)."""
    torch = torch_cuda
    import cudasep

    g = torch.Generator().manual_seed(3)
    N, D = 64, 64
    top = 2.0 ** torch.linspace(-129, -118, N, dtype=torch.float64)
    x = ((torch.rand((1, N, 1, D), generator=g, dtype=torch.float64) - 0.3) * top.view(1, N, 1, 1)).bfloat16()
    gr = x.double().unflatten(-1, (2, 32))
    lo, hi = gr.amin(-1, keepdim=True), gr.amax(-1, keepdim=True)
    step = ((hi - lo) / 15).float().bfloat16().double()  # exact quotient, rounded: 2^-149 is exact enough for bf16 here
    mid = (lo + 8 * step).bfloat16().double()
    q = torch.where(step > 0, (gr - mid) / torch.where(step > 0, step, torch.ones_like(step)), torch.zeros_like(gr))
    want = (torch.round(q) + 8).clamp(0, 15).flatten(-2)[0, :, 0]
    sure = (((q - torch.floor(q)) - 0.5).abs() > 1e-4).flatten(-2)[0, :, 0]
    assert (step < 2.0 ** -128).any() and (step > 2.0 ** -126).any() and sure.float().mean() > 0.7
    cache = cudasep.KVCache.empty(1, 1, N, D, torch.bfloat16, bits=4)
    src = x.cuda()
    if not aligned:
        buf = torch.zeros((1, N, 1, D + 1), dtype=torch.bfloat16, device="cuda")
        buf[..., 1:] = src
        src = buf[..., 1:]
    cudasep.op_cache_append(cache, src, src, torch.zeros(1, dtype=torch.int32, device="cuda"))
    assert torch.equal(cache.k_scale[0, 0, :, :, 0].cpu().double(), step[0, :, 0, :, 0])
    assert torch.equal(cache.k_scale[0, 0, :, :, 1].cpu().double(), mid[0, :, 0, :, 0])
    got = torch.stack([cache.k & 15, cache.k >> 4], -1).flatten(-2)[0, 0].cpu().double()
    assert torch.equal(got[sure], want[sure])
