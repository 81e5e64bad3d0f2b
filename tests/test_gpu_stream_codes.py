"""4-bit caches at the edges of their definition: steps below fp32's normal range, and values whose exact sum lies next to a
tie of the cache's type (one rounding, in every place that widens codes)."""
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


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("aligned", [True, False])
def test_values_are_rounded_once(torch_cuda, dtype, aligned):
    """m + s (c - 8) next to a tie of the type, nearer than fp32 can tell: read back and seen by the attention (one key a
    sequence, so that its value is the output) as the exact sum rounded once."""
    torch = torch_cuda
    import cudasep

    dt, bits, tiny = {"fp16": (torch.float16, 10, 2.0 ** -24), "bf16": (torch.bfloat16, 7, 2.0 ** -40)}[dtype]
    S, D = 4, 64
    s = torch.tensor([1 + 2.0 ** -bits, 1 + 3 * 2.0 ** -bits, 1 - 2.0 ** (-bits - 1), 1.0], dtype=torch.float64)
    m = torch.tensor([-tiny, tiny, -tiny, tiny], dtype=torch.float64)
    codes = torch.arange(D) % 16
    exact = (s[:, None] * (codes - 8) + m[:, None])  # 64 bits hold every sum
    fp32 = (s[:, None].float() * (codes - 8).float() + m[:, None].float()).to(dt).double()
    # one rounding from 64 bits: the two neighbours, the nearer one
    near = exact.float().to(dt).double()
    ulp = 2.0 ** (torch.floor(torch.log2(exact.abs().clamp_min(2.0 ** -14))) - bits)
    cands = torch.stack([near - ulp, near, near + ulp])
    want = torch.gather(cands, 0, (cands - exact).abs().argmin(0, keepdim=True))[0]
    assert (want != fp32).any()  # rounding twice shows
    cache = cudasep.KVCache.empty(S, 1, 1, D, dt, bits=4)
    cache.k.copy_((codes[0::2] | codes[1::2] << 4).to(torch.uint8).expand(S, 1, 1, D // 2))
    cache.v.copy_(cache.k)
    for t in (cache.k_scale, cache.v_scale):
        t[..., 0], t[..., 1] = s.to(dt).cuda().view(S, 1, 1, 1), m.to(dt).cuda().view(S, 1, 1, 1)
    assert torch.equal(cache.k_scale[:, 0, 0, 0].double().cpu(), torch.stack([s, m], -1))
    zero = torch.zeros(S, dtype=torch.int32, device="cuda")
    buf = torch.zeros((S, 1, 1, D + 8 * aligned + 1 * (not aligned)), dtype=dt, device="cuda")
    out = buf[..., 8:] if aligned else buf[..., 1:]
    k, v = cudasep.op_cache_read(cache, zero, 1, k=out, v=torch.empty_like(out))
    assert torch.equal(k[:, 0, 0].cpu().double(), want) and torch.equal(v[:, 0, 0].cpu().double(), want)
    q = torch.zeros((S, 1, 1, D), dtype=dt, device="cuda")
    got = cudasep.op_cache_attention(q, cache, zero + 1)
    assert torch.equal(got[:, 0, 0].cpu().double(), want)
    # the form that takes rows that are not finite again, by a NaN in a key: the values of the other keys stay
    q = torch.ones((S, 1, 1, D), dtype=dt, device="cuda")
    big = cudasep.KVCache.empty(S, 1, 3, D, dt, bits=4)
    for a, b in ((big.k, cache.k), (big.v, cache.v), (big.k_scale, cache.k_scale), (big.v_scale, cache.v_scale)):
        a[:, :, :1] = b
    big.v_scale[:, :, 1:] = float("nan")
    two = torch.cat([q, q], 1)
    got = cudasep.op_cache_attention(two, big, zero + 2)  # row 0 sees key 0 only, row 1 the NaN too
    assert torch.equal(got[:, 0, 0].cpu().double(), want) and got[:, 1].isnan().all()
