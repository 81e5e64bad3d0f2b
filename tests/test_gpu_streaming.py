"""GPU test of the streaming layer (mbr-cuda-tile_b200/streaming.py): frames one by one, in small groups and all at
once give the same heads' outputs, within twice the attention's bound (tests/stream_ref.py) at the same q, k and v; with a
4-bit cache, the same against attention over the rounded keys and values."""
import pytest

import stream_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch_cuda():
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch


def _reference(torch, layer, x, bits):
    """(heads' outputs, bound) [n, bands, heads, dim_head] from the layer's own q, k, v, gates."""
    q, k, v, gates = (t.cpu() for t in layer._project(x))
    if bits:
        k, v = ref.four_bits(k.contiguous())[3], ref.four_bits(v.contiguous())[3]
    n = x.shape[0]
    see = ref.visible(range(n), n, layer.left, 0, layer.sinks)
    pairs = [ref.attention(q[b], k[b], v[b], see, layer.dim_head ** -0.5, gates[b]) for b in range(layer.bands)]
    return torch.stack([p[0] for p in pairs], 1), torch.stack([p[1] for p in pairs], 1)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("bits", [0, 4])
@pytest.mark.parametrize("left,sinks", [(20, 3), (200, 0)])
def test_streaming_equals_one_pass(torch_cuda, dtype, bits, left, sinks):
    torch = torch_cuda
    import streaming

    make = dict(bands=3, dim=64, heads=2, left=left, sinks=sinks, dtype=dtype, seed=3)
    n = 90
    x = torch.randn((n, 3, 64), generator=torch.Generator().manual_seed(5)).cuda()
    one = streaming.random_layer(**make)
    x = x.to(one.dtype)
    want, bound = _reference(torch, one, x, 0)
    got = one.attend_prompt(x).cpu().double().view(want.shape)
    assert ((got - want).abs() <= bound).all()

    live = streaming.random_layer(bits=bits, **make)
    outs, at = [live.attend_prompt(x[:40])], 40
    for m in (1, 1, 5, 1, 17, 1, 24):
        outs.append(live.attend_step(x[at:at + m]))
        at += m
    assert at == n and live.frames == n
    if bits:
        want, bound = _reference(torch, streaming.random_layer(**make), x, bits)
    got = torch.cat(outs[1:]).cpu().double().view(want[40:].shape)
    assert ((got - want[40:]).abs() <= bound[40:]).all()


def test_streaming_layer_and_refusals(torch_cuda):
    torch = torch_cuda
    import streaming

    layer = streaming.random_layer(bands=4, dim=64, heads=2, left=10)
    x = torch.randn((30, 4, 64), generator=torch.Generator().manual_seed(6)).cuda().to(layer.dtype)
    y = layer.prompt(x[:20])
    z = layer.step(x[20:])
    assert y.shape == (20, 4, 64) and z.shape == (10, 4, 64)
    assert torch.isfinite(y.float()).all() and torch.isfinite(z.float()).all()
    with pytest.raises(ValueError):
        layer.prompt(x)
    with pytest.raises(ValueError):
        layer.step(torch.zeros((65, 4, 64), dtype=x.dtype, device="cuda"))


def test_streaming_command(torch_cuda, capsys):
    import streaming

    streaming.main(["--bands", "5", "--dim", "64", "--heads", "2", "--seconds", "0.4", "--left", "20", "--bits", "4"])
    assert "ms a frame" in capsys.readouterr().out
