"""GPU test of the end of a stream (mbr-cuda-tile_b200/streaming.py): frames past max_frames are refused before anything is
changed."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch_cuda():
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch


def test_frames_past_the_tables_are_refused(torch_cuda):
    torch = torch_cuda
    import streaming

    make = dict(bands=3, dim=64, heads=2, left=10, max_frames=32)
    x = torch.randn((40, 3, 64), generator=torch.Generator().manual_seed(7)).cuda().to(torch.bfloat16)
    with pytest.raises(ValueError, match="max_frames"):
        streaming.random_layer(**make).prompt(x)
    layer = streaming.random_layer(**make)
    y = [layer.prompt(x[:20]), layer.step(x[20:31])]
    with pytest.raises(ValueError, match="max_frames"):
        layer.step(x[31:33])
    assert layer.frames == 31
    y.append(layer.step(x[31:32]))  # the last one
    with pytest.raises(ValueError, match="max_frames"):
        layer.step(x[32:33])
    assert torch.isfinite(torch.cat(y).float()).all()
    # the same frames with room to spare, and the refused call not made
    other = streaming.random_layer(**{**make, "max_frames": 64})
    z = [other.prompt(x[:20]), other.step(x[20:31]), other.step(x[31:32])]
    assert torch.equal(torch.cat(y), torch.cat(z))


def test_the_default_ends_at_65536_frames(torch_cuda):
    torch = torch_cuda
    import streaming

    layer = streaming.random_layer(bands=2, dim=64, heads=1, left=5)
    x = torch.randn((2, 2, 64), device="cuda").to(torch.bfloat16)
    layer.prompt(x)
    layer.frames = 65535  # as if so many had passed
    assert torch.isfinite(layer.step(x[:1]).float()).all()
    with pytest.raises(ValueError, match="max_frames"):
        layer.step(x[:1])
