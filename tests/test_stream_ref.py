"""CPU checks of the references that the streaming-attention tests use, and of the C entry points' argument checks."""
import math
import struct

import numpy as np
import pytest
import torch

import stream_ref as ref


def test_reference_attention_equals_masked_softmax():
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(n, h, 16, generator=g, dtype=torch.float64).float() for n, h in ((5, 4), (9, 2), (9, 2)))
    see = ref.visible(range(4, 9), 9, 2, 1, 1)
    out, bound = ref.attention(q, k, v, see, 0.25, None)
    s = torch.einsum("ihd,jhd->hij", q.double(), k.double().repeat_interleave(2, 1)) * 0.25
    w = torch.softmax(s.masked_fill(~see, -math.inf), -1)
    want = torch.einsum("hij,jhd->ihd", w, v.double().repeat_interleave(2, 1))
    assert torch.allclose(out, want, atol=1e-12) and (bound > 0).all()


def test_reference_visibility():
    see = ref.visible([5], 9, 2, 1, 1)[0].tolist()
    assert see == [True, False, False, True, True, True, True, False, False]
    assert ref.visible([-1], 3, -1, 0, 0).sum() == 0
    assert ref.visible([-1], 3, -1, 1, 0).tolist() == [[True, False, False]]
    assert ref.visible([7], 8, -1, 0, 2, held_from=6)[0].tolist() == [True, True] + [False] * 4 + [True, True]


def test_reference_rotation_is_a_rotation():
    x = torch.randn(2, 3, 2, 8, generator=torch.Generator().manual_seed(1))
    ang = torch.rand(10, 4)
    pos = torch.randint(0, 10, (2, 3, 2), dtype=torch.int32)
    z, bound = ref.rotate(x, None, ang.cos(), ang.sin(), pos, [1, 2], 0.0)
    n = x.double() / x.double().pow(2).mean(-1, keepdim=True).sqrt()
    assert torch.allclose(z.pow(2).sum(-1), n.pow(2).sum(-1), rtol=1e-6)
    assert torch.allclose(z[..., 6:], n[..., 6:]) and (bound > 0).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_four_bits_stay_within_half_a_step(dtype):
    x = torch.randn(50, 64, generator=torch.Generator().manual_seed(2)).to(dtype)
    code, step, mid, values = ref.four_bits(x)
    assert code.min() == 0 and code.max() == 15
    err = (values.double() - x.double()).abs().unflatten(-1, (2, 32))
    # half a step, the ends moved by the roundings of step (8 steps of it) and offset, the value's own rounding
    u = ref.HALF_ULP[dtype]
    bound = step.double() * (0.5 + 8 * 2 * u) + u * (mid.double().abs() + 9 * step.double()) * 2
    assert (err.amax(-1) <= bound).all()


def test_entry_points_refuse_without_a_gpu():
    """Bad sizes are refused before anything is launched, with MBR_ERR_INVALID and a message."""
    import cudasep

    L = cudasep.lib()
    one = np.zeros(64, np.float32).ctypes.data
    view = struct.pack("@Pqqq", one, 64, 64, 64)

    def norm(D=64, axes=0, pairs=None, eps=1e-6, dtype=1, seqs=1):
        return L.mbr_op_qk_norm_rope(view, view, view, view, seqs, 1, 1, 1, D, None, None, eps, None, None, 0, None, axes,
                                     pairs, dtype, None)

    def window(Hq=1, Hkv=1, D=64, N=1, M=1, sinks=0, dtype=1, scale=0.0, q=view):
        return L.mbr_op_window_attention(q, view, view, view, 1, N, M, Hq, Hkv, D, None, None, -1, -1, sinks, scale, None,
                                         dtype, None, 0, None)

    def cache(dtype=1, bits=0, D=64, ring=4, sinks=0, k=4096):
        return struct.pack("@PPPPqiiiiii", k, k, k if bits else 0, k if bits else 0, 1, 1, D, sinks, ring, dtype, bits)

    def append(c, tokens=1, pos=one):
        return L.mbr_op_cache_append(c, view, view, pos, None, tokens, None)

    refused = [norm(D=63), norm(D=0), norm(D=258), norm(axes=5), norm(axes=1), norm(eps=-1.0), norm(dtype=2),
               norm(seqs=-1), window(Hq=3, Hkv=2), window(Hq=1, Hkv=0), window(D=12), window(D=136), window(N=-1),
               window(N=1 << 30), window(M=1 << 30), window(sinks=-1), window(dtype=7), window(scale=math.nan),
               window(q=None), append(None), append(cache(dtype=2)), append(cache(bits=3)), append(cache(dtype=0, bits=4)),
               append(cache(bits=4, D=40)), append(cache(ring=0)), append(cache(sinks=-1)), append(cache(D=4)),
               append(cache(k=4104)), append(cache(), tokens=-1), append(cache(), pos=None),
               L.mbr_op_cache_attention(view, cache(), view, None, 1, 1, -1, 0, 0.0, None, None, 0, None),
               L.mbr_op_cache_attention(view, cache(ring=100000), view, one, 1, 1, -1, 0, 0.0, None, None, 0, None),
               L.mbr_op_cache_attention(view, None, view, one, 1, 1, -1, 0, 0.0, None, None, 0, None)]
    assert refused == [1] * len(refused)
    assert L.mbr_last_error()
    # nothing to do is no error, and needs no buffers
    assert window(N=0) == 0 and norm(seqs=0) == 0 and append(cache(), tokens=0) == 0


def test_the_extension_refuses_cpu_tensors():
    """The Python calls check their tensors before anything else happens."""
    import cudasep

    x = torch.zeros(1, 2, 3, 64)
    for call in (lambda: cudasep.op_qk_norm_rope(x, x), lambda: cudasep.op_window_attention(x, x, x),
                 lambda: cudasep.KVCache(x, x), lambda: cudasep.KVCache(None, None)):
        with pytest.raises((ValueError, AttributeError)):
            call()
    with pytest.raises(ValueError):
        cudasep.KVCache.empty(1, 1, 8, 64, torch.float16, bits=3, device="cpu")
