"""Sizes of a cache at the ends of what is accepted (host checks of the C entry points, no GPU needed)."""
import ctypes
import struct

import pytest


def _bytes(sinks, ring, bits=0):
    """(status, workspace bytes) of one token's attention over a cache of one sequence and head of 32 channels."""
    import cudasep

    n = ctypes.c_int64(-1)
    c = struct.pack("@PPPPqiiiiii", 4096, 4096, 4096 if bits else 0, 4096 if bits else 0, 1, 1, 32, sinks, ring, 1, bits)
    return cudasep.lib().mbr_op_cache_attention_workspace(c, 1, 1, -1, 0, ctypes.byref(n)), n.value


@pytest.mark.parametrize("bits", [0, 4])
def test_slots_are_counted_in_32_bits(bits):
    for sinks, ring in ((0, 1), (0, 1 << 30), ((1 << 30) - 1, 1), (1 << 29, 1 << 29)):
        status, n = _bytes(sinks, ring, bits)
        assert status == 0 and n >= 0
    # keys rounded up to whole copies would pass 2^31
    for sinks, ring in (((1 << 30) - 1, (1 << 30) - 1), (1 << 30, 1), (1, 1 << 30), (2 ** 31 - 1, 2 ** 31 - 1), (0, 0), (0, -5)):
        assert _bytes(sinks, ring, bits)[0] == 1
