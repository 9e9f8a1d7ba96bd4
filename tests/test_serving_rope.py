"""CPU check of the paged front's rotary frequencies (host code of the library)
against decimal arithmetic."""
import ctypes
import struct
from decimal import Decimal, getcontext

import pytest

import jllm

HALF = 64                                    # entries of the table (head_dim <= 128)
PI = Decimal("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899862803")


def turns(head_dim, theta):
    """rope_turns(RopeTurns&, int, double) of csrc/paged_front.hip."""
    f = getattr(jllm.lib(), "_ZN8jllm_hip10rope_turnsERNS_9RopeTurnsEid")
    f.argtypes, f.restype = [ctypes.c_void_p, ctypes.c_int, ctypes.c_double], None
    out = (ctypes.c_uint64 * HALF)()
    f(out, head_dim, theta)
    return list(out)


THETAS = [1 + 2.0 ** -23, 1.001, 1.5, 2.0, 3.0, 10.0, 1234.5, 1e4, 5e5, 1e6, 2.0 ** 24, 1e8, 1e11, 2.0 ** 46, 2.0 ** 47, 2.0 ** 48,
          1e16, 2.0 ** 55, 1e18, 1e25, 3e38]


@pytest.mark.parametrize("head_dim", [8, 24, 40, 64, 96, 128])
@pytest.mark.parametrize("theta", THETAS)
def test_rotary_frequencies_are_exact(head_dim, theta):
    """theta^(-2 i / hd) / 2 pi rounded to 64 bits (half of 2^-64 turns and a hundredth;
    above 2^64, where the ratio of two entries has 63 bits, 2^-63 i r^i / 2 pi more), so
    that a position of 2^31 times it is within 2^-33 turns."""
    getcontext().prec = 80
    theta = struct.unpack("f", struct.pack("f", theta))[0]        # the entry point takes a float
    got = turns(head_dim, theta)
    ln = Decimal(theta).ln()
    for i in range(head_dim // 2):
        want = (-ln * 2 * i / head_dim).exp() / (2 * PI) * 2 ** 64
        assert abs(got[i] - want) < Decimal("0.51" if theta < 2.0 ** 64 else "0.7"), (i, float(got[i] - want))
    assert not any(got[head_dim // 2:])
