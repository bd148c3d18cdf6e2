"""CPU checks that calls whose launches would pass 2^32 threads are refused, with the reason, before the first launch
(the addresses are never read)."""
import ctypes

import pytest

from geoweave_amd import _lib

S2, S3 = _lib.strides2(64, 64), _lib.strides3(64, 64, 64)


def _last(lib):
    return lib.gw_last_error().decode()


def forward(lib, n=1, tq=8, tk=8, hq=4, hk=4, d=64):
    return lib.gw_packed_attn_fwd(0, 256, S2, 256, S2, 256, S2, 256, 256, 256, S2, None, None, n, tq, tk, hq, hk, d, 0, 0.125,
                                  256, 1 << 60, None)


def backward(lib, n=1, tq=8, tk=8, hq=4, hk=4, d=64):
    return lib.gw_packed_attn_bwd(0, 256, S2, 256, S2, 256, S2, 256, 256, 256, S2, 256, 256, S2, 256, 256, S2, 256, S2, 256,
                                  S2, n, tq, tk, hq, hk, d, 0, 0.125, 256, 1 << 60, None)


def paged(lib, b=1, n=1, hq=4, hk=2, d=64):
    return lib.gw_paged_attn_fwd(0, 256, S3, 256, S3, 256, S3, 256, 4, 256, 256, S3, None, b, n, hq, hk, d, 4, 16, 4, 1, 0.125,
                                 256, 1 << 60, None)


def rotary(lib, t=1):
    return lib.gw_rotary_axes(0, 256, S3, 256, S3, 1, None, None, None, None, 0, 0, 256, S3, 1, t, 64, 1, (ctypes.c_int32 * 1)(64),
                              (ctypes.c_double * 1)(100.0), 0, None)


@pytest.mark.parametrize("call,sizes", [
    (forward, dict(n=1 << 24)),
    (forward, dict(n=1 << 22)),  # times 4 key heads
    (forward, dict(n=1 << 22, tq=1 << 22, hk=4, d=128)),
    (backward, dict(n=1 << 24, hk=1)),
    (backward, dict(n=1 << 22)),
    (backward, dict(n=1 << 23, hq=1, hk=1, d=128)),  # dK/dV by 512 threads
    (backward, dict(n=1 << 24, tk=0, hq=1, hk=1)),
    (backward, dict(n=1 << 24, tq=0, hq=1, hk=1)),
    (backward, dict(tq=1 << 28, hq=1, hk=1)),  # 16 rows to a workgroup of the statistics
    (paged, dict(b=1 << 23)),
    (paged, dict(b=1 << 20, n=128)),
    (rotary, dict(t=1 << 27)),
])
def test_refused_before_a_launch(call, sizes):
    lib = _lib.load()
    assert call(lib, **sizes) == 2, _last(lib)
    assert "2^32 threads" in _last(lib)
