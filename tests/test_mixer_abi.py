"""CPU tests of the mixer's C entry points: what they refuse before any launch.
Pointers here are numbers that nothing dereferences."""

from __future__ import annotations

import ctypes

import pytest

from spikegpt_b200 import _capi

BASE = 1 << 20


def at(offset=0):
    return ctypes.c_void_p(BASE + offset)


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("offset", [1, 2, 4, 8, 15])
def test_q4_matvec_refuses_unaligned_weights(dtype, offset):
    p = at()
    assert _capi.lib().q4_matvec(dtype, p, at(offset), p, None, None, p, 1, 8, 64, 64, 64, None) == (
        _capi.WKV_ERR_INVALID_ARGUMENT)
    assert "packed must be 16-byte aligned" in _capi.last_error()
