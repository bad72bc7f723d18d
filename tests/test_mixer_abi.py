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


@pytest.mark.parametrize("offset", [1, 2, 4, 8])
def test_scan_refuses_an_unaligned_workspace(offset):
    """Its partial states move as 16-byte words."""
    lib, p, null = _capi.lib(), at(), None
    b, t, c, n = 1, 4096, 64, 16  # few channels and many steps: split over time
    strides = [t * c, c, t * c, c, t * n, n, t * n, n, 0, 0]
    size = lib.selective_scan_forward_workspace_size(0, b, t, c, n)
    assert size > 0
    assert lib.selective_scan_forward(0, p, p, p, p, p, null, null, null, null, null, p, null, null, 0, at(offset), size,
                                      b, t, c, n, *strides, 1, null) == _capi.WKV_ERR_INVALID_ARGUMENT
    assert "workspace must be 16-byte aligned" in _capi.last_error()
    for t in (8, 4096):
        strides = [t * c, c, t * c, c, t * c, c, t * n, n, t * n, n, 0, 0]
        size = lib.selective_scan_backward_workspace_size(0, b, t, c, n)
        assert lib.selective_scan_backward(0, p, p, p, p, p, p, null, null, null, p, null, null, p, p, p, p, p, null,
                                           null, null, null, at(offset), size, b, t, c, n, *strides, 1, null) == (
            _capi.WKV_ERR_INVALID_ARGUMENT)
        assert "workspace must be 16-byte aligned" in _capi.last_error()


def test_scan_backward_without_channels_has_sums_to_write():
    """grad_B and grad_C [B, T, N] exist where there is no channel to add up."""
    lib, p, null = _capi.lib(), at(), None
    strides = [0] * 12
    for b, t, want in ((2, 3, _capi.WKV_ERR_INVALID_ARGUMENT), (0, 3, 0), (2, 0, 0)):
        assert lib.selective_scan_backward(0, null, null, null, null, p, p, null, null, null, null, null, null, null,
                                           null, null, null, null, null, null, null, null, null, 0, b, t, 0, 4,
                                           *strides, 1, null) == want


def test_layer_norm_backward_fills_the_gpu_at_every_width():
    """The workspace holds one partial row of both sums for each CTA: at least one an SM where
    there are rows enough, whatever the CTAs' threads."""
    size, sms = _capi.lib().layer_norm_workspace_size, 148  # what the plan assumes without a GPU
    for c, want in ((64, 2 * sms), (4096, 2 * sms), (8192, sms), (8193, sms), (16384, sms)):
        assert -(-size(0, 100000, c) // (2 * c * 4)) >= want, c
    assert size(0, 3, 16384) == 3 * 2 * 16384 * 4
