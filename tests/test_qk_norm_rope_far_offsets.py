"""Offsets at which a 64-bit angle has no fraction left are refused before a device is touched."""
import ctypes

import pytest

from framework_amd import native as N


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("offset", [(1 << 32) + 1, -(1 << 32) - 1, 1 << 60, (1 << 63) - 1, -(1 << 63)])
def test_far_offsets_are_refused(offset, backward):
    lib = N.load_library()
    d = N.Rocm.rope_desc(None, batch=0, seq=1, head_dim=8, offset=offset)
    f = lib.mni_rocm_qk_norm_rope_backward if backward else lib.mni_rocm_qk_norm_rope
    assert f(ctypes.byref(d)) == 1
    assert "offset %d beyond 2^32" % offset in lib.mni_rocm_last_error().decode()


@pytest.mark.parametrize("offset", [1 << 32, -(1 << 32)])
def test_the_farthest_offsets_are_taken(offset):
    lib = N.load_library()
    d = N.Rocm.rope_desc(None, batch=0, seq=1, head_dim=8, offset=offset)
    assert lib.mni_rocm_qk_norm_rope(ctypes.byref(d)) == 0  # no rows: nothing to do
