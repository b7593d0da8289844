"""A theta so small that angles of far positions leave the range that is reduced to a quarter turn is refused before a device is
touched."""
import ctypes

import pytest

from framework_amd import native as N


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("theta,taken", [(2.0 ** -16, True), (0.5, True), (1.0, True), (2.0 ** -16 * (1 - 2.0 ** -53), False), (1e-12, False), (5e-324, False)])
def test_small_theta(theta, taken, backward):
    lib = N.load_library()
    # (a negative extent is refused earlier, an odd one of rotary_dims too: eps is looked at next)
    d = N.Rocm.rope_desc(None, batch=0, seq=1, head_dim=8, theta=theta, eps=-1.0)
    f = lib.mni_rocm_qk_norm_rope_backward if backward else lib.mni_rocm_qk_norm_rope
    assert f(ctypes.byref(d)) == 1
    error = lib.mni_rocm_last_error().decode()
    assert ("eps must not be negative" if taken else "below 2^-16") in error
