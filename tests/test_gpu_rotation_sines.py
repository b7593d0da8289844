"""The sines and cosines of the rotation alone: rows whose pairs are (1, 0) and whose norm is 1, so that outputs are (cos, sin)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.mark.parametrize("d,interleaved", [(64, False), (128, True), (20, False), (6, True), (256, False)])
@pytest.mark.parametrize("first,backwards", [(0, False), (90000, False), (0, True)])
def test_against_64_bit_sines(rocm, d, interleaved, first, backwards):
    s = 8192
    x = np.zeros(d, np.float32)
    lo, hi = (np.arange(0, d, 2), np.arange(1, d, 2)) if interleaved else (np.arange(d // 2), np.arange(d // 2, d))
    x[lo] = 1.0
    p, g, y = rocm.to_device(x), rocm.to_device(np.ones(d, np.float32)), rocm.malloc(s * d * 4)
    at = first + np.arange(s)
    pos = rocm.to_device((-at if backwards else at).astype(np.int32))
    # mean(x^2) + eps = 1 / 2 + 1 / 2: the norm's factor is 1
    rocm.qk_norm_rope(dict(x=p, heads=1, strides=(0, 0, 0), gamma=g, out=y), batch=1, seq=s, head_dim=d, positions=pos, eps=0.5, interleaved=interleaved)
    got = rocm.to_host(y, (s, d)).astype(np.float64)
    angle = at.astype(np.longdouble)[:, None] * np.longdouble(10000.0) ** (np.arange(d // 2) * np.longdouble(-2.0) / d) * (-1 if backwards else 1)
    # The rest r of a quarter turn, |r| <= 1/2, rounded to 32 bits: pi / 2 * 2^-26 = 0.39 U of the angle.  Sine (at most 0.71): the last
    # rounding 0.5 U, the tail of at most 0.08 with three half steps 0.24 U, the next term of the series 0.03 U: 1.2 U.  Cosine (from 0.71
    # on): 0.39 * 0.71 U, the last rounding 0.5 U, what is taken off (at most 0.29, two half steps) 0.6 U: 1.4 U.  The 64-bit angle: 1.5 * 2^-53
    # of at most 98192, below 0.001 U.  Relative to a small sine: one half step of r, one of the result, half a one of the tail
    # and 1.5 * 2^-53 * 98192 = 0.0000003 U over the sine itself.
    for cols, want in ((lo, np.cos(angle)), (hi, np.sin(angle))):
        err = np.abs(got[:, cols] - want).astype(np.float64)
        assert err.max() <= 1.5 * U, err.max() / U
        assert (err <= 3.0 * U * np.abs(want).astype(np.float64) + 1.5 * 2.0 ** -53 * 98192).all(), (err / np.abs(want).astype(np.float64)).max() / U
    for ptr in (p, g, y, pos):
        rocm.free(ptr)
