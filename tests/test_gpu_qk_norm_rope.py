"""Norm and rotation of queries and keys (mni_qk_norm_rope, mni_rocm_qk_norm_rope and its backward) against 64-bit
references: every head size class, partial and interleaved rotations, far and unequal positions, views, and gradients
against the formula and against differences."""
import math

import numpy as np
import pytest
import torch

from framework_amd import native as N
from framework_amd import synth

pytestmark = pytest.mark.gpu

U = 2.0 ** -24  # half a step of fp32, relative


def _rotate64(x, g, positions, rotary, interleaved, theta, eps):
    """x [B, H, S, D] and positions [B, S] in torch float64."""
    half = rotary // 2
    j = torch.arange(half)
    lo, hi = (2 * j, 2 * j + 1) if interleaved else (j, j + half)
    z = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * g
    a = positions.double()[:, None, :, None] * theta ** (-2.0 * j.double() / max(rotary, 1))
    out = z.clone()
    out[..., lo] = z[..., lo] * torch.cos(a) - z[..., hi] * torch.sin(a)
    out[..., hi] = z[..., hi] * torch.cos(a) + z[..., lo] * torch.sin(a)
    return out


def _tensor(api, a, grad=False):
    return api.Tensor.fromFloat32(a, list(a.shape)).setRequiresGrad(grad)


def _close_rows(got, want, d, scale):
    # sum of squares: D roundings, half of them felt through the root; product with the gain 2, sine and cosine 2 steps
    # each and their angle pi, the two products and their sum 3: per output (D / 2 + 10) half steps of |z_lo| + |z_hi|
    tol = 2.0 * (d / 2 + 10) * U * scale
    err = np.abs(got.astype(np.float64) - want)
    assert (err <= tol).all(), (float(err.max()), float(tol if np.isscalar(tol) else np.max(tol)))


CASES = [  # B, S, Hq, Hk, D, rotary, interleaved, offset, positions ("none", "shared", "each")
    (1, 1, 1, 1, 64, 64, False, 0, "none"),
    (8, 1, 12, 12, 64, 64, False, 100003, "each"),
    (2, 33, 4, 2, 128, 128, False, 0, "none"),
    (2, 31, 6, 2, 128, 64, True, 7, "shared"),
    (3, 5, 2, 1, 32, 32, True, 2 ** 20, "each"),
    (1, 17, 3, 3, 96, 96, False, 0, "none"),
    (1, 9, 5, 1, 80, 40, False, 0, "none"),
    (2, 4, 2, 2, 256, 256, False, 3, "none"),
    (2, 5, 2, 1, 256, 128, True, 0, "shared"),
    (1, 6, 2, 3, 20, 12, False, 1, "none"),     # not in eights: the form for any size
    (2, 3, 1, 1, 7, 2, True, 0, "each"),
    (1, 4, 2, 2, 1, 0, False, 0, "none"),
    (1, 5, 2, 2, 64, 0, False, 0, "none"),      # no rotation: the norm alone
    (1, 3, 2, 1, 200, 100, True, 2 ** 31 - 4, "none"),
    (4, 700, 8, 4, 64, 64, False, 0, "none"),   # enough rows for several heads per group of lanes
    (4, 701, 7, 4, 64, 32, True, 0, "shared"),
]


@pytest.mark.parametrize("b,s,hq,hk,d,rotary,interleaved,offset,given", CASES)
def test_forward_and_gradients(gpu, b, s, hq, hk, d, rotary, interleaved, offset, given):
    theta, eps = 10000.0, 1e-6
    x = [synth.normal(1 + i, (b, s, h, d), stream=i) for i, h in enumerate((hq, hk))]
    g = [1.0 + 0.25 * synth.normal(5 + i, (d,), stream=i) for i in range(2)]
    up = [synth.normal(9 + i, (b, h, s, d), stream=i) for i, h in enumerate((hq, hk))]
    pos = {"none": np.tile(np.arange(s), (b, 1)), "shared": np.tile(synth.integers(3, (s,), 0, 5000), (b, 1)),
           "each": synth.integers(4, (b, s), 0, 5000)}[given]
    buf = None
    if given != "none":
        buf = gpu.native.createDataset((pos[0] if given == "shared" else pos).reshape(-1).astype(np.int32))
    x_t = [_tensor(gpu, a, True) for a in x]
    g_t = [_tensor(gpu, a.astype(np.float32), True) for a in g]
    out = gpu.qkNormRope(x_t[0].permute(0, 2, 1, 3), x_t[1].permute(0, 2, 1, 3), g_t[0], g_t[1], positions=buf, offset=offset, rotaryDims=rotary,
                         interleaved=interleaved, theta=theta, eps=eps)
    loss = None
    for y, u in zip(out, up):
        term = y.mul(_tensor(gpu, u)).sum()
        loss = term if loss is None else loss.add(term)
    loss.backward()
    at = torch.from_numpy(pos.astype(np.float64)) + offset
    for i, h in enumerate((hq, hk)):
        xr = torch.from_numpy(x[i]).double().permute(0, 2, 1, 3).clone().requires_grad_(True)
        gr = torch.from_numpy(g[i].astype(np.float32)).double().requires_grad_(True)
        want = _rotate64(xr, gr, at, rotary, interleaved, theta, eps)
        (want * torch.from_numpy(up[i]).double()).sum().backward()
        z = np.abs((xr / torch.sqrt((xr * xr).mean(-1, keepdim=True) + eps) * gr).detach().numpy())
        assert out[i].shape == [b, h, s, d]
        _close_rows(out[i].numpy(), want.detach().numpy(), d, z.max(-1, keepdims=True))
        # dx = r dz g - x r^3 mean(dz g x): the rotated gradient (|dz| up to sqrt 2 |dy|) with the errors of the forward,
        # a sum of D products, and the difference of the two terms
        r = 1.0 / np.sqrt((x[i].astype(np.float64) ** 2).mean(-1) + eps)
        r = r.transpose(0, 2, 1)[..., None]
        xa, ga, ua = np.abs(x[i]).transpose(0, 2, 1, 3).astype(np.float64), np.abs(g[i]).max(), np.abs(up[i]).max(-1, keepdims=True)
        scale = math.sqrt(2) * ua * ga * (r + xa * r ** 3 * xa.mean(-1, keepdims=True))
        err = np.abs(x_t[i].grad.numpy().transpose(0, 2, 1, 3) - xr.grad.numpy())
        assert (err <= 2.0 * (2 * d + 16) * U * scale).all(), float((err / scale).max() / U)
        rows = b * h * s
        scale = (math.sqrt(2) * ua * xa * r).sum((0, 1, 2))
        err = np.abs(g_t[i].grad.numpy() - gr.grad.numpy())
        assert (err <= (rows + d + 16) * U * scale).all(), float((err / scale).max() / U)


@pytest.mark.parametrize("d,rotary,interleaved", [(32, 32, False), (32, 16, True), (6, 4, False)])
def test_gradients_against_differences(gpu, d, rotary, interleaved):
    b, s, h = 1, 3, 2
    x, g, up = synth.normal(1, (b, h, s, d)), (1.0 + 0.25 * synth.normal(2, (d,))).astype(np.float32), synth.normal(3, (b, h, s, d), stream=1)
    x_t, g_t = _tensor(gpu, x, True), _tensor(gpu, g, True)
    k = _tensor(gpu, x)
    y, _ = gpu.qkNormRope(x_t, k, g_t, g_t, offset=11, rotaryDims=rotary, interleaved=interleaved)
    y.mul(_tensor(gpu, up)).sum().backward()
    at = torch.arange(s)[None].double() + 11

    def loss(xv, gv):
        return float((_rotate64(torch.from_numpy(xv), torch.from_numpy(gv), at, rotary, interleaved, 10000.0, 1e-6) * torch.from_numpy(up).double()).sum())

    step = 1e-5  # in 64 bits: the quotient's own error is about step^2 and 2^-52 |loss| / step, both below 1e-9
    for got, which in ((x_t.grad.numpy(), 0), (g_t.grad.numpy(), 1)):
        base = [x.astype(np.float64), g.astype(np.float64)]
        flat = base[which].reshape(-1)
        for e in range(0, flat.size, 5):
            keep = flat[e]
            flat[e] = keep + step
            hi = loss(*base)
            flat[e] = keep - step
            lo = loss(*base)
            flat[e] = keep
            assert abs(got.reshape(-1)[e] - (hi - lo) / (2 * step)) <= 1e-4 * (1 + np.abs(up).max() * 4), (which, e)


def test_rows_inside_a_fused_projection_and_kernel_level(rocm):
    # queries and keys read where they lie in one [B, S, Hq + 2 Hk, D] buffer, an operand left out, an empty call
    b, s, hq, hk, d = 2, 19, 6, 2, 64
    w = hq + 2 * hk
    qkv, g = synth.normal(1, (b, s, w, d)), np.ones(d, np.float32)
    p, gp = rocm.to_device(qkv), rocm.to_device(g)
    oq, ok = rocm.malloc(b * hq * s * d * 4), rocm.malloc(b * hk * s * d * 4)
    strides = (s * w * d, d, w * d)
    plan = dict(batch=b, seq=s, head_dim=d)
    rocm.qk_norm_rope(dict(x=p, heads=hq, strides=strides, gamma=gp, out=oq), dict(x=p + hq * d * 4, heads=hk, strides=strides, gamma=gp, out=ok), **plan)
    at = torch.arange(s)[None].double().expand(b, s)
    for first, h, o in ((0, hq, oq), (hq, hk, ok)):
        x = torch.from_numpy(qkv[:, :, first:first + h]).double().permute(0, 2, 1, 3)
        want = _rotate64(x, torch.ones(d).double(), at, d, False, 10000.0, 1e-6).numpy()
        _close_rows(rocm.to_host(o, (b, h, s, d)), want, d, np.abs(want).max() * 1.5)
    both = rocm.to_host(oq, (b, hq, s, d))
    rocm.fill(oq, 0.0, b * hq * s * d)
    rocm.qk_norm_rope(dict(x=p, heads=hq, strides=strides, gamma=gp, out=oq), **plan)
    assert np.array_equal(rocm.to_host(oq, (b, hq, s, d)), both)
    # the same rows off a 16-byte boundary take the other kernel: the same values within both bounds
    odd = rocm.malloc(qkv.nbytes + 16)
    rocm._check(rocm.lib.mni_rocm_h2d(odd + 4, qkv.ctypes.data, qkv.nbytes))
    rocm.qk_norm_rope(dict(x=odd + 4, heads=hq, strides=strides, gamma=gp, out=oq), **plan)
    _close_rows(rocm.to_host(oq, (b, hq, s, d)), both.astype(np.float64), d, 2 * np.abs(both).max() * 1.5)
    rocm.qk_norm_rope(dict(x=p, heads=hq, strides=strides, gamma=gp, out=oq), batch=0, seq=s, head_dim=d)
    dg = rocm.to_device(np.full(d, 7.0, np.float32))
    rocm.qk_norm_rope_backward(dict(x=p, heads=hq, gamma=gp, grad=oq, dx=oq, dgamma=dg), batch=0, seq=s, head_dim=d)
    assert (rocm.to_host(dg, (d,)) == 0).all()
    for ptr in (p, gp, oq, ok, odd, dg):
        rocm.free(ptr)


def test_the_same_bits_every_time_and_rows_of_zeros(gpu):
    b, s, h, d = 3, 257, 4, 64
    x, up = synth.normal(1, (b, h, s, d)), synth.normal(2, (b, h, s, d), stream=1)
    x[0, 0, :5] = 0.0  # eps alone under the root
    seen = []
    for _ in range(3):
        x_t, g_t = _tensor(gpu, x, True), _tensor(gpu, np.ones(d, np.float32), True)
        y, z = gpu.qkNormRope(x_t, _tensor(gpu, x), g_t, g_t)
        y.mul(_tensor(gpu, up)).sum().backward()
        seen.append([y.numpy(), z.numpy(), x_t.grad.numpy(), g_t.grad.numpy()])
    for a in seen[1:]:
        assert all(np.array_equal(p, q) for p, q in zip(a, seen[0]))
    assert np.array_equal(seen[0][0], seen[0][1]) and (seen[0][0][0, 0, :5] == 0).all()
    assert all(np.isfinite(a).all() for a in seen[0])


def test_engine_refusals(gpu):
    T = lambda *shape: gpu.Tensor.zeros(list(shape))  # noqa: E731
    q, g = T(2, 3, 4, 8), T(8)
    for args, kw, text in [((T(2, 3, 4), q, g, g), {}, r"must be \[B, H, S, D\]"), ((q, T(2, 3, 5, 8), g, g), {}, "differ in batch, length or head_dim"),
                           ((q, q, T(4), g), {}, r"gains must be \[8\]"), ((q, q, g, g), {"rotaryDims": 3}, "must be even"),
                           ((q, q, g, g), {"rotaryDims": 10}, "must be even"), ((q, q, g, g), {"theta": 0.0}, "theta must be positive"),
                           ((q, q, g, g), {"eps": -1.0}, "eps must not be negative"), ((T(1, 1, 1, 300), T(1, 1, 1, 300), T(300), T(300)), {}, "head_dim 300"),
                           ((q, q, g, g), {"positions": gpu.native.createDataset(np.arange(3, dtype=np.int32))}, "expected 4 or 8"),
                           ((q, q, g, g), {"positions": 12345}, "int buffer already freed")]:
        with pytest.raises(N.MniError, match=text):
            gpu.qkNormRope(*args, **kw)
