"""Gradients of norm and rotation where an operand has no rows: the gain's is a sum over nothing, zeros."""
import numpy as np
import pytest

from framework_amd import synth

pytestmark = pytest.mark.gpu


def _t(gpu, a):
    a = np.ascontiguousarray(a, dtype=np.float32)
    return gpu.Tensor.fromFloat32(a, list(a.shape))


@pytest.mark.parametrize("d", [6, 64])
@pytest.mark.parametrize("hq,hk", [(3, 0), (0, 2), (0, 0)])
def test_an_operand_without_heads(gpu, hq, hk, d):
    b, s = 2, 5
    x = [gpu.Tensor.zeros([b, h, s, d]) if h == 0 else _t(gpu, synth.normal(1, (b, h, s, d))) for h in (hq, hk)]
    g = [_t(gpu, np.ones(d)) for _ in range(2)]
    for t in x + g:
        t.setRequiresGrad(True)
    out = gpu.qkNormRope(*x, *g)
    loss = out[0].sum().add(out[1].sum())
    for t in [_t(gpu, np.full(d, 7.0)) for _ in range(64)]:  # what the gradients' memory held before
        t.free()
    loss.backward()
    for h, t in zip((hq, hk), g):
        got = t.grad.numpy()
        assert (got == 0).all() if h == 0 else (got != 0).any() and (got != 7).all()


@pytest.mark.parametrize("d", [6, 32])
def test_kernel_level(rocm, d):
    b, s, h = 1, 3, 2
    x, up = synth.normal(1, (b, h, s, d)), synth.normal(2, (b, h, s, d), stream=1)
    p, g, dy = rocm.to_device(x), rocm.to_device(np.ones(d, np.float32)), rocm.to_device(up)
    dx, dg, none = rocm.malloc(x.nbytes), rocm.to_device(np.full(d, 7.0, np.float32)), rocm.to_device(np.full(d, 7.0, np.float32))
    full, empty = dict(x=p, heads=h, gamma=g, grad=dy, dx=dx, dgamma=dg), dict(x=p, heads=0, gamma=g, grad=dy, dx=dx, dgamma=none)
    plan = dict(batch=b, seq=s, head_dim=d)
    rocm.qk_norm_rope_backward(full, **plan)
    want = rocm.to_host(dg, (d,))
    for pair in ((full, empty), (empty, full), (empty, empty)):
        for ptr in (dg, none):
            rocm.fill(ptr, 7.0, d)
        rocm.qk_norm_rope_backward(*pair, **plan)
        assert (rocm.to_host(none, (d,)) == 0).all()
        if full in pair:
            assert np.array_equal(rocm.to_host(dg, (d,)), want)
    # an operand without a gradient is left out
    rocm.fill(none, 7.0, d)
    rocm.qk_norm_rope_backward(full, dict(x=p, heads=0, gamma=g, dgamma=none), **plan)
    assert (rocm.to_host(none, (d,)) == 7).all() and np.array_equal(rocm.to_host(dg, (d,)), want)
    for ptr in (p, g, dy, dx, dg, none):
        rocm.free(ptr)
