"""Calls whose threads are more than one grid holds (2^32 along an axis) take several launches."""
import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _values(n):
    """n different small values, cheap to make."""
    return ((np.arange(n, dtype=np.uint32) * np.uint32(2654435761)) >> np.uint32(8)).astype(np.float32)


def test_append_of_more_rows_than_a_grid_holds(gpu, rocm):
    n, tokens = 5, 1 << 24  # a wavefront per row of one value: 5.4e9 threads
    cache = gpu.PagedKvCache(n, tokens + 2, n * (tokens // 1024 + 1), 1024, 1, 1, quantized=False)
    seqs = [cache.add() for _ in range(n)]
    k = _values(n * tokens).reshape(n, 1, tokens, 1)
    t = gpu.Tensor.fromFloat32(k, list(k.shape))
    counts = [tokens, tokens, tokens - 3, tokens, tokens - 1]
    cache.append(seqs, t, t, counts)
    for i, s in enumerate(seqs):
        assert cache.length(s) == counts[i]
        for got in cache.read(s):
            assert np.array_equal(got.numpy(), k[i, :, :counts[i]]), i
            got.free()
    cache.free()
    gpu.native.resetEngine()
    rocm.clear_cache()


def test_eviction_and_reading_of_more_rows_than_a_grid_holds(gpu, rocm):
    budget = (1 << 26) + 9  # a wavefront per row that moves or is read
    length = 2 * budget
    cache = gpu.PagedKvCache(1, length, -(-length // 1024), 1024, 1, 1, quantized=False, tracked=True)
    s = cache.add()
    k = _values(length)
    for first in range(0, length, 1 << 24):
        t = gpu.Tensor.fromFloat32(k[first:first + (1 << 24)], [1, 1, min(1 << 24, length - first), 1])
        cache.append([s], t, t)
        t.free()

    def rows(want):
        for got in cache.read(s):
            assert np.array_equal(got.numpy().reshape(-1), want)
            got.free()

    rows(k)
    w = np.zeros((1, 1, length), np.float32)
    w[0, 0, budget:] = 1.0  # every row behind the budget takes a place below it, in order
    t = gpu.Tensor.fromFloat32(w, list(w.shape))
    cache.addWeights([s], t)
    t.free()
    cache.evict([s], budget)
    assert cache.length(s) == budget
    rows(k[budget:])
    weights, positions = cache.track([s])
    assert (weights.numpy() == 1).all()
    assert np.array_equal(gpu.native.intBufferToHost(positions), np.arange(budget, length, dtype=np.int32))
    cache.free()
    gpu.native.resetEngine()
    rocm.clear_cache()


def test_rotation_of_more_rows_than_a_grid_holds_in_single_values(rocm):
    s = (1 << 26) + 5  # a wavefront per row of one value: the norm alone
    x = _values(s) - np.float32(1 << 23)
    p, g, y = rocm.to_device(x), rocm.to_device(np.full(1, 3.0, np.float32)), rocm.malloc(x.nbytes)
    rocm.fill(y, 7.0, s)
    rocm.qk_norm_rope(dict(x=p, heads=1, gamma=g, out=y), batch=1, seq=s, head_dim=1, rotary_dims=0, eps=0.5)
    got = rocm.to_host(y, (s,))
    xd = x.astype(np.float64)
    # the square, the sum with eps, the root (2 steps) and two products: 6 half steps of an output of at most 3
    assert np.abs(got - 3.0 * xd / np.sqrt(xd * xd + 0.5)).max() <= 6 * 3.0 * 2.0 ** -24 * 2
    for ptr in (p, g, y):
        rocm.free(ptr)
    rocm.clear_cache()


def test_rotation_of_more_rows_than_a_grid_holds_in_pieces(rocm):
    s, d = (1 << 30) + 70, 8  # four lanes per row; every token reads the same row, 34 GB of outputs
    x = np.arange(1, 9, dtype=np.float32)
    p, g, y = rocm.to_device(x), rocm.to_device(np.ones(d, np.float32)), rocm.malloc(s * d * 4)
    rocm.qk_norm_rope(dict(x=p, heads=1, strides=(0, 0, 0), gamma=g, out=y), batch=1, seq=s, head_dim=d)
    z = x.astype(np.float64) / np.sqrt((x.astype(np.float64) ** 2).mean() + 1e-6)
    for first in (0, (1 << 29) - 3, (1 << 30) - 260, s - 90):
        at = np.arange(first, first + 90, dtype=np.float64)[:, None] * 10000.0 ** (-2.0 * np.arange(4) / d)
        want = np.concatenate([z[:4] * np.cos(at) - z[4:] * np.sin(at), z[4:] * np.cos(at) + z[:4] * np.sin(at)], 1)
        got = np.empty((90, d), np.float32)
        rocm._check(rocm.lib.mni_rocm_d2h(got.ctypes.data_as(ctypes.c_void_p), y + first * d * 4, got.nbytes))
        # the sum of squares and its root (d / 2 + 2 half steps), gain, sine and cosine (2 steps and their angle's pi each), products
        # and their sum, of |z_lo| + |z_hi|; the 64-bit angle itself is good to 2^-52 of up to 2^30 turns
        assert np.abs(got - want).max() <= 2.0 * (d / 2 + 10) * 2.0 ** -24 * 2 * np.abs(z).max()
    for ptr in (p, g, y):
        rocm.free(ptr)
    rocm.clear_cache()
