"""Calls whose threads are more than one grid holds (2^32 along an axis) take several launches."""
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
