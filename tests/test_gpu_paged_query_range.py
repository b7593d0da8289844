"""Attention over int8 rows with queries of very unequal values: a value that is thousands of times the others, in a dim where the
keys are zero, must not cost the others their bits."""
import numpy as np
import pytest

from framework_amd import synth
from test_gpu_paged_cache import Model, _t

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("ratio", [1.0, 1e3, 4e3, 1e4])
@pytest.mark.parametrize("heads,group,d,page,length", [(2, 1, 64, 16, 700), (2, 3, 128, 16, 4096), (1, 8, 128, 64, 300), (2, 2, 96, 8, 900), (1, 16, 256, 16, 500),
                                                       (2, 2, 80, 4, 333), (1, 1, 7, 8, 100), (1, 4, 100, 16, 257)])
def test_one_large_value(gpu, heads, group, d, page, length, ratio):
    k, v = (synth.normal(1 + i, (1, heads, length, d), stream=i) for i in range(2))
    q = synth.normal(3, (1, heads * group, 1, d))
    for j in range(heads * group):
        k[:, j // group, :, j % 5] = 0.0  # (up to five of the dims hold the large values)
    for j in range(heads * group):
        q[0, j, 0, j % 5] = ratio * (1 - 2 * (j % 2))
    cache = gpu.PagedKvCache(1, length, -(-length // page), page, heads, d, quantized=True, tracked=True)
    s = cache.add()
    cache.append([s], _t(gpu, k), _t(gpu, v))
    m = Model(heads, d)
    m.append(k[0], v[0], True)
    got = cache.attend([s], _t(gpu, q), 0.35, accumulate=True).numpy()
    want, tol, wtol = m.attend(q[0, :, 0], 0.35, True)  # (its bound goes by |k| |q|, which the large value is no part of)
    assert (np.abs(got[0, :, 0] - want) <= tol[:, None]).all(), float((np.abs(got[0, :, 0] - want) / tol[:, None]).max())
    assert (np.abs(cache.track([s])[0].numpy()[0] - np.stack(m.w)) <= wtol).all()


@pytest.mark.parametrize("size", [1e-36, 1e-20, 1e20, 3e38])
def test_queries_of_any_size(gpu, size):
    heads, d, length = 2, 128, 300
    k, v = (synth.normal(1 + i, (1, heads, length, d), stream=i) for i in range(2))
    q = synth.normal(3, (1, 4, 1, d))
    q = (q / np.abs(q).max() * size).astype(np.float32)
    cache = gpu.PagedKvCache(1, length, 32, 16, heads, d, quantized=True)
    s = cache.add()
    cache.append([s], _t(gpu, k), _t(gpu, v))
    m = Model(heads, d)
    m.append(k[0], v[0], True)
    scale = min(1.0 / size, 1e30)
    got = cache.attend([s], _t(gpu, q), scale).numpy()
    want, tol, _ = m.attend(q[0, :, 0], float(np.float32(scale)), False)
    if size < 1e-29:  # (so small that the queries' own bits are lost: their scores are off by half a unit of 1e-29 / 2^31)
        tol = tol + 2 * 0.5 * 1e-29 / 2 ** 31 * scale * np.abs(np.stack(m.k)).sum(-1).max() * np.abs(v).max()
    assert (np.abs(got[0, :, 0] - want) <= tol[:, None]).all()
