"""What calls with more rows than one grid holds do, on small sizes: the limit that they split themselves by is lowered."""
import numpy as np
import pytest

from framework_amd import native as N
from framework_amd import synth
from test_gpu_paged_cache import U, Model, _check_contents, _t

pytestmark = pytest.mark.gpu


@pytest.fixture()
def small_grids(rocm):
    rocm.test_grid_threads(4096)  # 16 workgroups
    yield
    rocm.test_grid_threads(0)


@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("heads,group,d,page", [(2, 2, 64, 16), (3, 1, 7, 8), (1, 4, 128, 4), (2, 1, 96, 32)])
def test_paged_cache(gpu, small_grids, heads, group, d, page, quantized):
    lens = [3000, 1, 700, 0, 2100]
    n = len(lens)
    cache = gpu.PagedKvCache(n, 3008, sum(-(-(x + 1) // page) for x in lens), page, heads, d, quantized=quantized, tracked=True)
    seqs, models = [cache.add() for _ in lens], [Model(heads, d) for _ in lens]
    k, v = (synth.normal(1 + i, (n, heads, 3000, d), stream=i) for i in range(2))
    cache.append(seqs, _t(gpu, k), _t(gpu, v), lens)
    one = [synth.normal(5 + i, (n, heads, 1, d), stream=i) for i in range(2)]
    cache.append(seqs, _t(gpu, one[0]), _t(gpu, one[1]))
    q = synth.normal(3, (n, heads * group, 1, d))
    plain = cache.attend(seqs, _t(gpu, q), 0.1).numpy()
    got = cache.attend(seqs, _t(gpu, q), 0.1, accumulate=True).numpy()
    weights = cache.track(seqs)[0].numpy()
    for i, m in enumerate(models):
        m.append(k[i, :, :lens[i]], v[i, :, :lens[i]], quantized)
        m.append(one[0][i], one[1][i], quantized)
        want, tol, wtol = m.attend(q[i, :, 0], 0.1, True)
        for out in (plain, got):
            assert (np.abs(out[i, :, 0] - want) <= tol[:, None]).all(), i
        w = weights[i, :, :len(m)]
        assert (np.abs(w - np.stack(m.w)) <= wtol + 4 * U).all() and (weights[i, :, len(m):] == 0).all()
        m.w = list(w.astype(np.float64))
    cache.evict(seqs, 1000, 17)
    for s, m in zip(seqs, models):
        m.evict(1000, 17)
        _check_contents(gpu, cache, s, m, True)


@pytest.mark.parametrize("b,s,hq,hk,d,rotary", [(2, 301, 3, 1, 64, 64), (1, 403, 2, 1, 7, 4), (1, 9001, 6, 2, 32, 16), (3, 77, 2, 2, 256, 256)])
def test_norm_and_rotation(gpu, rocm, b, s, hq, hk, d, rotary):
    q, k, g = _t(gpu, synth.normal(1, (b, hq, s, d))), _t(gpu, synth.normal(2, (b, hk, s, d))), _t(gpu, np.ones(d))
    want = [t.numpy() for t in gpu.qkNormRope(q, k, g, g, rotaryDims=rotary)]
    rocm.test_grid_threads(4096)
    try:
        got = [t.numpy() for t in gpu.qkNormRope(q, k, g, g, rotaryDims=rotary)]
    finally:
        rocm.test_grid_threads(0)
    assert all(np.array_equal(x, y) for x, y in zip(want, got))


def test_the_limit_is_checked(rocm):
    for bad in (-1, 1, 4095, 1 << 32):
        with pytest.raises(N.MniError, match="test_grid_threads"):
            rocm.test_grid_threads(bad)
