"""What a launch that fails in the middle of a call leaves of a paged cache: every sequence as it was, or wholly changed."""
import numpy as np
import pytest

from framework_amd import native as N
from framework_amd import synth
from test_gpu_paged_cache import Model, _check_contents, _t

pytestmark = pytest.mark.gpu


@pytest.fixture()
def fail(rocm):
    yield rocm.test_fail_paged_launch
    rocm.test_fail_paged_launch(0)


def _attends(gpu, cache, seqs, models, heads, d):
    q = synth.normal(77, (len(seqs), heads, 1, d))
    got = cache.attend(seqs, _t(gpu, q), 0.2).numpy()
    for i, m in enumerate(models):
        want, tol, _ = m.attend(q[i, :, 0], 0.2, False)
        assert (np.abs(got[i, :, 0] - want) <= tol[:, None]).all(), i


@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("n,tokens,launch", [(300, 1, 1), (300, 1, 2), (300, 1, 3), (70, 9, 1), (70, 9, 3), (3, 720, 1)])
def test_an_append_that_fails_leaves_every_sequence_as_it_was(gpu, fail, n, tokens, launch, quantized):
    heads, d, page = 2, 16, 1
    cache = gpu.PagedKvCache(n, 2 * tokens + 8, n * (2 * tokens + 8), page, heads, d, quantized=quantized, tracked=True)
    seqs, models = [cache.add() for _ in range(n)], [Model(heads, d) for _ in range(n)]
    lens = [i % 4 for i in range(n)]
    k, v = (synth.normal(1 + i, (n, heads, 3, d), stream=i) for i in range(2))
    cache.append(seqs, _t(gpu, k), _t(gpu, v), lens)
    for i, m in enumerate(models):
        m.append(k[i, :, :lens[i]], v[i, :, :lens[i]], quantized)
    free = cache.freePages()
    k, v = (synth.normal(11 + i, (n, heads, tokens, d), stream=i) for i in range(2))
    fail(launch)
    with pytest.raises(N.MniError, match="paged_append failed"):
        cache.append(seqs, _t(gpu, k), _t(gpu, v))
    assert cache.freePages() == free
    for i in list(range(0, n, 37)) + [n - 1]:
        _check_contents(gpu, cache, seqs[i], models[i], True)
    _attends(gpu, cache, seqs, models, heads, d)
    # others may take the pages; the same call again is as if nothing had happened
    for i in range(1, n, 2):
        cache.append([seqs[i]], _t(gpu, v[i:i + 1]), _t(gpu, k[i:i + 1]))
        models[i].append(v[i], k[i], quantized)
    even = list(range(0, n, 2))
    cache.append([seqs[i] for i in even], _t(gpu, k[even]), _t(gpu, v[even]))
    for i in even:
        models[i].append(k[i], v[i], quantized)
    for i in list(range(0, n, 37)) + [n - 1]:
        _check_contents(gpu, cache, seqs[i], models[i], True)
    _attends(gpu, cache, seqs, models, heads, d)


@pytest.mark.parametrize("launch", [1, 2, 3])  # both launches of copies, then the append's own
@pytest.mark.parametrize("tokens", [1, 7])
def test_copies_that_fail_leave_the_pages_shared(gpu, fail, tokens, launch):
    heads, d, page, n = 1, 16, 8, 260
    cache = gpu.PagedKvCache(n, 32, 3 * n, page, heads, d, quantized=False, tracked=True)
    first = cache.add()
    k, v = (synth.normal(1 + i, (1, heads, 11, d), stream=i) for i in range(2))
    cache.append([first], _t(gpu, k), _t(gpu, v))
    seqs = [first] + [cache.fork(first) for _ in range(n - 1)]
    models = []
    for _ in range(n):
        models.append(Model(heads, d))
        models[-1].append(k[0], v[0], False)
    free = cache.freePages()
    k, v = (synth.normal(11 + i, (n, heads, tokens, d), stream=i) for i in range(2))
    fail(launch)
    with pytest.raises(N.MniError, match="paged_copy failed" if launch < 3 else "paged_append failed"):
        cache.append(seqs, _t(gpu, k), _t(gpu, v))
    assert cache.freePages() == (free if launch == 1 else free - 224 if launch == 2 else free - (n - 1))
    for i in (0, 1, 100, 223, 224, 225, n - 1):
        _check_contents(gpu, cache, seqs[i], models[i], True)
    fail(0)
    cache.append(seqs, _t(gpu, k), _t(gpu, v))
    for i, m in enumerate(models):
        m.append(k[i], v[i], False)
        _check_contents(gpu, cache, seqs[i], m, True)
    for s in seqs:
        cache.drop(s)
    assert cache.freePages() == 3 * n


@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("launch,cut", [(1, 0), (2, 128), (3, 256)])
def test_an_eviction_that_fails_has_cut_sequences_wholly_or_not_at_all(gpu, fail, launch, cut, quantized):
    heads, d, page, n, length = 1, 16, 4, 300, 40
    cache = gpu.PagedKvCache(n, length + 4, n * (length // page + 1), page, heads, d, quantized=quantized, tracked=True)
    seqs, models = [cache.add() for _ in range(n)], [Model(heads, d) for _ in range(n)]
    k, v = (synth.normal(1 + i, (n, heads, length, d), stream=i) for i in range(2))
    w = np.abs(synth.normal(5, (n, heads, length)))
    cache.append(seqs, _t(gpu, k), _t(gpu, v))
    cache.addWeights(seqs, _t(gpu, w))
    for i, m in enumerate(models):
        m.append(k[i], v[i], quantized)
        m.w = [w[i, h].astype(np.float64) for h in range(heads)]
    fail(launch)
    with pytest.raises(N.MniError, match="paged_select failed"):
        cache.evict(seqs, 18, 5)
    for i, m in enumerate(models):
        if i < cut:
            m.evict(18, 5)
        if i % 37 == 0 or i in (127, 128, 255, 256, n - 1):
            _check_contents(gpu, cache, seqs[i], m, True)
    _attends(gpu, cache, seqs, models, heads, d)
    cache.evict(seqs, 18, 5)
    for i, m in enumerate(models):
        m.evict(18, 5)
        _check_contents(gpu, cache, seqs[i], m, True)
