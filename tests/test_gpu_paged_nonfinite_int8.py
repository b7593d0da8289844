"""Infinities and NaN in rows that a paged cache stores as int8: such a row is NaN throughout, as read and as attended to, and
nothing else is touched by it."""
import numpy as np
import pytest

from framework_amd import synth
from test_gpu_paged_cache import Model, _stored, _t

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens", [1, 5])  # appended one by one, and as a prompt
@pytest.mark.parametrize("value", [np.nan, -np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("how", ["first", "last", "all"])
@pytest.mark.parametrize("heads,group,d,page", [(2, 1, 64, 16), (2, 3, 128, 16), (2, 1, 16, 4), (2, 2, 20, 8), (2, 1, 7, 2), (2, 2, 256, 16), (2, 1, 96, 8)])
def test_a_row_with_a_value_that_is_not_finite(gpu, heads, group, d, page, how, value, tokens):
    n, length, bad_at = 3, 5, 2
    k, v = (synth.normal(1 + i, (n, heads, length, d), stream=i) for i in range(2))
    # sequence 0: a key of head 1, sequence 1: a value of head 0; sequence 2 stays as it is
    put = {"first": slice(0, 1), "last": slice(d - 1, d), "all": slice(0, d)}[how]
    k[0, 1, bad_at, put] = value
    v[1, 0, bad_at, put] = value
    cache = gpu.PagedKvCache(n, 16, 16 * n // page + n, page, heads, d, quantized=True, tracked=True)
    seqs = [cache.add() for _ in range(n)]
    for t in range(0, length, tokens):
        cache.append(seqs, _t(gpu, k[:, :, t:t + tokens]), _t(gpu, v[:, :, t:t + tokens]))
    for i, s in enumerate(seqs):
        for got, x, hit in zip((t.numpy() for t in cache.read(s)), (k[i], v[i]), ((0, 1), (1, 0))):
            for h in range(heads):
                for t in range(length):
                    if (i, h) == hit and t == bad_at:
                        assert np.isnan(got[h, t]).all()
                    else:
                        assert np.array_equal(got[h, t], _stored(x[h, t], True))
    q = synth.normal(3, (n, heads * group, 1, d))
    for accumulate in (False, True):
        got = cache.attend(seqs, _t(gpu, q), 0.25, accumulate=accumulate).numpy()
        for i in range(n):
            m = Model(heads, d)
            m.append(np.nan_to_num(k[i], nan=0.0, posinf=0.0, neginf=0.0), np.nan_to_num(v[i], nan=0.0, posinf=0.0, neginf=0.0), True)
            want, tol, _ = m.attend(q[i, :, 0], 0.25, False)
            for j in range(heads * group):
                if (i, j // group) in ((0, 1), (1, 0)):
                    assert np.isnan(got[i, j]).all()
                else:
                    assert (np.abs(got[i, j, 0] - want[j]) <= tol[j]).all()
    w = cache.track(seqs)[0].numpy()
    assert np.isnan(w[0, 1]).all() and np.isfinite(w[0, 0]).all() and np.isfinite(w[1:]).all()
