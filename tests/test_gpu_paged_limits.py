"""The paged cache and the norm with rotation where sizes and values are unusual: rows behind 2^32 elements of a pool, prompts
of more pages and sequences than one launch takes, empty calls, infinite scores and values, one tensor as queries and keys,
and two threads at once."""
import threading

import numpy as np
import pytest
import torch

from framework_amd import synth
from test_gpu_paged_cache import U, Model, _check_contents, _t
from test_gpu_qk_norm_rope import _close_rows, _rotate64

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("quantized", [False, True])
def test_rows_behind_the_first_four_billion_elements(gpu, rocm, quantized):
    heads, d, page, pages = 64, 256, 1024, 260  # 16.8 million elements a page
    cache = gpu.PagedKvCache(3, 300000, pages, page, heads, d, quantized=quantized, tracked=True)
    front, back = cache.add(), cache.add()
    zeros = gpu.Tensor.zeros([1, heads, 16384, d])
    for _ in range(16):
        cache.append([front], zeros, zeros)
    assert pages - cache.freePages() == 256 and cache.length(front) == 262144
    m, q = Model(heads, d), synth.normal(3, (1, 2 * heads, 1, d))
    k, v = (synth.normal(1 + i, (1, heads, 1100, d), stream=i) for i in range(2))
    cache.append([back], _t(gpu, k), _t(gpu, v))
    m.append(k[0], v[0], quantized)
    got = cache.attend([back], _t(gpu, q), 0.1, accumulate=True).numpy()
    want, tol, wtol = m.attend(q[0, :, 0], 0.1, True)
    assert (np.abs(got[0, :, 0] - want) <= tol[:, None]).all()
    w = _check_contents(gpu, cache, back, m, True)
    assert (np.abs(w - np.stack(m.w)) <= wtol + 4 * U).all()
    m.w = list(w.astype(np.float64))
    cache.evict([back], 1030, 10)
    m.evict(1030, 10)
    _check_contents(gpu, cache, back, m, True)
    # the copy that a fork's first row takes of the page that both end in
    fork, n = cache.fork(back), m.copy()
    cache.append([fork], _t(gpu, k[:, :, :1]), _t(gpu, v[:, :, :1]))
    n.append(k[0, :, :1], v[0, :, :1], quantized)
    _check_contents(gpu, cache, fork, n, False)
    _check_contents(gpu, cache, back, m, False)
    cache.free()
    gpu.native.resetEngine()
    rocm.clear_cache()


def test_prompts_of_more_pages_and_sequences_than_a_launch_takes(gpu):
    heads, d, n = 2, 8, 40
    cache = gpu.PagedKvCache(n, 1600, 8000, 1, heads, d, quantized=False)
    seqs = [cache.add() for _ in range(n)]
    for lens in ([1500, 700, 3, 1, 0, 704, 705] + [20 + i for i in range(n - 7)], [1] * 5 + [30] * (n - 5)):
        longest = max(lens)
        k, v = (synth.normal(longest + i, (n, heads, longest, d), stream=i) for i in range(2))
        before = [cache.length(s) for s in seqs]
        cache.append(seqs, _t(gpu, k), _t(gpu, v), lens)
        for i, s in enumerate(seqs):
            if before[i] + lens[i]:
                got = [t.numpy()[:, before[i]:] for t in cache.read(s)]
                assert np.array_equal(got[0], k[i, :, :lens[i]]) and np.array_equal(got[1], v[i, :, :lens[i]]), i


def test_nothing_to_do(gpu):
    heads, d = 2, 16
    cache = gpu.PagedKvCache(3, 16, 4, 8, heads, d, quantized=True, tracked=True)
    a, b = cache.add(), cache.add()
    T = lambda *shape: gpu.Tensor.zeros(list(shape))  # noqa: E731
    cache.append([], T(0, heads, 3, d), T(0, heads, 3, d))
    cache.append([a, b], T(2, heads, 0, d), T(2, heads, 0, d))
    cache.append([a, b], T(2, heads, 3, d), T(2, heads, 3, d), [0, 0])
    assert cache.length(a) == 0 and cache.freePages() == 4
    assert cache.attend([], T(0, 4, 1, d), 1.0).shape == [0, 4, 1, d]
    assert (cache.attend([a, b], T(2, 4, 1, d), 1.0, accumulate=True).numpy() == 0).all()
    assert [t.shape for t in cache.read(a)] == [[heads, 0, d]] * 2
    w, _ = cache.track([a, b])
    assert w.shape == [2, heads, 0]
    cache.addWeights([a, b], T(2, heads, 0))
    cache.evict([a, b], 0)
    cache.truncate([a, b], [0, 0])
    cache.truncate([], [])
    cache.evict([], 4)
    c = cache.fork(a)
    one = gpu.Tensor.ones([1, heads, 1, d])
    cache.append([c], one, one)
    cache.evict([c], 0)  # everything leaves
    assert cache.length(c) == 0 and cache.seen(c) == 1 and cache.freePages() == 4
    y, z = gpu.qkNormRope(T(2, 3, 0, d), T(2, 1, 0, d), T(d), T(d))
    assert y.shape == [2, 3, 0, d] and z.shape == [2, 1, 0, d]


@pytest.mark.parametrize("d,page", [(64, 16), (128, 8), (7, 16), (256, 64), (96, 2)])
def test_infinite_scores_and_values(gpu, d, page):
    """Scores of -inf weigh nothing, whole chunks of them neither; an infinite value shows in its own dim alone."""
    heads, group, gone, left = 2, 2, 1700, 301
    cache = gpu.PagedKvCache(1, 2048, 2048 // page, page, heads, d, quantized=False, tracked=True)
    s = cache.add()
    k, v = (synth.normal(1 + i, (1, heads, gone + left, d), stream=i) for i in range(2))
    q = synth.normal(3, (1, heads * group, 1, d))
    q[..., 0] = 1.0
    k[:, :, :gone, 0] = -np.inf
    v[:, :, -1, 3] = np.inf
    cache.append([s], _t(gpu, k), _t(gpu, v))
    got = cache.attend([s], _t(gpu, q), 0.125, accumulate=True).numpy()[0, :, 0]
    m = Model(heads, d)
    v[:, :, -1, 3] = 0.0
    m.append(k[0, :, gone:], v[0, :, gone:], False)
    want, tol, wtol = m.attend(q[0, :, 0], 0.125, True)
    rest = np.arange(d) != 3
    assert (got[:, 3] == np.inf).all() and (np.abs(got - want)[:, rest] <= tol[:, None]).all()
    w = cache.track([s])[0].numpy()[0]
    assert (w[:, :gone] == 0).all() and (np.abs(w[:, gone:] - np.stack(m.w)) <= wtol).all()
    # nothing but -inf: 0 / 0, as the formula has it
    cache.truncate([s], [gone])
    assert np.isnan(cache.attend([s], _t(gpu, q), 0.125).numpy()).all()


def test_one_tensor_as_queries_and_keys(gpu):
    b, h, s, d = 2, 3, 5, 32
    x, g = synth.normal(1, (b, h, s, d)), (1.0 + 0.25 * synth.normal(2, (d,))).astype(np.float32)
    up = [synth.normal(3 + i, (b, h, s, d), stream=i) for i in range(2)]
    x_t, g_t = _t(gpu, x).setRequiresGrad(True), _t(gpu, g).setRequiresGrad(True)
    y, z = gpu.qkNormRope(x_t, x_t, g_t, g_t, offset=-9)
    y.mul(_t(gpu, up[0])).sum().add(z.mul(_t(gpu, up[1])).sum()).backward()
    xr, gr = torch.from_numpy(x).double().requires_grad_(True), torch.from_numpy(g).double().requires_grad_(True)
    want = _rotate64(xr, gr, torch.arange(s)[None].double().repeat(b, 1) - 9, d, False, 10000.0, 1e-6)
    (want * torch.from_numpy(up[0].astype(np.float64) + up[1])).sum().backward()
    assert np.array_equal(y.numpy(), z.numpy())
    r = 1.0 / np.sqrt((x.astype(np.float64) ** 2).mean(-1, keepdims=True) + 1e-6)
    _close_rows(y.numpy(), want.detach().numpy(), d, (np.abs(x) * r * np.abs(g)).max(-1, keepdims=True))
    # as one operand's gradients (2 d + 16 half steps of the two terms, twice that for a margin), once for each use, and
    # half a step for their sum
    xa, ua = np.abs(x).astype(np.float64), sum(np.abs(u).max(-1, keepdims=True) for u in up)
    scale = np.sqrt(2.0) * ua * np.abs(g).max() * (r + xa * r ** 3 * xa.mean(-1, keepdims=True))
    assert (np.abs(x_t.grad.numpy() - xr.grad.numpy()) <= 2.0 * (2 * d + 17) * U * scale).all()
    scale = (np.sqrt(2.0) * ua * xa * r).sum((0, 1, 2))
    assert (np.abs(g_t.grad.numpy() - gr.grad.numpy()) <= (b * h * s + d + 17) * U * scale).all()


def test_two_threads(gpu):
    """Calls from several threads take turns: every thread's cache holds and answers what it would alone."""
    heads, d, steps = 4, 64, 40
    caches = [gpu.PagedKvCache(2, 64, 16, 8, heads, d, quantized=False) for _ in range(2)]
    seqs = [[c.add(), c.add()] for c in caches]
    rows = [[synth.normal(10 * t + i, (steps, 2, heads, 1, d), stream=i) for i in range(3)] for t in range(2)]
    out, failed = [[None] * steps for _ in range(2)], []

    def work(t):
        try:
            for j in range(steps):
                q, k, v = (_t(gpu, r[j]) for r in rows[t])
                caches[t].append(seqs[t], k, v)
                out[t][j] = caches[t].attend(seqs[t], q, 0.125).numpy()
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(t,)) for t in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    for t in range(2):
        models = [Model(heads, d) for _ in range(2)]
        for j in range(steps):
            for i, m in enumerate(models):
                m.append(rows[t][1][j][i], rows[t][2][j][i], False)
                want, tol, _ = m.attend(rows[t][0][j][i, :, 0], 0.125, False)
                assert (np.abs(out[t][j][i, :, 0] - want) <= tol[:, None]).all()


@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("heads,group,d,page", [(12, 1, 64, 16), (2, 4, 128, 16), (3, 2, 7, 8)])
def test_the_same_bits_whichever_workgroup_ends_last(gpu, heads, group, d, page, quantized):
    """Rows of one to nine chunks: every call gives the first one's bits, and the first one's are right."""
    lens = [1, 64, 128, 129, 300, 577, 1024, 1100]
    n = len(lens)
    cache = gpu.PagedKvCache(n, 1152, sum(-(-x // page) for x in lens), page, heads, d, quantized=quantized)
    seqs, models = [cache.add() for _ in lens], [Model(heads, d) for _ in lens]
    k, v = (synth.normal(1 + i, (n, heads, max(lens), d), stream=i) for i in range(2))
    cache.append(seqs, _t(gpu, k), _t(gpu, v), lens)
    q = synth.normal(3, (n, heads * group, 1, d))
    q_t = _t(gpu, q)
    first = cache.attend(seqs, q_t, 0.2).numpy()
    for i, m in enumerate(models):
        m.append(k[i, :, :lens[i]], v[i, :, :lens[i]], quantized)
        want, tol, _ = m.attend(q[i, :, 0], 0.2, False)
        assert (np.abs(first[i, :, 0] - want) <= tol[:, None]).all(), lens[i]
    outs = [cache.attend(seqs, q_t, 0.2) for _ in range(150)]  # queued one behind the other
    assert all(np.array_equal(o.numpy(), first) for o in outs)
    # one sequence alone is cut into other chunks: as right, not the same bits
    for i, m in enumerate(models):
        got = cache.attend([seqs[i]], _t(gpu, q[i:i + 1]), 0.2).numpy()
        want, tol, _ = m.attend(q[i, :, 0], 0.2, False)
        assert (np.abs(got[0, :, 0] - want) <= tol[:, None]).all(), lens[i]


@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("heads,group,d,page", [(1, 40, 64, 16), (2, 17, 128, 64), (1, 33, 256, 16), (2, 19, 80, 4), (1, 20, 20, 1)])
def test_more_query_heads_than_a_tile_holds(gpu, heads, group, d, page, quantized):
    lens = [3, 700, 0, 131]
    cache = gpu.PagedKvCache(4, 704, sum(-(-x // page) for x in lens), page, heads, d, quantized=quantized, tracked=True)
    seqs, models = [cache.add() for _ in lens], [Model(heads, d) for _ in lens]
    k, v = (synth.normal(1 + i, (4, heads, 700, d), stream=i) for i in range(2))
    cache.append(seqs, _t(gpu, k), _t(gpu, v), lens)
    q = synth.normal(3, (4, heads * group, 1, d))
    plain = cache.attend(seqs, _t(gpu, q), 0.1).numpy()
    got = cache.attend(seqs, _t(gpu, q), 0.1, accumulate=True).numpy()
    weights = cache.track(seqs)[0].numpy()
    for i, m in enumerate(models):
        m.append(k[i, :, :lens[i]], v[i, :, :lens[i]], quantized)
        want, tol, wtol = m.attend(q[i, :, 0], 0.1, True)
        for out in (plain, got):
            assert (np.abs(out[i, :, 0] - want) <= tol[:, None]).all(), i
        assert (np.abs(weights[i, :, :lens[i]] - np.stack(m.w)) <= wtol + 4 * U).all() and (weights[i, :, lens[i]:] == 0).all()


@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("heads,group,d,page,lens", [  # rows that fill the chip, and every width of a tile
    (16, 1, 64, 16, [7000]), (16, 1, 128, 64, [3500, 2701]), (16, 1, 192, 32, [6200]), (32, 1, 256, 16, [3111]),
    (4, 3, 192, 16, [900, 33]), (2, 3, 160, 32, [701]), (2, 2, 224, 16, [500, 1]), (3, 2, 192, 8, [300]), (2, 2, 36, 16, [200, 17])])
def test_every_form_of_attention(gpu, heads, group, d, page, lens, quantized):
    n, longest = len(lens), max(lens)
    cache = gpu.PagedKvCache(n, longest, sum(-(-x // page) for x in lens), page, heads, d, quantized=quantized, tracked=True)
    seqs, models = [cache.add() for _ in lens], [Model(heads, d) for _ in lens]
    k, v = (synth.normal(1 + i, (n, heads, longest, d), stream=i) for i in range(2))
    cache.append(seqs, _t(gpu, k), _t(gpu, v), lens)
    q = synth.normal(3, (n, heads * group, 1, d))
    plain = cache.attend(seqs, _t(gpu, q), 0.08).numpy()
    got = cache.attend(seqs, _t(gpu, q), 0.08, accumulate=True).numpy()
    weights = cache.track(seqs)[0].numpy()
    for i, m in enumerate(models):
        m.append(k[i, :, :lens[i]], v[i, :, :lens[i]], quantized)
        want, tol, wtol = m.attend(q[i, :, 0], 0.08, True)
        for out in (plain, got):
            assert (np.abs(out[i, :, 0] - want) <= tol[:, None]).all(), i
        assert (np.abs(weights[i, :, :lens[i]] - np.stack(m.w)) <= wtol + 4 * U).all()


@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("lens,budget,recent,d", [([20000], 19800, 90, 16), ([16384, 9000], 8999, 8, 7), ([16385], 16384, 0, 4), ([700, 20, 650], 600, 40, 128),
                                                  ([700, 20, 650], 300, 40, 100)])
def test_eviction_by_the_selection_itself_and_by_moves(gpu, lens, budget, recent, d, quantized):
    """Few and many bytes to move, rows of every kind of width, sequences that stay as they are between others."""
    heads, page, n = 2, 16, len(lens)
    cache = gpu.PagedKvCache(n, max(lens), sum(-(-x // page) for x in lens), page, heads, d, quantized=quantized, tracked=True)
    seqs, models = [cache.add() for _ in lens], [Model(heads, d) for _ in lens]
    k, v = (synth.normal(1 + i, (n, heads, max(lens), d), stream=i) for i in range(2))
    cache.append(seqs, _t(gpu, k), _t(gpu, v), lens)
    w = np.abs(synth.normal(5, (n, heads, max(lens))))
    cache.addWeights(seqs, _t(gpu, w))
    cache.evict(seqs, budget, recent)
    for i, m in enumerate(models):
        m.append(k[i, :, :lens[i]], v[i, :, :lens[i]], quantized)
        m.w = [w[i, h, :lens[i]].astype(np.float64) for h in range(heads)]
        m.evict(budget, recent)
        got = _check_contents(gpu, cache, seqs[i], m, True)
        assert np.array_equal(got, np.stack(m.w).astype(np.float32))
