"""The paged key-value cache against a plain model in 64 bits: what is stored, attention of one token over ragged
sequences, accumulated weights, eviction, forks, truncation, refusals, and a decoding run next to flashAttention."""
import math

import numpy as np
import pytest

from framework_amd import native as N
from framework_amd import synth

pytestmark = pytest.mark.gpu

U = 2.0 ** -24  # half a step of fp32, relative


def _t(gpu, a):
    a = np.ascontiguousarray(a, dtype=np.float32)
    return gpu.Tensor.fromFloat32(a, list(a.shape))


def _stored(x, quantized):
    """The values a row stands for once stored, computed in fp32 as the cache's rule says."""
    x = np.asarray(x, np.float32)
    if not quantized:
        return x
    scale = np.maximum(np.abs(x).max(-1, keepdims=True) * (np.float32(1.0) / np.float32(127.0)), np.float32(1e-8)).astype(np.float32)
    y = (x * (np.float32(1.0) / scale).astype(np.float32)).astype(np.float32).astype(np.float64)
    codes = np.clip(np.sign(y) * np.floor(np.abs(y) + 0.5), -127, 127).astype(np.float32)
    return (codes * scale).astype(np.float32)


class Model:
    """One sequence: per key head the rows held, their positions and weights."""

    def __init__(self, heads, d):
        self.k, self.v = [[np.zeros((0, d), np.float32) for _ in range(heads)] for _ in range(2)]
        self.pos, self.w = [np.zeros(0, np.int64) for _ in range(heads)], [np.zeros(0, np.float64) for _ in range(heads)]
        self.seen, self.floor, self.heads, self.d = 0, 0, heads, d

    def copy(self):
        m = Model(self.heads, self.d)
        for name in ("k", "v", "pos", "w"):
            setattr(m, name, [a.copy() for a in getattr(self, name)])
        m.seen, m.floor = self.seen, self.floor
        return m

    def __len__(self):
        return len(self.pos[0])

    def append(self, k, v, quantized):
        n = k.shape[1]
        for h in range(self.heads):
            self.k[h] = np.concatenate([self.k[h], _stored(k[h], quantized)])
            self.v[h] = np.concatenate([self.v[h], _stored(v[h], quantized)])
            self.pos[h] = np.concatenate([self.pos[h], self.seen + np.arange(n)])
            self.w[h] = np.concatenate([self.w[h], np.zeros(n)])
        self.seen += n

    def cut(self, n):
        self.seen -= len(self) - n
        for name in ("k", "v", "pos", "w"):
            setattr(self, name, [a[:n] for a in getattr(self, name)])

    def attend(self, q, scale, accumulate):
        """q [H, d]: outputs and how far an fp32 computation may be off them."""
        group = len(q) // self.heads
        out, tol = np.zeros((len(q), self.d)), np.zeros(len(q))
        if len(self) == 0:
            return out, tol + 1e-30, 0.0
        wtol = 0.0
        for j in range(len(q)):
            h = j // group
            k, v = self.k[h].astype(np.float64), self.v[h].astype(np.float64)
            s = k @ q[j].astype(np.float64) * scale
            p = np.exp(s - s.max())
            p /= p.sum()
            out[j] = p @ v
            # a score: d products and their sum, the scale, the row's scale and log2 e (4 more), the difference from the
            # maximum; a probability: e^(twice that), the exponential (2 steps) and the rescaling of every tile and join
            # (at most 24 factors); the two sums over the row: len terms each
            ds = (self.d + 6) * U * (np.abs(k) @ np.abs(q[j].astype(np.float64))).max() * abs(scale) + 2 * U * np.abs(s).max()
            rel = 2 * ds + (2 * len(self) + 64) * U
            tol[j] = rel * np.abs(v).max()
            wtol = max(wtol, rel * p.max() * group)
            if accumulate:
                self.w[h] = self.w[h] + p
        return out, tol, wtol

    def evict(self, budget, recent):
        if len(self) <= budget:
            return
        for h in range(self.heads):
            protected = self.pos[h] >= self.seen - recent
            order = np.lexsort((self.pos[h], -self.w[h], ~protected))
            stays = np.zeros(len(self.pos[h]), bool)
            stays[order[:budget]] = True
            pick = np.arange(budget)
            pick[~stays[:budget]] = np.arange(budget, len(stays))[stays[budget:]]
            for name in ("k", "v", "pos", "w"):
                getattr(self, name)[h] = getattr(self, name)[h][pick]
        self.floor = budget


def _check_contents(gpu, cache, seq, m, tracked):
    n = len(m)
    assert cache.length(seq) == n and cache.seen(seq) == m.seen
    if n == 0:
        return
    k, v = (t.numpy() for t in cache.read(seq))
    assert np.array_equal(k, np.stack(m.k)) and np.array_equal(v, np.stack(m.v))
    if tracked:
        w, p = cache.track([seq])
        assert np.array_equal(gpu.native.intBufferToHost(p).reshape(m.heads, n), np.stack(m.pos))
        return w.numpy()[0]


SHAPES = [  # kv heads, group, D, page size, lengths, longest appended at once
    (12, 1, 64, 16, [57]),
    (2, 1, 64, 16, [1, 15, 16, 17, 0, 33]),
    (3, 2, 128, 8, [1000, 3, 127, 128, 129]),
    (2, 4, 80, 32, [300, 31]),
    (1, 3, 20, 4, [33, 1]),
    (2, 8, 32, 1, [65, 7]),
    (1, 5, 96, 64, [700, 64, 65]),
    (4, 1, 256, 2, [5, 130]),
    (1, 16, 128, 128, [2500]),
    (1, 1, 1, 16, [40]),
    (2, 2, 7, 8, [19, 513]),
    (1, 6, 48, 1024, [1023, 1025]),
    (8, 4, 128, 16, [4097, 1, 900]),
    (2, 7, 64, 16, [0, 0]),
]


@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("heads,group,d,page,lengths", SHAPES)
def test_attention_over_ragged_sequences(gpu, heads, group, d, page, lengths, quantized):
    n, longest = len(lengths), max(max(lengths), 1)
    cache = gpu.PagedKvCache(n + 2, longest + 3, sum(-(-(x + 3) // page) for x in lengths) + 4, page, heads, d, quantized=quantized, tracked=True)
    spare = cache.add()
    seqs = [cache.add() for _ in range(n)][::-1]
    models = [Model(heads, d) for _ in range(n)]
    k, v = (2.0 * synth.normal(1 + i, (n, heads, longest, d), stream=i) for i in range(2))
    cache.append(seqs, _t(gpu, k), _t(gpu, v), lengths)
    for i, m in enumerate(models):
        m.append(k[i, :, :lengths[i]], v[i, :, :lengths[i]], quantized)
    scale = 1.0 / math.sqrt(d)
    for step in range(3):
        q = synth.normal(20 + step, (n, heads * group, 1, d))
        k1, v1 = (synth.normal(30 + step, (n, heads, 1, d), stream=i) for i in range(2))
        if step:
            cache.append(seqs, _t(gpu, k1), _t(gpu, v1))
        q_t = _t(gpu, q if step < 2 else q.reshape(n * heads * group, 1, d))
        out = cache.attend(seqs, q_t, scale, accumulate=step > 0)
        assert out.shape == q_t.shape
        got, wtol = out.numpy().reshape(n, heads * group, d), 0.0
        for i, m in enumerate(models):
            if step:
                m.append(k1[i], v1[i], quantized)
            want, tol, wt = m.attend(q[i, :, 0], scale, step > 0)
            wtol = max(wtol, wt)
            assert (np.abs(got[i] - want) <= tol[:, None]).all(), (step, i, float((np.abs(got[i] - want) / tol[:, None]).max()))
            if len(m) == 0:
                assert (got[i] == 0).all()
    for i, m in enumerate(models):
        w = _check_contents(gpu, cache, seqs[i], m, True)
        if len(m):  # two accumulations
            assert (np.abs(w - np.stack(m.w)) <= 2 * wtol + 4 * U).all()
    assert cache.length(spare) == 0
    # the same call again gives the same bits, in any order of the sequences
    if n:
        a = cache.attend(seqs, _t(gpu, q), scale).numpy()
        b = cache.attend(seqs[::-1], _t(gpu, q[::-1]), scale).numpy()
        c = cache.attend(seqs, _t(gpu, q), scale).numpy()
        assert np.array_equal(a, c)
        if all(len(m) < 2000 for m in models):
            assert np.allclose(a, b[::-1], rtol=0, atol=float(max(m.attend(q[i, :, 0], scale, False)[1].max() for i, m in enumerate(models))) * 2)
    cache.free()


@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("seed,heads,group,d,page", [(1, 2, 2, 64, 8), (2, 3, 1, 32, 4), (3, 1, 4, 128, 16), (4, 2, 1, 20, 1)])
def test_random_program(gpu, seed, heads, group, d, page, quantized):
    """Appends, forks, truncations, evictions, drops in a seeded order: contents, positions, weights and the number of free
    pages stay those of the model, and a refused call changes nothing."""
    rng = np.random.default_rng(seed)
    pages, limit = 96, 40 * page
    cache = gpu.PagedKvCache(6, limit, pages, page, heads, d, quantized=quantized, tracked=True)
    held = {}
    draw = lambda *shape: rng.standard_normal(shape).astype(np.float32)  # noqa: E731
    for turn in range(60):
        what = rng.choice(["add", "fork", "append", "append", "append", "truncate", "evict", "drop", "weigh"])
        live = sorted(held)
        some = [int(x) for x in rng.permutation(live)[:rng.integers(1, 4)]] if live else []
        if what == "add" and len(live) < 6:
            seq = cache.add()
            assert seq not in held
            held[seq] = Model(heads, d)
        elif what == "fork" and live and len(live) < 6:
            seq = cache.fork(some[0])
            held[seq] = held[some[0]].copy()
        elif what == "append" and some:
            t = int(rng.choice([1, 1, page, 3 * page + 1, 7]))
            counts = [int(c) for c in rng.integers(0, t + 1, len(some))] if rng.random() < 0.5 else None
            k, v = draw(len(some), heads, t, d), draw(len(some), heads, t, d)
            before = cache.freePages()
            try:
                cache.append(some, _t(gpu, k), _t(gpu, v), counts)
            except N.MniError as e:
                assert "full" in str(e) and cache.freePages() == before
                continue
            for i, s in enumerate(some):
                c = t if counts is None else counts[i]
                held[s].append(k[i, :, :c], v[i, :, :c], quantized)
        elif what == "truncate" and some:
            lens = [int(rng.integers(min(held[s].floor, len(held[s])), len(held[s]) + 1)) for s in some]
            cache.truncate(some, lens)
            for s, n in zip(some, lens):
                held[s].cut(n)
        elif what == "weigh" and some:
            longest = max(len(held[s]) for s in some) + int(rng.integers(0, 3))
            if longest:
                w = (rng.integers(0, 9, (len(some), heads, longest)) / 4).astype(np.float32)  # exact sums, many ties
                cache.addWeights(some, _t(gpu, w))
                for i, s in enumerate(some):
                    for h in range(heads):
                        held[s].w[h] = held[s].w[h] + w[i, h, :len(held[s])]
        elif what == "evict" and some:
            budget = int(rng.integers(0, 12 * page))
            recent = int(rng.integers(0, budget + 1))
            try:
                cache.evict(some, budget, recent)
            except N.MniError as e:
                assert "shared" in str(e)
                continue
            for s in some:
                held[s].evict(budget, recent)
        elif what == "drop" and live and rng.random() < 0.5:
            cache.drop(some[0])
            del held[some[0]]
        for s in some:
            if s in held:
                w = _check_contents(gpu, cache, s, held[s], True)
                if w is not None:
                    assert np.array_equal(w, np.stack(held[s].w).astype(np.float32)), turn
        gpu.native.gcTensors([])
    for s in sorted(held):  # what was not touched lately as well, and attention over all of it
        _check_contents(gpu, cache, s, held[s], True)
    live = sorted(held)
    if live:
        q = draw(len(live), heads * group, 1, d)
        got = cache.attend(live, _t(gpu, q), 0.3).numpy()
        for i, s in enumerate(live):
            want, tol, _ = held[s].attend(q[i, :, 0], 0.3, False)
            assert (np.abs(got[i, :, 0] - want) <= tol[:, None]).all()
    for s in live:
        cache.drop(s)
    assert cache.freePages() == pages


@pytest.mark.parametrize("length,budget,recent", [(65, 64, 0), (5000, 500, 100), (300, 299, 299), (1100, 1024, 7), (2048, 1, 0), (2048, 1, 1), (700, 650, 0), (40, 0, 0),
                                                  (9000, 8100, 1000), (33000, 3000, 50)])
@pytest.mark.parametrize("kind", ["spread", "equal", "extremes"])
def test_eviction_keeps_the_heaviest(gpu, length, budget, recent, kind):
    heads, d, page = 2, 16, 16
    cache = gpu.PagedKvCache(2, length + 8, 2 * (-(-length // page)) + 8, page, heads, d, quantized=False, tracked=True)
    s = cache.add()
    m = Model(heads, d)
    k, v = (synth.normal(1 + i, (1, heads, length, d), stream=i) for i in range(2))
    cache.append([s], _t(gpu, k), _t(gpu, v))
    m.append(k[0], v[0], False)
    w = np.abs(synth.normal(5, (1, heads, length)))
    if kind == "equal":
        w[:] = 0.0
    elif kind == "extremes":  # lowest, highest, infinite, negative, minus zero, subnormal
        special = np.array([0.0, -0.0, np.inf, -np.inf, 3e38, -3e38, 1e-42, -1e-42], np.float32)
        w = special[synth.integers(6, (1, heads, length), 0, len(special))]
    cache.addWeights([s], _t(gpu, w))
    for h in range(heads):
        m.w[h] = (np.float32(0.0) + w[0, h]).astype(np.float64)
    cache.evict([s], budget, recent)
    m.evict(budget, recent)
    got = _check_contents(gpu, cache, s, m, True)
    if budget:
        assert np.array_equal(got, np.stack(m.w).astype(np.float32))
    assert cache.freePages() == 2 * (-(-length // page)) + 8 - -(-budget // page)
    # nothing to do the second time
    cache.evict([s], budget, recent)
    _check_contents(gpu, cache, s, m, True)
    with pytest.raises(N.MniError, match="cannot be cut"):
        if budget:
            cache.truncate([s], [budget - 1])
        else:
            cache.truncate([s], [1])


def test_a_nan_weight_is_the_largest(gpu):
    cache = gpu.PagedKvCache(1, 64, 8, 16, 1, 8, quantized=False, tracked=True)
    s = cache.add()
    k = synth.normal(1, (1, 1, 40, 8))
    cache.append([s], _t(gpu, k), _t(gpu, k))
    w = np.arange(40, dtype=np.float32)[None, None] + 1
    w[0, 0, [3, 9]] = np.nan
    cache.addWeights([s], _t(gpu, w))
    cache.evict([s], 4, 0)
    _, p = cache.track([s])
    assert sorted(gpu.native.intBufferToHost(p)) == [3, 9, 38, 39]


def test_forks_share_pages_until_one_writes(gpu):
    heads, d, page = 2, 32, 8
    cache = gpu.PagedKvCache(4, 64, 12, page, heads, d, quantized=True, tracked=True)
    a = cache.add()
    k, v = (synth.normal(1 + i, (1, heads, 20, d), stream=i) for i in range(2))
    cache.append([a], _t(gpu, k), _t(gpu, v))
    assert cache.freePages() == 9
    b, c = cache.fork(a), cache.fork(a)
    assert cache.freePages() == 9 and cache.length(b) == 20
    rest = [synth.normal(9 + i, (3, heads, 1, d), stream=i) for i in range(2)]
    cache.append([b, a, c], _t(gpu, rest[0]), _t(gpu, rest[1]))  # two copies of the last page; the third writes in place
    assert cache.freePages() == 7
    models = []
    for i in range(3):
        m = Model(heads, d)
        m.append(k[0], v[0], True)
        m.append(rest[0][i], rest[1][i], True)
        models.append(m)
    for s, m in zip((b, a, c), models):
        _check_contents(gpu, cache, s, m, True)
    # weights are a sequence's own
    q = synth.normal(30, (1, heads, 1, d))
    cache.attend([b], _t(gpu, q), 0.2, accumulate=True)
    assert (cache.track([a])[0].numpy() == 0).all() and cache.track([b])[0].numpy().sum() == pytest.approx(heads, rel=1e-5)
    # eviction of one fork leaves the others as they are, and is refused when its copies find no room
    cache.addWeights([b], _t(gpu, np.arange(heads * 21, dtype=np.float32).reshape(1, heads, 21)))
    got = cache.track([b])[0].numpy()[0].astype(np.float64)
    models[0].w = [got[h] for h in range(heads)]
    cache.evict([b], 10, 2)
    models[0].evict(10, 2)
    for s, m in zip((b, a, c), models):
        _check_contents(gpu, cache, s, m, True)
    fill = cache.add()
    free = cache.freePages()
    cache.append([fill], _t(gpu, np.zeros((1, heads, free * page, d))), _t(gpu, np.zeros((1, heads, free * page, d))))
    with pytest.raises(N.MniError, match="pages are shared and only 0 are free"):
        cache.evict([a], 10, 2)
    with pytest.raises(N.MniError, match=r"the cache is full \(1 pages wanted, 0 free\)"):
        cache.append([fill], _t(gpu, np.zeros((1, heads, 1, d))), _t(gpu, np.zeros((1, heads, 1, d))))
    for s, m in zip((b, a, c), models):
        _check_contents(gpu, cache, s, m, True)


def test_many_sequences_take_several_launches(gpu):
    n, heads, d, page = 300, 1, 32, 4
    cache = gpu.PagedKvCache(n, 24, n * 5, page, heads, d, quantized=False, tracked=True)
    seqs = [cache.add() for _ in range(n)]
    lens = [int(x) for x in synth.integers(1, (n,), 0, 18)]
    k, v = (synth.normal(1 + i, (n, heads, 17, d), stream=i) for i in range(2))
    cache.append(seqs, _t(gpu, k), _t(gpu, v), lens)
    one = [synth.normal(4 + i, (n, heads, 1, d), stream=i) for i in range(2)]
    cache.append(seqs, _t(gpu, one[0]), _t(gpu, one[1]))
    q = synth.normal(7, (n, 2, 1, d))
    got = cache.attend(seqs, _t(gpu, q), 0.2, accumulate=True).numpy()
    w, p = cache.track(seqs)
    w, p = w.numpy(), gpu.native.intBufferToHost(p).reshape(n, heads, -1)
    models = []
    for i in range(n):
        m = Model(heads, d)
        m.append(k[i, :, :lens[i]], v[i, :, :lens[i]], False)
        m.append(one[0][i], one[1][i], False)
        want, tol, wtol = m.attend(q[i, :, 0], 0.2, True)
        assert (np.abs(got[i, :, 0] - want) <= tol[:, None]).all(), i
        assert (np.abs(w[i, 0, :len(m)] - m.w[0]) <= wtol).all() and (w[i, 0, len(m):] == 0).all()
        assert list(p[i, 0]) == list(range(len(m))) + [-1] * (p.shape[2] - len(m))
        m.w = [w[i, 0, :len(m)].astype(np.float64)]
        models.append(m)
    cache.evict(seqs, 9, 3)
    for i in range(0, n, 17):
        models[i].evict(9, 3)
        _check_contents(gpu, cache, seqs[i], models[i], True)


def test_views_non_finite_rows_and_what_lies_behind_the_end(gpu):
    heads, d, page = 2, 16, 8
    cache = gpu.PagedKvCache(2, 64, 16, page, heads, d, quantized=False)
    a, b = cache.add(), cache.add()
    # NaN and infinity in rows that leave again, so that they lie behind the end of what is attended to
    bad = np.full((1, heads, 13, d), np.nan, np.float32)
    bad[:, :, ::2] = np.inf
    cache.append([a], _t(gpu, bad), _t(gpu, bad))
    cache.truncate([a], [0])
    x = synth.normal(1, (2, 5, 2 * heads, d))  # [B, T, heads, D], read as views
    cache.append([a, b], _t(gpu, x[:, :, :heads]).permute(0, 2, 1, 3), _t(gpu, x[:, :, heads:]).permute(0, 2, 1, 3))
    odd = _t(gpu, x[:, :, :heads].transpose(0, 2, 3, 1).copy()).permute(0, 1, 3, 2)  # last extent not contiguous: gathered first
    cache.append([a, b], odd, odd)
    q = synth.normal(3, (2, heads, 1, d))
    got = cache.attend([a, b], _t(gpu, q), 0.25).numpy()
    for i in range(2):
        m = Model(heads, d)
        rows = x[i].transpose(1, 0, 2)
        m.append(rows[:heads], rows[heads:], False)
        m.append(rows[:heads], rows[:heads], False)
        want, tol, _ = m.attend(q[i, :, 0], 0.25, False)
        assert (np.abs(got[i, :, 0] - want) <= tol[:, None]).all()
    # a row of infinities that is attended to shows, as the formula says
    cache.append([a], _t(gpu, bad[:, :, :1]), _t(gpu, bad[:, :, :1]))
    got = cache.attend([a, b], _t(gpu, q), 0.25).numpy()
    assert np.isnan(got[0]).all() and np.isfinite(got[1]).all()


def test_refusals_change_nothing(gpu):
    heads, d = 2, 16
    cache = gpu.PagedKvCache(2, 20, 3, 8, heads, d, quantized=True)
    a = cache.add()
    T = lambda *shape: gpu.Tensor.zeros(list(shape))  # noqa: E731
    k = T(1, heads, 4, d)
    cache.append([a], k, k)
    for f, text in [(lambda: cache.append([a, a], T(2, heads, 1, d), T(2, heads, 1, d)), "occurs twice"),
                    (lambda: cache.append([5], k, k), "invalid paged cache sequence id: 5"), (lambda: cache.append([1], k, k), "invalid paged cache sequence id: 1"),
                    (lambda: cache.append([a], k, T(1, heads, 3, d)), "k/v shapes must match"), (lambda: cache.append([a], T(1, 1, 4, d), T(1, 1, 4, d)), r"expected \[1, 2, T, 16\]"),
                    (lambda: cache.append([a], T(heads, 4, d), T(heads, 4, d)), r"expected \[1, 2, T, 16\]"), (lambda: cache.append([a], k, k, [5]), r"counts\[0\] = 5 of 4"),
                    (lambda: cache.append([a], k, k, [-1]), r"counts\[0\] = -1"), (lambda: cache.append([a], k, k, [1, 2]), "2 counts for 1"),
                    (lambda: cache.append([a], T(1, heads, 17, d), T(1, heads, 17, d)), "is full"),
                    (lambda: cache.attend([a], T(1, 3, 1, d), 1.0), "no multiple"), (lambda: cache.attend([a], T(1, 1, 1, d), 1.0), "no multiple"),
                    (lambda: cache.attend([a], T(1, 2, 2, d), 1.0), r"expected \[1, H, 1, 16\]"), (lambda: cache.attend([a], T(2, 2, 1, d), 1.0), r"expected \[1, H, 1, 16\]"),
                    (lambda: cache.attend([a], T(1, 2, 1, 8), 1.0), r"expected \[1, H, 1, 16\]"), (lambda: cache.attend([a], T(1, 2, 1, d), 1.0, True), "needs a tracked cache"),
                    (lambda: cache.evict([a], 2), "not tracked"), (lambda: cache.track([a]), "not tracked"), (lambda: cache.addWeights([a], T(1, heads, 4)), "not tracked"),
                    (lambda: cache.truncate([a], [5]), "cannot be cut to 5"), (lambda: cache.truncate([a], [-1]), "cannot be cut to -1"), (lambda: cache.read(9), "sequence id: 9"),
                    (lambda: cache.drop(1), "sequence id: 1"), (lambda: cache.fork(1), "sequence id: 1")]:
        with pytest.raises(N.MniError, match=text):
            f()
        assert cache.length(a) == 4 and cache.seen(a) == 4 and cache.freePages() == 2
    cache.add()
    with pytest.raises(N.MniError, match="all 2 sequences are in use"):
        cache.add()
    tracked = gpu.PagedKvCache(1, 20, 3, 8, heads, d, tracked=True)
    s = tracked.add()
    tracked.append([s], k, k)
    for f, text in [(lambda: tracked.evict([s], 2, 3), "must hold the 3 recent"), (lambda: tracked.evict([s], -1, 0), "must hold"), (lambda: tracked.evict([s, s], 2, 0), "occurs twice"),
                    (lambda: tracked.addWeights([s], T(1, heads, 3)), "at least 4"), (lambda: tracked.attend([s, s], T(2, 2, 1, d), 1.0, True), "occurs twice")]:
        with pytest.raises(N.MniError, match=text):
            f()
    assert tracked.attend([s, s], T(2, 2, 1, d), 1.0).shape == [2, 2, 1, d]  # reading twice is fine
    first = cache.cacheId
    gpu.native.resetEngine()
    assert gpu.PagedKvCache(1, 8, 1, 8, 1, 8).cacheId == 1 and first >= 1


@pytest.mark.parametrize("quantized", [False, True])
def test_decoding_next_to_attention_over_the_prompt(gpu, quantized):
    """As a program uses them: a prompt through norm, rotation and flashAttention into the cache, then token after token;
    every token's attention is what one causal pass over the whole sequence gives, within the cache's rounding."""
    b, heads, d, prompt, steps, page = 2, 4, 64, 37, 9, 16
    total = prompt + steps
    q, k, v = (synth.normal(1 + i, (b, total, heads, d), stream=i) for i in range(3))
    g = (1.0 + 0.1 * synth.normal(7, (d,))).astype(np.float32)
    gain = _t(gpu, g)
    scale = 1.0 / math.sqrt(d)
    view = lambda a, lo, hi: _t(gpu, a[:, lo:hi]).permute(0, 2, 1, 3)  # noqa: E731
    qr, kr = gpu.qkNormRope(view(q, 0, total), view(k, 0, total), gain, gain)
    flat = lambda t: t.contiguous().view(b * heads, total, d)  # noqa: E731
    whole = gpu.flashAttention(flat(qr), flat(kr), flat(view(v, 0, total)), scale, True).numpy().reshape(b, heads, total, d)
    cache = gpu.PagedKvCache(b, 64, 8, page, heads, d, quantized=quantized, tracked=True)
    seqs = [cache.add() for _ in range(b)]
    qp, kp = gpu.qkNormRope(view(q, 0, prompt), view(k, 0, prompt), gain, gain)
    assert np.array_equal(kp.numpy(), kr.numpy()[:, :, :prompt])
    cache.append(seqs, kp, view(v, 0, prompt))
    for t in range(prompt, total):
        at = gpu.native.createDataset(np.array([cache.seen(s) for s in seqs], np.int32))
        qt, kt = gpu.qkNormRope(view(q, t, t + 1), view(k, t, t + 1), gain, gain, positions=at)
        cache.append(seqs, kt, view(v, t, t + 1))
        got = cache.attend(seqs, qt, scale, accumulate=True).numpy()
        krn = np.abs(kr.numpy()).max()
        # fp32: two computations of the same sums; int8: half a code of 1 / 127 in every key and value
        tol = 2e-5 * np.abs(v).max() if not quantized else np.abs(v).max() / 254 + np.abs(v).max() * 2 * d * scale * np.abs(qt.numpy()).max() * krn / 254
        assert np.abs(got[:, :, 0] - whole[:, :, t]).max() <= tol
    weights = cache.track(seqs)[0].numpy()
    assert np.abs(weights.sum(-1) - steps).max() <= 1e-4
    cache.evict(seqs, 24, 8)
    kept = gpu.native.intBufferToHost(cache.track(seqs)[1]).reshape(b, heads, 24)
    for i in range(b):
        for h in range(heads):
            rest = np.sort(weights[i, h, :total - 8])[::-1]
            assert set(range(total - 8, total)) <= set(kept[i, h]) and len(set(kept[i, h])) == 24
            assert weights[i, h, [p for p in kept[i, h] if p < total - 8]].min() >= rest[15]
