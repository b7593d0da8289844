"""What the norm-and-rotation and paged-cache entry points refuse before they touch a device."""
import ctypes

import pytest

from framework_amd import native as N


@pytest.fixture(scope="module")
def lib():
    return N.load_library()


def _error(lib):
    return lib.mni_rocm_last_error().decode()


@pytest.mark.parametrize("args,text", [
    ((0, 16, 4, 16, 1, 8, 0, 0), "from 1 up to"), ((1, 0, 4, 16, 1, 8, 0, 0), "from 1 up to"), ((1, 16, 0, 16, 1, 8, 0, 0), "from 1 up to"),
    ((-1, 16, 4, 16, 1, 8, 0, 0), "from 1 up to"), ((1, 1 << 40, 4, 16, 1, 8, 0, 0), "from 1 up to"), ((1 << 30, 16, 4, 16, 1, 8, 0, 0), "from 1 up to"),
    ((1, 16, 4, 12, 1, 8, 0, 0), "no power of two"), ((1, 16, 4, 0, 1, 8, 0, 0), "no power of two"), ((1, 16, 4, 2048, 1, 8, 0, 0), "no power of two"),
    ((1, 16, 4, 16, 0, 8, 0, 0), "from 1 to 256"), ((1, 16, 4, 16, 1, 0, 0, 0), "from 1 to 256"), ((1, 16, 4, 16, 1, 257, 0, 0), "from 1 to 256"),
    ((1, 16, 4, 16, 300, 8, 0, 0), "from 1 to 256"),
    ((1, 16, 1 << 30, 1024, 256, 256, 0, 0), "does not fit"), ((1 << 20, 1 << 30, 1, 16, 1, 8, 0, 1), "does not fit")])
def test_create_refuses(lib, args, text):
    assert lib.mni_paged_cache_create(*args) == N.BAD_ID
    assert text in _error(lib)


def test_unknown_caches_are_errors(lib):
    seqs, lens, ids = (ctypes.c_uint32 * 1)(0), (ctypes.c_int64 * 1)(0), (ctypes.c_uint32 * 2)()
    for got, bad in [(lib.mni_paged_cache_free_pages(77), -1), (lib.mni_paged_cache_add(77), N.BAD_ID), (lib.mni_paged_cache_fork(77, 0), N.BAD_ID),
                     (lib.mni_paged_cache_drop(77, 0), 1), (lib.mni_paged_cache_len(77, 0), -1), (lib.mni_paged_cache_seen(77, 0), -1),
                     (lib.mni_paged_cache_append(77, seqs, 1, 0, 0, None), 1), (lib.mni_paged_cache_truncate(77, seqs, 1, lens), 1),
                     (lib.mni_paged_cache_attend(77, seqs, 1, 0, 1.0, 0), N.BAD_ID), (lib.mni_paged_cache_add_weights(77, seqs, 1, 0), 1),
                     (lib.mni_paged_cache_evict(77, seqs, 1, 1, 0), 1), (lib.mni_paged_cache_track(77, seqs, 1, ids, ids), 1),
                     (lib.mni_paged_cache_read(77, 0, ids), 1)]:
        assert got == bad and "invalid paged cache id: 77" in _error(lib)
    lib.mni_paged_cache_free(77)  # a no-op


def test_norm_and_rotation_refuse(lib):
    def call(backward=False, **kw):
        d = N.Rocm.rope_desc(None, **{**dict(batch=1, seq=1, head_dim=8), **kw})
        if kw.get("batch", 1):
            d.q = N.RopeHeads(None, 1, 8, 8, 8, None)
        return (lib.mni_rocm_qk_norm_rope_backward if backward else lib.mni_rocm_qk_norm_rope)(ctypes.byref(d))

    for kw, text in [({"head_dim": 0}, "head_dim 0"), ({"head_dim": 257}, "head_dim 257"), ({"rotary_dims": 5}, "must be even"), ({"rotary_dims": 10}, "must be even"),
                     ({"rotary_dims": -2}, "must be even"), ({"theta": 0.0}, "theta"), ({"theta": float("nan")}, "theta"), ({"theta": float("inf")}, "theta"),
                     ({"eps": -1e-6}, "eps"), ({"eps": float("nan")}, "eps"), ({"batch": -1}, "negative extent"), ({"seq": -1}, "negative extent"),
                     ({"batch": 1 << 20, "seq": 1 << 20}, "2^31 tokens"), ({"batch": 1 << 62, "seq": 1 << 62}, "2^31 tokens"), ({}, "null operand")]:
        for backward in (False, True):
            assert call(backward, **kw) == 1
            assert text in _error(lib), (kw, _error(lib))
    assert lib.mni_rocm_qk_norm_rope(None) == 1 and "null descriptor" in _error(lib)
    assert lib.mni_rocm_qk_norm_rope_backward(None) == 1 and "null descriptor" in _error(lib)
    assert lib.mni_qk_norm_rope(0, 0, 0, 0, N.BAD_ID, 0, 8, 0, 1e4, 1e-6, None) == 1 and "null out_ids" in _error(lib)


def test_binding_layout():
    # mni_rope_heads: pointer, 4 x int64, 5 pointers; mni_rope_desc as laid out in the header
    assert ctypes.sizeof(N.RopeHeads) == 80 and N.RopeHeads.gamma.offset == 40
    assert ctypes.sizeof(N.RopeDesc) == 9 * 8 + 8 + 160 and N.RopeDesc.q.offset == 80
    d = N.Rocm.rope_desc(dict(x=5, heads=2, strides=(9, 8, 7), gamma=6, out=4), dict(x=1, heads=3, gamma=2, dgamma=11), batch=2, seq=3, head_dim=8, rotary_dims=4,
                         positions=13, position_stride=3, offset=-1, interleaved=True, theta=2.0, eps=0.5)
    assert (d.batch, d.seq, d.head_dim, d.rotary_dims, d.positions, d.position_stride, d.offset, d.theta, d.eps, d.interleaved) == (2, 3, 8, 4, 13, 3, -1, 2.0, 0.5, 1)
    assert (d.q.x, d.q.heads, d.q.batch_stride, d.q.head_stride, d.q.token_stride, d.q.gamma, d.q.out, d.q.grad) == (5, 2, 9, 8, 7, 6, 4, None)
    assert (d.k.x, d.k.batch_stride, d.k.head_stride, d.k.token_stride, d.k.dgamma) == (1, 72, 24, 8, 11)
