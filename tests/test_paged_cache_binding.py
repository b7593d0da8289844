"""Ids and lengths that do not fit the C ABI's types are errors of the Python binding; ctypes would cut them to others."""
import pytest

from framework_amd import native as N


@pytest.fixture()
def native():
    class Lib:
        def __getattr__(self, name):
            def called(*args):
                raise AssertionError("the library was called: " + name)
            return called
    n = N.Native.__new__(N.Native)
    n.lib = Lib()
    return n


@pytest.mark.parametrize("bad", [-1, 1 << 32, (1 << 32) + 1, 1 << 64])
def test_ids(native, bad):
    for f in ("Fork", "Drop", "Len", "Seen", "Read"):
        for args in ((1, bad), (bad, 0)):
            with pytest.raises(N.MniError, match="out of range"):
                getattr(native, "pagedCache" + f)(*args)
    for f in (native.pagedCacheFree, native.pagedCacheFreePages, native.pagedCacheAdd):
        with pytest.raises(N.MniError, match="out of range"):
            f(bad)
    for c, s in ((bad, [0]), (1, [bad]), (1, [0, bad])):
        for f, rest in (("Append", (0, 0)), ("Truncate", ([0] * len(s),)), ("Attend", (0, 1.0, False)), ("AddWeights", (0,)), ("Evict", (4, 0)), ("Track", ())):
            with pytest.raises(N.MniError, match="out of range"):
                getattr(native, "pagedCache" + f)(c, s, *rest)
    with pytest.raises(N.MniError, match="out of range"):
        native.qkNormRope(0, 0, 0, 0, bad, 0, 8, False, 1e4, 1e-6)


@pytest.mark.parametrize("bad", [1 << 63, -(1 << 63) - 1, 1 << 64])
def test_lengths(native, bad):
    for f in (lambda: native.pagedCacheEvict(1, [0], bad, 0), lambda: native.pagedCacheEvict(1, [0], 4, bad), lambda: native.pagedCacheTruncate(1, [0], [bad]),
              lambda: native.pagedCacheAppend(1, [0], 0, 0, [bad]), lambda: native.pagedCacheCreate(1, bad, 1, 1, 1, 1, False, False),
              lambda: native.qkNormRope(0, 0, 0, 0, None, bad, 8, False, 1e4, 1e-6), lambda: native.qkNormRope(0, 0, 0, 0, None, 0, bad, False, 1e4, 1e-6)):
        with pytest.raises(N.MniError, match="out of range"):
            f()
