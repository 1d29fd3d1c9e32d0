"""MoeContext.MatMulGrouped's device buffers, without a GPU: none is left behind when a later one cannot be had."""
import ctypes as C

import numpy as np
import pytest


class Library:
    """Device memory for `most` buffers at a time; products do nothing."""

    def __init__(self, most):
        self.most, self.kept = most, {}

    def phx_weight_shape(self, h, *sizes):
        for p, v in zip(sizes, (2, 16, 8)):
            p._obj.value = v
        return 0

    def phx_moe_dev_alloc(self, h, n, out):
        if len(self.kept) == self.most:
            return -2
        b = C.create_string_buffer(n)
        self.kept[C.addressof(b)] = b
        out._obj.value = C.addressof(b)
        return 0

    def phx_moe_dev_free(self, h, p):
        del self.kept[p]
        return 0

    def phx_moe_memcpy_h2d(self, h, to, at, n):
        C.memmove(to, at, n)
        return 0

    phx_moe_memcpy_d2h = phx_moe_memcpy_h2d

    def phx_moe_last_error(self, h):
        return b""

    def __getattr__(self, name):
        return lambda *args: 0


@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("most", range(5))
def test_no_buffer_is_left(pkg, most, gather):
    c = pkg.MoeContext.__new__(pkg.MoeContext)
    c.lib, c.h = Library(most), 1
    x, src = np.ones((5, 8), np.float16), np.arange(5) if gather else None
    if most < 3 + gather:
        with pytest.raises(pkg.MoeError):
            c.MatMulGrouped(7, 0, np.array([0, 2, 5]), x, src)
    else:
        assert (c.MatMulGrouped(7, 0, np.array([0, 2, 5]), x, src) == np.zeros((5, 16))).all()
    assert not c.lib.kept
