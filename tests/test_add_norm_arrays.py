"""The arrays that MoeContext.AddNormI8 takes: by a stand-in for the library which type it is asked for and which bytes it is given,
and on the GPU bf16 rows, as their bits, against the definition."""
import ctypes as C

import numpy as np
import pytest

import half_ref as ref
import i8_ref

F32 = np.float32


class Library:
    """Device buffers are host memory; phx_add_norm_i8 notes its type and the bytes of x and branch, and answers zeros."""

    def __init__(self):
        self.kept, self.calls = {}, []

    def phx_moe_dev_alloc(self, h, n, out):
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

    def phx_moe_sync(self, h):
        return 0

    def phx_add_norm_i8(self, h, type_, x, branch, w, rows, n, ld, eps, total, out_type, out, qs, d):
        size = rows * n * (4 if type_ == 0 else 2)
        self.calls.append((type_, C.string_at(x, size), C.string_at(branch, size)))
        return 0


@pytest.fixture
def host(pkg):
    c = pkg.MoeContext.__new__(pkg.MoeContext)
    c.lib, c.h = Library(), 1
    return c


@pytest.mark.parametrize("dtype,type_", [(F32, 0), (np.float16, 1), (np.uint16, 30)])
def test_types(host, dtype, type_):
    rng = np.random.default_rng(type_)
    x, b = ((100 * rng.random((3, 32))).astype(dtype) for _ in range(2))
    s, v, q, d = host.AddNormI8(x, b, np.ones(32))
    assert host.lib.calls == [(type_, x.tobytes(), b.tobytes())]
    assert s.dtype == dtype and v.dtype == F32 and q.dtype == np.int8 and d.dtype == F32
    assert not host.lib.kept


def test_float_types_beside_each_other(host):
    """float64 goes as float32, a branch as x's type: what these calls did before."""
    host.AddNormI8(np.ones((1, 32)), np.ones((1, 32), np.float16), np.ones(32))
    host.AddNormI8(np.ones((1, 32), np.float16), np.ones((1, 32)), np.ones(32))
    assert [c[0] for c in host.lib.calls] == [0, 1]
    assert host.lib.calls[0][2] == np.ones(32, F32).tobytes() and host.lib.calls[1][2] == np.ones(32, np.float16).tobytes()


@pytest.mark.parametrize("other", [F32, np.float16, np.float64, np.int32])
def test_bf16_bits_beside_numbers_are_refused(host, pkg, other):
    bits, numbers = np.full((2, 32), 0x3F80, np.uint16), np.ones((2, 32), other)
    for x, b in ((bits, numbers), (numbers, bits)):
        with pytest.raises(pkg.ArgumentError):
            host.AddNormI8(x, b, np.ones(32))
    assert not host.lib.calls


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n", [(1, 32), (5, 2816), (300, 1056)])
def test_bf16_rows(ctx, rows, n):
    rng = np.random.default_rng(n)
    raw_x, x = ref.held(3 * rng.standard_normal((rows, n)), 30)
    raw_b, b = ref.held(rng.standard_normal((rows, n)), 30)
    w = (1 + 0.2 * rng.standard_normal(n)).astype(F32)
    s, v, q, d = ctx.AddNormI8(raw_x, raw_b, w)
    bits, total = ref.held(x.astype(F32) + b.astype(F32), 30)
    np.testing.assert_array_equal(s, bits)
    normed = i8_ref.rms_norm(total, w, 1e-6)
    np.testing.assert_array_equal(v, normed.astype(F32))
    for got, want in zip((q, d), i8_ref.quant(normed)):
        np.testing.assert_array_equal(got, want)
