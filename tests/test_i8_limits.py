"""The limits that the header declares for the int8 calls are the ones the calls have: taken at the limit, refused past it with
the limit named."""
import re
from pathlib import Path

import numpy as np
import pytest

import i8_ref as ref

HEADER = (Path(__file__).resolve().parent.parent / "include" / "phx_moe.h").read_text()
NAMES = ("MAX_ROWS_I8", "MAX_COLS_I8", "MAX_MATRIX_I8")


def comment_of(function):
    """The header's comment right above a function's declaration."""
    return re.search(r"/\*((?:(?!\*/).)*)\*/\s*int " + function + r"\(", HEADER, flags=re.S).group(1)


@pytest.mark.parametrize("name", NAMES)
def test_python_mirror(pkg, name):
    assert f"#define PHX_{name} {getattr(pkg.PHX, name)}\n" in HEADER


@pytest.mark.parametrize("function,names", [("phx_route", NAMES[:1]), ("phx_quant_i8", NAMES[:2]), ("phx_weight_upload_i8", NAMES),
                                            ("phx_matmul_i8", NAMES[:1]), ("phx_experts_i8", NAMES[:1])])
def test_declared_by_name(function, names):
    text = comment_of(function)
    for name in names:
        assert f"<= PHX_{name}" in text or f"at most PHX_{name}" in text, name
    assert not re.search(r"<= 2\^|<= \d{5}|at most \d{5}", text)


@pytest.mark.gpu
def test_rows_at_the_limit(ctx, pkg):
    n, most = 32, pkg.PHX.MAX_ROWS_I8
    x = np.random.default_rng(0).integers(-128, 128, (most, n)).astype(np.float32)
    x[:, 5] = 127 * (1 + np.arange(most) % 5)
    q, d = ctx.QuantI8(0, x)
    rq, rd = ref.quant(x)
    np.testing.assert_array_equal(q, rq)
    np.testing.assert_array_equal(d, rd)
    w, scale = ref.weights_of(np.random.default_rng(1), 3, n)
    h = ctx.weight_upload_i8(1, 3, n, w, scale)
    try:
        np.testing.assert_array_equal(ctx.MatMulI8(h, 3, n, q, d), ref.product_f32(q, d, w, scale))
        a = ctx.alloc(4096)
        with pytest.raises(pkg.ArgumentError, match=str(most)):
            ctx.quant_i8_device(0, 0, a.ptr, None, most + 1, n, n, 0.0, a.ptr, a.ptr)
        with pytest.raises(pkg.ArgumentError):
            ctx.matmul_i8_device(h, most + 1, a.ptr, a.ptr, 0, a.ptr)
        a.free()
    finally:
        ctx.weight_free(h)


@pytest.mark.gpu
def test_matrix_limits(ctx, pkg):
    P, at = pkg.PHX, np.zeros(16, np.float32).ctypes.data  # refused by the sizes alone: nothing is read
    for rows, cols, limit in ((P.MAX_ROWS_I8 + 1, 32, P.MAX_ROWS_I8), (32, P.MAX_COLS_I8 + 32, P.MAX_COLS_I8),
                              (P.MAX_MATRIX_I8 // P.MAX_COLS_I8 + 1, P.MAX_COLS_I8, P.MAX_MATRIX_I8)):
        with pytest.raises(pkg.ArgumentError, match=str(limit)):
            ctx.weight_upload_i8(1, rows, cols, at, at)
