"""The residual's addition and the norm of the sum as int8 rows (phx_add_norm_i8): sums, quants and scales equal to the definition
(tests/i8_ref.py) and to phx_quant_i8 of the stored sum bit for bit, at odd sizes, each type, in place and apart, rows that hold
an infinity or a NaN, and the refusals."""
import numpy as np
import pytest

import half_ref as ref
import i8_ref
from test_gpu_i8 import Bufs

pytestmark = pytest.mark.gpu

F32 = np.float32
EPS = 1e-6


def check(ctx, rows, n, type_, out_type, in_place=False, extra=0, x=None, with_out=True):
    print(f"add_norm rows {rows} n {n} type {type_} out {out_type} in place {in_place} ld +{extra}", flush=True)
    rng = np.random.default_rng(rows + n + type_)
    raw_x, xv = ref.held(3 * rng.standard_normal((rows, n)) if x is None else x, type_)
    raw_b, bv = ref.held(rng.standard_normal((rows, n + extra)), type_)
    w = (1 + 0.2 * rng.standard_normal(n)).astype(F32)
    item, out_item = raw_x.itemsize, 4 if out_type == 0 else 2
    with Bufs(ctx) as B:
        fill = lambda size: B.of(np.full(size + 64, 0x3C, np.uint8))  # noqa: E731
        xb, out, qs, d = B.of(raw_x), fill(rows * n * out_item), fill(rows * n), fill(rows * 4)
        total = xb if in_place else fill(rows * n * item)
        bb, wb = B.of(raw_b), B.of(w)
        ctx.add_norm_i8_device(type_, xb.ptr, bb.ptr, wb.ptr, rows, n, n + extra, EPS, total.ptr, out_type,
                               out.ptr if with_out else None, qs.ptr, d.ptr)
        q2, d2 = B.empty(rows * n), B.empty(rows * 4)
        ctx.quant_i8_device(2, type_, total.ptr, wb.ptr, rows, n, n, EPS, q2.ptr, d2.ptr)
        ctx.sync()
        s = ref.read(total, (rows, n), type_)
        v, q, dv = ref.read(out, (rows, n), out_type), qs.download((rows, n), np.int8), d.download(rows)
        same = q2.download((rows, n), np.int8), d2.download(rows)
        for b, size in ((out, rows * n * out_item if with_out else 0), (qs, rows * n), (d, rows * 4)) + (() if in_place else ((total, rows * n * item),)):
            assert (b.download(size + 64, np.uint8)[size:] == 0x3C).all()
        if not in_place:
            np.testing.assert_array_equal(xb.download(raw_x.shape, raw_x.dtype).view(np.uint8), raw_x.view(np.uint8))
    with np.errstate(over="ignore", invalid="ignore"):
        want = ref.held(xv.astype(F32) + bv[:, :n].astype(F32), type_)[1]
    np.testing.assert_array_equal(s, want)
    np.testing.assert_array_equal(q, same[0])
    np.testing.assert_array_equal(dv.view(np.uint32), same[1].view(np.uint32))
    with np.errstate(over="ignore", invalid="ignore"):
        normed = i8_ref.rms_norm(want, w, EPS)
        rq, rd = i8_ref.quant(normed)
        if with_out:
            np.testing.assert_array_equal(v, ref.held(normed, out_type)[1])
    np.testing.assert_array_equal(q, rq)
    np.testing.assert_array_equal(dv, rd)


@pytest.mark.parametrize("type_,out_type", [(0, 0), (0, 30), (1, 1), (1, 0), (30, 30), (30, 1)])
@pytest.mark.parametrize("n", [32, 96, 704, 1056, 2048, 2080, 4096, 4128, 8192, 8224, 20000])
def test_rows(ctx, n, type_, out_type):
    check(ctx, 5, n, type_, out_type, extra=24)
    check(ctx, 3, n, type_, out_type, in_place=True)


@pytest.mark.parametrize("n", [16384, 16416, 32768, 32800, 65504, 65536])
def test_long_rows(ctx, n):
    check(ctx, 4, n, 30, 0, extra=8)
    check(ctx, 2, n, 0, 1, in_place=True)


@pytest.mark.parametrize("rows,n", [(1, 2816), (1200, 1088), (70001, 32), (1 << 20, 32)])
def test_many_rows(ctx, rows, n):
    check(ctx, rows, n, 30, 30, in_place=True)


@pytest.mark.parametrize("n", [64, 3200, 9000 // 32 * 32])
def test_without_float_rows(ctx, n):
    check(ctx, 7, n, 30, 30, with_out=False)
    check(ctx, 7, n, 0, 0, in_place=True, with_out=False)


def test_longest_rows(ctx):
    check(ctx, 2, 65536, 0, 30, in_place=True)
    check(ctx, 2, 65536, 30, 0)


def test_in_place_often(ctx):
    """Long rows over several waves in place: no wave reads what another has stored."""
    for seed in range(5):
        check(ctx, 700 + seed, 2400, 30, 30, in_place=True)


def test_sums_of_the_other_sign(ctx):
    """Sums that cancel to zero: rows of zeros."""
    x = np.zeros((3, 64), F32)
    got = ctx.AddNormI8(x + 1, x - 1, np.ones(64, F32))
    assert (got[0] == 0).all() and (got[1] == 0).all() and (got[2] == 0).all() and (got[3] == 0).all()


@pytest.mark.parametrize("n", [64, 1120, 5024])
@pytest.mark.parametrize("dtype", [np.float16, F32])
def test_infinities_and_nans(ctx, n, dtype):
    """A row that holds one after the addition says so in its scale; the others are as they would be."""
    rng = np.random.default_rng(n)
    x, b = rng.standard_normal((7, n)).astype(dtype), rng.standard_normal((7, n)).astype(dtype)
    w = np.ones(n, F32)
    clean = ctx.AddNormI8(x, b, w)
    x[1, n - 1], x[3, 0], b[5, n // 2] = np.inf, np.nan, -np.inf
    x[6, 0] = b[6, 0] = 6e4 if dtype == np.float16 else 3e38  # the sum overflows
    s, v, q, d = ctx.AddNormI8(x, b, w)
    bad = np.array([1, 3, 5, 6])
    assert np.isnan(d[bad]).all() and (q[bad] == 0).all()
    for got, same in zip((s, v, q, d), clean):
        np.testing.assert_array_equal(np.delete(got, bad, 0), np.delete(same, bad, 0))


def test_refusals(ctx, pkg):
    A, N, P = pkg.ArgumentError, pkg.NotSupportedError, pkg.PHX
    with Bufs(ctx) as B:
        x, b, w, s, o, q, d = (B.empty(4096).ptr for _ in range(7))
        host = np.zeros(4096, np.uint8).ctypes.data

        def call(type_=0, x=x, b=b, w=w, rows=2, n=64, ld=64, eps=EPS, s=s, out_type=0, o=o, q=q, d=d):
            ctx.add_norm_i8_device(type_, x, b, w, rows, n, ld, eps, s, out_type, o, q, d)
        call()
        call(o=None)
        call(s=x)
        for bad in (dict(rows=0), dict(rows=P.MAX_ROWS_I8 + 1), dict(n=0), dict(n=48), dict(n=P.MAX_COLS_I8 + 32, ld=P.MAX_COLS_I8 + 32), dict(ld=56),
                    dict(ld=68), dict(ld=(1 << 40) + 8), dict(eps=-1.0), dict(eps=float("nan")), dict(x=None), dict(b=None), dict(w=None), dict(s=None),
                    dict(q=None), dict(d=None), dict(x=x + 8), dict(b=b + 8), dict(w=w + 4), dict(s=s + 8), dict(o=o + 8), dict(q=q + 4), dict(d=d + 2),
                    dict(x=host), dict(b=host), dict(w=host), dict(s=host), dict(o=host), dict(q=host), dict(d=host), dict(s=x + 16), dict(s=b),
                    dict(s=w), dict(o=x), dict(o=s), dict(q=o), dict(d=q), dict(s=x, o=x), dict(q=b)):
            with pytest.raises(A):
                call(**bad)
        for bad in (dict(type_=2), dict(out_type=8)):
            with pytest.raises(N):
                call(**bad)
        ctx.sync()
    for bad in ((np.zeros((2, 32)), np.zeros((2, 64)), np.zeros(32)), (np.zeros((2, 32)), np.zeros((2, 32)), np.zeros(64)), (np.zeros(32), np.zeros(32), np.zeros(32))):
        with pytest.raises(A):
            ctx.AddNormI8(*bad)


@pytest.mark.parametrize("n,what", enumerate(("x", "sum", "branch", "w", "qs", "d", "out"), 1))
def test_memory_of_another_gpu(pkg, monkeypatch, n, what):
    monkeypatch.setenv("PHX_FAULT", f"device:{n}")
    with pkg.MoeContext(0) as c:
        x = np.ones((2, 32), F32)
        with pytest.raises(pkg.ArgumentError, match=f"{what} is memory of device"):
            c.AddNormI8(x, x, x[0])
        assert (c.AddNormI8(x, x, x[0])[0] == 2).all()
