"""NaN and infinities through the int8 rows and experts: the row that holds one says so in its scale, whatever the mode, and the
rows beside it are as they would be without it."""
import numpy as np
import pytest

import i8_ref as ref

pytestmark = pytest.mark.gpu

F32 = np.float32
EPS = 1e-6


@pytest.mark.parametrize("mode", [0, 1, 2, 3])
@pytest.mark.parametrize("type_", [0, 1])
@pytest.mark.parametrize("n", [32, 1056, 2048, 4128, 9024])
def test_rows(ctx, orc, n, type_, mode):
    """A NaN or infinity at the first, a middle or the last place of a row, in x and in aux."""
    print(f"quant_i8 nan: mode {mode} type {type_} n {n}", flush=True)
    rng = np.random.default_rng(n + mode)
    places, values = (0, n // 2 + 3, n - 1), (np.nan, np.inf, -np.inf)
    rows = 2 * len(places) * len(values) + 3
    x = rng.standard_normal((rows, n)).astype(F32)
    aux = rng.standard_normal((rows, n)).astype(F32)
    r = 1
    for a in (x, aux):
        for at in places:
            for v in values:
                a[r, at] = v
                r += 1
    if type_:
        x, aux = x.astype(np.float16), aux.astype(np.float16)
    weight = (1 + 0.2 * rng.standard_normal(n)).astype(F32)
    q, d = ctx.QuantI8(mode, x, None if mode == 0 else weight if mode == 2 else aux, EPS)
    xf, af = x.astype(F32), aux.astype(F32)
    with np.errstate(all="ignore"):
        v = xf if mode == 0 else ref.rms_norm(xf, weight, EPS) if mode == 2 else (
            (orc.silu(xf) if mode == 1 else orc.gelu(xf)) * af).astype(F32)
    bad = ~np.isfinite(v).all(axis=1)
    nan = np.isnan(xf).any(axis=1) | (np.isnan(af).any(axis=1) & (mode in (1, 3)))
    assert nan.any() and bad[nan].all() and not bad[0] and not bad[-1]
    rq, rd = ref.quant(v)
    np.testing.assert_array_equal(np.isnan(d), bad)
    np.testing.assert_array_equal(q, rq)
    np.testing.assert_array_equal(d[~bad], rd[~bad])


@pytest.mark.parametrize("mode", [0, 1, 3])
def test_rows_of_bf16(ctx, orc, mode):
    n, rows = 2048, 6
    rng = np.random.default_rng(mode)
    x, aux = (ref.bf16_bits(rng.standard_normal((rows, n)).astype(F32)) for _ in range(2))
    x[1, 7], x[3, n - 1], aux[4, 0] = 0x7FC1, 0xFFC0, 0x7FC0
    bufs = [ctx.alloc(b) for b in (x.nbytes, aux.nbytes, rows * n, rows * 4)]
    try:
        bufs[0].upload(x)
        bufs[1].upload(aux)
        ctx.quant_i8_device(mode, 30, bufs[0].ptr, bufs[1].ptr if mode else None, rows, n, n, EPS, bufs[2].ptr, bufs[3].ptr)
        ctx.sync()
        q, d = bufs[2].download((rows, n), np.int8), bufs[3].download(rows)
    finally:
        for b in bufs:
            b.free()
    bad = np.isin(np.arange(rows), [1, 3, 4] if mode else [1, 3])
    np.testing.assert_array_equal(np.isnan(d), bad)
    assert (q[bad] == 0).all()
    xf, af = ref.bf16_value(x), ref.bf16_value(aux)
    with np.errstate(all="ignore"):
        v = xf if mode == 0 else ((orc.silu(xf) if mode == 1 else orc.gelu(xf)) * af).astype(F32)
    rq, rd = ref.quant(v)
    np.testing.assert_array_equal(q, rq)
    np.testing.assert_array_equal(d[~bad], rd[~bad])


@pytest.mark.parametrize("act", [1, 3])
@pytest.mark.parametrize("T", [1, 20, 400])
def test_experts_with_a_nan_gate(ctx, T, act):
    """A gate channel whose scale is a NaN reaches every token of its expert and no other: in single assignments, in lists and
    in the tile kernel."""
    E, d, nf, k = 6, 64, 96, 2
    rng = np.random.default_rng(T)
    wg, sg = ref.weights_of(rng, E, 2 * nf, d)
    wd, sd = ref.weights_of(rng, E, d, nf)
    sg[4, nf - 1] = np.nan  # the up half stays finite
    xq, xd = ref.rows_of(rng, T, d)
    ids = np.argsort(rng.random((T, E)), axis=1)[:, :k].astype(np.int32)
    ids[0] = 4, 1
    hs = ctx.weight_upload_i8(E, 2 * nf, d, wg, sg, paired=True), ctx.weight_upload_i8(E, d, nf, wd, sd)
    try:
        out = ctx.ExpertsI8(*hs, act, xq, xd, ids, np.ones((T, k), F32))
    finally:
        for h in hs:
            ctx.weight_free(h)
    has = (ids == 4).any(axis=1)
    assert np.isnan(out[has]).all() and np.isfinite(out[~has]).all()
