"""Long reductions of the float products, experts and adapters on small whole numbers, whose sums are exact in float whatever their order: results
equal to the definition to the last bit, so that a step of a reduction that is lost, or counted twice, shows."""
import numpy as np
import pytest

import half_ref as ref
import half_rules as rules
from test_gpu_experts_terms import call as experts_call
from test_gpu_half import upload
from test_gpu_i8 import Bufs
from test_gpu_lora import run as lora_run

pytestmark = pytest.mark.gpu

F32 = np.float32


def whole(rng, shape, most, type_):
    v = rng.integers(-most, most + 1, shape).astype(F32)
    return ref.held(v, type_)[0], v


# single places, the row kernel's two tiles, the tile kernel's two; columns that end inside a step
@pytest.mark.parametrize("type_", [1, 30])
@pytest.mark.parametrize("E,n,rows,cols,cap", [(1, 1, 40, 65536, 16), (2, 9, 20, 65528, 16), (1, 100, 70, 16392, 32), (9, 60, 40, 4104, 16), (1, 700, 2432, 4104, 128),
                                               (1, 700, 2432, 4096, 128), (3, 2100, 4128, 1000, 128), (1, 2200, 16384, 520, 256)])
@pytest.mark.parametrize("paired", [False, True])
def test_products(ctx, type_, E, n, rows, cols, cap, paired):
    """Paired: a gate of 64 and more, whose act(g) is g itself."""
    print(f"exact: type {type_} E {E} n {n} {rows} x {cols} paired {paired}", flush=True)
    assert rules.capacity(n, E, rows, paired) == cap
    rng = np.random.default_rng(n + rows + cols)
    raw_x, x = whole(rng, (n, cols), 2, type_)
    raw_w, w = whole(rng, (E, rows, cols), 2, type_)
    offsets = np.linspace(0, n, E + 1).astype(np.int32)
    if paired:  # gate rows: a one in the first column alone, against 64 and more; up: nothing there
        raw_w[:, :rows // 2] = 0
        raw_w[:, rows // 2:, 0] = 0
        w[:, :rows // 2], w[:, rows // 2:, 0] = 0, 0
        raw_w[:, :rows // 2, 0] = ref.held(np.ones(1), type_)[0]
        raw_x[:, 0], x[:, 0] = ref.held(64 + np.arange(n) % 64, type_)
    h = ctx.weight_upload_half(type_, E, rows, cols, raw_w, paired=paired)
    try:
        with Bufs(ctx) as B:
            out = rows // 2 if paired else rows
            y = B.empty(n * out * 4)
            ctx.matmul_grouped_device(h, 1 if paired else 0, n, B.of(offsets).ptr, B.of(raw_x).ptr, n, None, 0, y.ptr)
            ctx.sync()
            got = y.download((n, out))
    finally:
        ctx.weight_free(h)
    for e in range(E):
        p = slice(offsets[e], offsets[e + 1])
        want = x[p] @ w[e][-out:].T  # exact in float: at most 2^18 in magnitude, in any order
        np.testing.assert_array_equal(got[p], want * x[p, :1] if paired else want)


@pytest.mark.parametrize("type_", [1, 30])
@pytest.mark.parametrize("T,k,E,d,nf", [(1, 4, 8, 1024, 1704), (12, 2, 20, 1032, 1704), (60, 4, 8, 1024, 1704), (900, 2, 4, 1032, 1704), (1500, 2, 4, 1032, 520)])
def test_experts(ctx, type_, T, k, E, d, nf):
    """h = g u with g from 64 to 95 and u of up to 600 or so: 16 bits, whole in two terms; the second sum under 2^24."""
    print(f"exact experts: type {type_} T {T} k {k} E {E} d {d} nf {nf}", flush=True)
    rng = np.random.default_rng(T + d + nf)
    raw_x, x = whole(rng, (T, d), 1, type_)
    raw_x[:, 0], x[:, 0] = ref.held(64 + np.arange(T) % 32, type_)
    raw_g, wg = whole(rng, (E, 2 * nf, d), 1, type_)
    raw_g[:, :nf], wg[:, :nf] = 0, 0
    raw_g[:, nf:, 0], wg[:, nf:, 0] = 0, 0
    raw_g[:, :nf, 0], wg[:, :nf, 0] = ref.held(np.ones(1), type_)[0], 1
    raw_d, wd = whole(rng, (E, d, nf), 1, type_)
    ids = rng.integers(-1, E, (T, k)).astype(np.int32)
    weights = rng.integers(1, 3, (T, k)).astype(F32)
    hs = upload(ctx, type_, (raw_g, raw_d), E, d, nf)
    try:
        got = experts_call(ctx, hs, 1, raw_x, ids, weights, 0, d)
    finally:
        for h in hs:
            ctx.weight_free(h)
    want = np.zeros((T, d))
    for e in range(E):
        t, j = np.nonzero(ids == e)
        u = x[t].astype(np.float64) @ wg[e, nf:].astype(np.float64).T
        hv = u * x[t, :1]
        assert np.abs(hv).max(initial=0) < 65504
        y = hv @ wd[e].astype(np.float64).T
        assert (np.abs(hv) @ np.abs(wd[e]).astype(np.float64).T).max(initial=0) < 2 ** 23  # so exact in any order
        np.add.at(want, t, y * weights[t, j][:, None])
    assert np.abs(want).max() < 2 ** 24
    np.testing.assert_array_equal(got, want)


@pytest.mark.parametrize("type_", [1, 30])
@pytest.mark.parametrize("T,rows,cols,rank", [(1, 70, 65536, 20), (40, 130, 16392, 33), (1100, 72, 8200, 16), (700, 64, 4104, 128)])
def test_adapters(ctx, type_, T, rows, cols, rank):
    """A x at most 2^9 or so in magnitude: whole in the first term and the second."""
    rng = np.random.default_rng(T + cols)
    raw_x, x = whole(rng, (T, cols), 1, type_)
    raw_a, a = whole(rng, (2, rank, cols), 1, type_)
    raw_b, b = whole(rng, (2, rows, rank), 2, type_)
    ids = np.arange(T) // 3 % 3 - 1
    h = ctx.lora_create(type_, 2, rank, rows, cols)
    try:
        for s in range(2):
            ctx.lora_set(h, s, rank, raw_a[s], raw_b[s])
        got = lora_run(ctx, h, T, raw_x, ids, 0, rows, rows, np.ones((T, rows), F32))
    finally:
        ctx.lora_free(h)
    want = np.ones((T, rows))
    for s in range(2):
        low = x[ids == s].astype(np.float64) @ a[s].T
        assert np.abs(low).max(initial=0) < 2 ** 14
        want[ids == s] += low @ b[s].T
    np.testing.assert_array_equal(got, want)
