"""The int8 kernels at the lengths of real layers, where each form runs its steady state: reductions longer than the loads kept
ahead, rows of several steps a thread, a wave's second place of the down kernel, every expert that a router may have.  What a
call launches tells its form: two launches for single assignments, five for lists."""
import functools
import os

import numpy as np
import pytest

import i8_ref as ref
from test_gpu_i8 import EPS, F32, Bufs, check_experts, check_product, held, transformed, upload

pytestmark = pytest.mark.gpu


@functools.lru_cache(maxsize=1)
def experts_of(E, d, nf):
    """Matrices of random bytes: quick to make where there are many."""
    rng = np.random.default_rng(E + nf)
    return (rng.integers(-90, 91, (E, 2 * nf, d), dtype=np.int8), (6e-4 * (1 + 0.3 * rng.random((E, 2 * nf)))).astype(F32),
            rng.integers(-90, 91, (E, d, nf), dtype=np.int8), (6e-4 * (1 + 0.3 * rng.random((E, d)))).astype(F32))


def launches(pkg, W, T, k):
    """How many kernels an experts call of these sizes launches, 2 or more than 2: the fault plan skips the third."""
    E, n2, d = W[0].shape
    tiny = np.zeros((E, n2, d), np.int8), np.ones((E, n2), F32), np.zeros((E, d, n2 // 2), np.int8), np.ones((E, d), F32)
    os.environ["PHX_FAULT"] = f"launch:{2 * E + 3}"  # after a launch for each uploaded matrix
    try:
        c = pkg.MoeContext(0)
    finally:
        del os.environ["PHX_FAULT"]
    with c:
        hs = upload(c, tiny)
        try:
            c.ExpertsI8(*hs, 1, np.zeros((T, d), np.int8), np.zeros(T, F32), np.zeros((T, k), np.int32), np.zeros((T, k), F32))
            return 2
        except pkg.GpuDeviceLostError:
            return 3
        finally:
            for h in hs:
                c.weight_free(h)


def run(ctx, pkg, orc, W, T, k, act, types=(0, 1, 30), skip=()):
    rng = np.random.default_rng(T * k)
    E, _, d = W[0].shape
    xq, xd = ref.rows_of(rng, T, d)
    ids = rng.integers(0, E, (T, k)).astype(np.int32)
    for t, j in skip:
        ids[t, j] = -1
    check_experts(ctx, pkg, orc, W, xq, xd, ids, rng.standard_normal((T, k)).astype(F32), act, types=types)


# E, d, nf, T, k: nf within one load of 12 steps, past it, past two, and of no whole step; a wave's second and further places (k
# past 8, or past 4 with 4 waves' rows); gate|up by 8 waves past their 8 steps ahead (d = 5120) and by 4
@pytest.mark.parametrize("act", [1, 3])
@pytest.mark.parametrize("dims", [(8, 2816, 704, 1, 8), (8, 2816, 1408, 1, 8), (8, 1056, 1408, 2, 8), (6, 1056, 800, 2, 3),
                                  (12, 544, 2112, 2, 16), (12, 1056, 1408, 1, 16), (12, 1056, 1408, 2, 13), (8, 5120, 160, 1, 8),
                                  (4, 2080, 1696, 3, 4), (5, 96, 3808, 2, 5)])
def test_single_assignments(ctx, pkg, orc, dims, act):
    E, d, nf, T, k = dims
    W = experts_of(E, d, nf)
    assert launches(pkg, W, T, k) == 2
    run(ctx, pkg, orc, W, T, k, act, skip=[(0, k - 1), (T - 1, k // 2)] if k > 3 else [])


@pytest.mark.parametrize("dims", [(32, 2080, 1408, 16, 4), (32, 2080, 1408, 50, 4), (32, 2080, 1408, 100, 4), (32, 2080, 1408, 130, 4),
                                  (14, 2080, 1408, 7, 4), (14, 2080, 1408, 25, 4), (14, 2080, 1408, 45, 4), (14, 2080, 1408, 60, 4),
                                  (12, 1056, 1408, 9, 16), (12, 1056, 1408, 60, 1)])
def test_lists(ctx, pkg, orc, dims):
    """Tiles of 16, 32, 64 and 128 places past the steps kept ahead, with weights read once (32 experts, 281 MB) and without."""
    E, d, nf, T, k = dims
    W = experts_of(E, d, nf)
    assert launches(pkg, W, T, k) > 2
    run(ctx, pkg, orc, W, T, k, 1 + 2 * (T & 1), types=(0, 30), skip=[(T // 2, 0)])


@pytest.mark.parametrize("dims", [(256, 64, 32, 3, 8), (256, 64, 32, 300, 8), (256, 128, 96, 70, 16), (250, 64, 64, 2000, 6)])
def test_every_expert(ctx, pkg, orc, dims):
    E, d, nf, T, k = dims
    W = experts_of(E, d, nf)
    rng = np.random.default_rng(T)
    xq, xd = ref.rows_of(rng, T, d)
    ids = ((np.arange(T * k) * 97 + 255) % E).reshape(T, k).astype(np.int32)  # the last expert first
    check_experts(ctx, pkg, orc, W, xq, xd, ids, rng.random((T, k)).astype(F32), 1, types=(0, 30))


@pytest.mark.parametrize("shape", [(1, 100, 8224), (16, 50, 6176), (20, 100, 8224), (32, 8200, 4160), (50, 100, 2816), (64, 8200, 2816),
                                   (77, 2816, 2112), (100, 100, 2816), (100, 8200, 2816), (128, 16416, 2816), (65, 16400, 1184),
                                   (129, 300, 8224), (161, 513, 2848), (700, 257, 4128)])
@pytest.mark.parametrize("type_", [0, 30])
def test_long_products(ctx, shape, type_):
    """Every token count's form, and the row tiles of 16, 32 and 64 by the outputs, past the steps kept ahead."""
    check_product(ctx, *shape, type_, seed=sum(shape))


@pytest.mark.parametrize("mode", [0, 1, 2, 3])
@pytest.mark.parametrize("type_", [0, 1, 30])
@pytest.mark.parametrize("shape", [(1030, 1056), (1027, 1408), (1024, 2048), (3, 14336), (2, 28672), (2, 65536)])
def test_rows(ctx, orc, shape, type_, mode):
    """Many rows of up to 2048 values (a wave each) and rows past 8192 (1024 threads, several steps)."""
    rows, n = shape
    print(f"quant_i8 rows {rows} n {n} type {type_} mode {mode}", flush=True)
    rng = np.random.default_rng(n + mode)
    rx, x = held((2 * rng.standard_normal((rows, n))).astype(F32), type_)
    ra, aux = held(rng.standard_normal((rows, n)).astype(F32), type_)
    if mode == 2:
        ra = aux = (1 + 0.2 * rng.standard_normal(n)).astype(F32)
    with Bufs(ctx) as B:
        qs, d = B.empty(rows * n), B.empty(rows * 4)
        ctx.quant_i8_device(mode, type_, B.of(rx).ptr, B.of(ra).ptr if mode else None, rows, n, n, EPS, qs.ptr, d.ptr)
        ctx.sync()
        got, gd = qs.download((rows, n), np.int8), d.download(rows)
    rq, rd = ref.quant(transformed(orc, mode, x, aux))
    np.testing.assert_array_equal(gd.view(np.uint32), rd.view(np.uint32))
    np.testing.assert_array_equal(got, rq)
