"""The tile kernel of the products with fp16 and bf16 matrices, each call of which the library's own rule is asked for: all widths of
both its sizes, each type, plain, paired and with rows in two terms; infinities, offsets out of order and the scatter to the assignments' own
places, where other tests' shapes go to the row kernel."""
import numpy as np
import pytest

import half_ref as ref
import half_rules as rules
from test_gpu_experts_terms import call as experts_call
from test_gpu_experts_terms import experts
from test_gpu_half import check, expert_weights, spread, upload

pytestmark = pytest.mark.gpu

NARROW = [1, 31, 32, 33, 63, 64, 65, 95, 96, 97, 127, 128, 129, 160, 0, 193, 257, 300]  # widths 1 to 4, single tiles and several
WIDE = [20, 32, 50, 90, 120, 150, 180, 220, 256, 513, 700, 257]  # widths 1 to 8


def bounds(lengths, first=2):
    return (first + np.concatenate([[0], np.cumsum(lengths)])).astype(np.int32)


def strange(type_, rows_of_x, row_of_w):
    """An infinity or a NaN in the first and the last column of some rows of x, one in a row of the last matrix."""
    inf, minus, nan = (np.inf, -np.inf, np.nan) if type_ == 1 else (0x7F80, 0xFF80, 0x7FC0)

    def alter(raw_x, x, raw_w, w):
        for i, row in enumerate(rows_of_x):
            col = (0, -1)[i % 2]
            k = i // 2 % 3
            raw_x[row, col], x[row, col] = (inf, minus, nan)[k], (np.inf, -np.inf, np.nan)[k]
        raw_w[-1, row_of_w, 0], w[-1, row_of_w, 0] = minus, -np.inf
    return alter


@pytest.mark.parametrize("type_,y_type", [(1, 1), (1, 0), (30, 30), (30, 0)])
@pytest.mark.parametrize("rows,cols,act", [(3080, 72, 0), (2304, 200, 0), (2304, 72, 1), (2570, 1032, 3)])
def test_narrow_widths(ctx, type_, y_type, rows, cols, act):
    offsets = bounds(NARROW)
    n = int(offsets[-1]) + 5
    assert rules.capacity(n, len(NARROW), rows, act != 0) == 128
    check(ctx, type_, y_type, len(NARROW), n, rows, cols, act=act, offsets=offsets)


@pytest.mark.parametrize("type_", [1, 30])
@pytest.mark.parametrize("act,cols,gather", [(0, 72, None), (0, 128, 900), (1, 72, None), (3, 136, 900)])
def test_wide_widths(ctx, type_, act, cols, gather):
    rows = 14400
    offsets = bounds(WIDE)
    n = int(offsets[-1]) + 5
    assert rules.capacity(n, len(WIDE), rows, act != 0) == 256
    check(ctx, type_, type_, len(WIDE), n, rows, cols, act=act, gather=gather, offsets=offsets)


@pytest.mark.parametrize("type_", [1, 30])
@pytest.mark.parametrize("rows,cols,act,lengths", [(2304, 72, 0, NARROW), (2304, 72, 1, NARROW), (2304, 40, 0, NARROW), (14400, 72, 0, WIDE), (14400, 104, 1, WIDE)])
def test_infinities_stay_in_their_row(ctx, type_, rows, cols, act, lengths):
    """Where the last step's columns end past the row, and what the loads bring in their place is the row's first."""
    offsets = bounds(lengths)
    n = int(offsets[-1]) + 5
    assert rules.capacity(n, len(lengths), rows, act != 0) >= 128
    at = np.unique(np.concatenate([offsets[:-1], offsets[1:] - 1, [n // 2, n - 7]]))
    check(ctx, type_, 0, len(lengths), n, rows, cols, act=act, offsets=offsets, alter=strange(type_, at[(at >= 0) & (at < n)], 3 if act == 0 else rows // 2 + 3))


@pytest.mark.parametrize("rows,n,E,cap", [(2304, 1500, 18, 128), (14400, 2600, 12, 256)])
def test_offsets_out_of_order(ctx, rows, n, E, cap):
    """Outside 0 .. n, falling, all the same: no place of two groups, and no place outside the call's."""
    assert rules.capacity(n, E, rows) == cap
    rng = np.random.default_rng(n)
    cases = [[-7] + [n // 2] * (E - 1) + [n + 1000], rng.integers(-20, n + 20, E + 1), [0] + [2 ** 31 - 1] * E]
    if cap == 128:
        cases += [np.linspace(n, 0, E + 1).astype(int), [n - 1] * E + [n], np.full(E + 1, 2 ** 31 - 1), np.full(E + 1, -2 ** 31)]
    for offsets in cases:
        check(ctx, 30, 30, E, n, rows, 72, offsets=np.array(offsets, np.int32))
    check(ctx, 1, 0, E, n, rows, 72, act=1, gather=n // 2, offsets=np.sort(rng.integers(-20, n + 20, E + 1)).astype(np.int32))


@pytest.mark.parametrize("type_,paired", [(1, False), (30, True)])
def test_gathered_rows_far_apart(ctx, type_, paired):
    """src naming the first and the last of many rows, the same row often, and rows that are not there."""
    offsets = bounds(NARROW)
    n = int(offsets[-1]) + 5
    assert rules.capacity(n, len(NARROW), 2304, paired) == 128
    check(ctx, type_, 0, len(NARROW), n, 2304, 72, act=3 if paired else 0, gather=1, offsets=offsets)
    check(ctx, type_, 0, len(NARROW), n, 2304, 72, act=3 if paired else 0, gather=20000, offsets=offsets)


# the down product's rows to their assignments' own places; several chunks of it; one expert, none, all assignments skipped
@pytest.mark.parametrize("type_", [1, 30])
@pytest.mark.parametrize("T,k,E,d,nf,spoil", [(900, 4, 8, 1032, 72, None), (9001, 8, 4, 264, 8, None), (900, 4, 8, 1032, 136, "one"), (900, 4, 8, 1032, 72, "most"),
                                              (900, 4, 8, 1032, 72, "all"), (1100, 3, 16, 1032, 64, "even")])
def test_scatter_of_the_down_product(ctx, type_, T, k, E, d, nf, spoil):
    chunk = min(T, 65535 // k) * k
    assert rules.capacity(chunk, E, d, x_terms=2) == 96
    rng = np.random.default_rng(T + d + nf)
    raw, (wg, wd) = expert_weights(rng, E, d, nf, type_)
    raw_x, x = ref.held(rng.standard_normal((T, d)), type_)
    ids = rng.integers(0, E, (T, k)).astype(np.int32)
    if spoil == "one":
        ids[:] = E - 2
    elif spoil == "most":
        ids[rng.random((T, k)) < 0.9] = -1
        ids[rng.random((T, k)) < 0.02] = 2 ** 31 - 1
    elif spoil == "all":
        ids[:] = E
    elif spoil == "even":
        ids[:] = np.arange(T * k).reshape(T, k) % E
    weights = rng.standard_normal((T, k)).astype(np.float32)
    hs = upload(ctx, type_, raw, E, d, nf)
    try:
        got = experts_call(ctx, hs, 1, raw_x, ids, weights, type_, d)
    finally:
        for h in hs:
            ctx.weight_free(h)
    want, bound = experts(x, ids, weights, wg, wd, 1, type_)
    assert (np.abs(got - want) <= ref.rounded(want, bound, type_)).all()


def test_one_matrix_of_few_rows_and_many_places(ctx):
    """Up to 32 rows go to the row kernel whatever the places: more tiles than it has elsewhere."""
    for rows, n in ((32, 70001), (2, 1 << 20)):
        assert rules.capacity(n, 1, rows) == 32
        check(ctx, 30, 30, 1, n, rows, 8, offsets=np.array([0, n], np.int32))
    check(ctx, 1, 0, 200, 100000, 20, 16, offsets=spread(np.random.default_rng(3), 100000, 200, True))
