"""Products with fp16 and bf16 matrices in runs of ragged length and the experts over them (phx_weight_upload_half,
phx_matmul_grouped, phx_experts_half) against plain implementations in 64 bits (tests/half_ref.py): odd sizes, each type, empty
groups, places without a row, infinities that must not spread, the refusals, and the whole run from a router's logits."""
import numpy as np
import pytest

import half_ref as ref
from test_gpu_i8 import Bufs

pytestmark = pytest.mark.gpu

F32 = np.float32


def spread(rng, n, E, empty):
    """Offsets of E groups over n places, some empty, not all places used."""
    at = np.sort(rng.integers(0, n + 1, E + 1))
    if empty:
        at[1:-1:3] = at[0:-2:3][:len(at[1:-1:3])]
    return at.astype(np.int32)


def check(ctx, type_, y_type, E, n, rows, cols, act=0, gather=None, offsets=None, seed=0, alter=None):
    """One call against the definition; rows of y outside the groups, and bytes behind y, stay as they were."""
    print(f"grouped type {type_} y {y_type} E {E} n {n} {rows} x {cols} act {act} gather {gather}", flush=True)
    rng = np.random.default_rng(seed + E + 7 * n + rows + cols)
    n_x = n if gather is None else gather
    raw_x, x = ref.held(rng.standard_normal((n_x, cols)), type_)
    raw_w, w = ref.held(rng.standard_normal((E, rows, cols)) / np.sqrt(cols), type_)
    src = np.arange(n) if gather is None else rng.integers(-2, n_x + 2, n)
    if offsets is None:
        offsets = spread(rng, n, E, empty=E > 3)
    if alter is not None:
        alter(raw_x, x, raw_w, w)
    out = rows if act == 0 else rows // 2
    item = 4 if y_type == 0 else 2
    before = rng.integers(0, 120, n * out * item + 64).astype(np.uint8)
    h = ctx.weight_upload_half(type_, E, rows, cols, raw_w, paired=act != 0)
    try:
        with Bufs(ctx) as B:
            y = B.of(before)
            ctx.matmul_grouped_device(h, act, n, B.of(offsets).ptr, B.of(raw_x).ptr, n_x,
                                      None if gather is None else B.of(src.astype(np.int32)).ptr, y_type, y.ptr)
            ctx.sync()
            got, raw = ref.read(y, (n, out), y_type), y.download(before.shape, np.uint8)
    finally:
        ctx.weight_free(h)
    assert (raw[n * out * item:] == before[n * out * item:]).all()
    at = np.maximum.accumulate(np.clip(offsets, 0, n))
    stored = np.zeros(n, bool)
    for e in range(E):
        p = np.arange(at[e], max(at[e], at[e + 1]))
        p = p[(src[p] >= 0) & (src[p] < n_x)]
        stored[p] = True
        if len(p):
            v = x[src[p]]
            with np.errstate(invalid="ignore", over="ignore"):
                want, bound = ref.product(v, w[e]) if act == 0 else ref.gated(act, v, w[e])
                bound = ref.rounded(want, bound, y_type)
                off = np.abs(got[p] - want)
            fine = np.isfinite(want)
            assert (off[fine] <= bound[fine]).all(), (off[fine] / bound[fine]).max()
            np.testing.assert_array_equal(got[p][~fine], want[~fine])
    left = raw[:n * out * item].reshape(n, -1)[~stored]
    np.testing.assert_array_equal(left, before[:n * out * item].reshape(n, -1)[~stored])
    return got


SIZES = [(1, 1, 1, 8), (1, 3, 33, 24), (2, 5, 64, 64), (7, 20, 50, 40), (5, 60, 100, 72), (16, 40, 130, 200), (3, 90, 64, 520),
         (1, 129, 96, 1024), (4, 300, 260, 264), (2, 700, 513, 96), (256, 300, 34, 64), (3, 1500, 40, 32)]


@pytest.mark.parametrize("type_,y_type", [(1, 0), (1, 1), (30, 0), (30, 30), (30, 1)])
@pytest.mark.parametrize("size", SIZES)
def test_plain(ctx, size, type_, y_type):
    E, n, rows, cols = size
    check(ctx, type_, y_type, E, n, rows, cols)


@pytest.mark.parametrize("act", [1, 3])
@pytest.mark.parametrize("type_,y_type", [(1, 1), (30, 30), (30, 0)])
@pytest.mark.parametrize("size", [(1, 1, 2, 8), (3, 20, 66, 40), (7, 50, 128, 72), (16, 100, 40, 520), (4, 300, 130, 264), (2, 700, 258, 96),
                                  (1, 200, 1408, 128)])
def test_paired_and_gathered(ctx, size, type_, y_type, act):
    E, n, rows, cols = size
    check(ctx, type_, y_type, E, n, rows, cols, act=act, gather=max(1, n // 3))


@pytest.mark.parametrize("n", [1, 2, 17, 130, 600])
def test_plain_gathered(ctx, n):
    check(ctx, 30, 30, 6, n, 70, 136, gather=9)


def test_longest_rows(ctx):
    check(ctx, 30, 0, 2, 9, 20, 65536)
    check(ctx, 1, 0, 1, 300, 20, 65536)


@pytest.mark.parametrize("n,E", [(5, 3), (200, 3), (900, 2)])
def test_offsets_outside(ctx, n, E):
    """Values outside 0 .. n count as the nearest of these; groups may all be empty; the first may begin late."""
    check(ctx, 30, 30, E, n, 48, 64, offsets=np.array([-7] + [n // 2] * (E - 1) + [n + 1000], np.int32))
    check(ctx, 30, 30, E, n, 48, 64, offsets=np.full(E + 1, n // 2, np.int32))
    check(ctx, 30, 30, E, n, 48, 64, offsets=np.full(E + 1, 2 ** 31 - 1, np.int32))
    check(ctx, 30, 30, E, n, 48, 64, offsets=np.array([n - 1] * E + [n], np.int32))


@pytest.mark.parametrize("n,E", [(60, 5), (400, 200), (900, 3), (3000, 256)])
def test_offsets_that_fall(ctx, n, E):
    """A value below the one before it counts as that one: no place has two groups."""
    check(ctx, 1, 1, E, n, 48, 64, offsets=np.random.default_rng(n).integers(-20, n + 20, E + 1).astype(np.int32))
    check(ctx, 30, 30, E, n, 48, 64, offsets=np.linspace(n, 0, E + 1).astype(np.int32))


# long reductions and odd ones, more and fewer tiles than compute units
@pytest.mark.parametrize("E,n,rows,cols", [(1, 200, 64, 8192), (1, 1000, 300, 4096), (2, 700, 2000, 2048), (9, 2500, 1030, 1536), (3, 97, 700, 16384),
                                           (40, 6000, 520, 1024), (5, 2100, 4096, 1608), (1, 3000, 2816, 2056)])
def test_reductions(ctx, E, n, rows, cols):
    check(ctx, 30, 30, E, n, rows, cols)
    check(ctx, 1, 0, E, n, rows // 2 * 2, cols, act=1, gather=n // 2)


@pytest.mark.parametrize("places", range(30, 290, 20))
def test_tile_widths(ctx, places):
    check(ctx, 30, 0, 2, 2 * places + 5, 600, 1032, offsets=np.array([2, 2 + places, 2 * places + 3], np.int32))


@pytest.mark.parametrize("n", [9, 40, 300])
@pytest.mark.parametrize("cols", [40, 64, 72])
def test_infinities_stay_in_their_row(ctx, n, cols):
    """Rows with an infinity or a NaN, a matrix row with one, and the padding of an odd length."""
    def alter(raw_x, x, raw_w, w):
        for row, v in ((0, np.inf), (n // 2, -np.inf), (n - 1, np.nan)):
            raw_x[row, cols - 1] = x[row, cols - 1] = v
        raw_w[0, 3, 0] = w[0, 3, 0] = -np.inf
    check(ctx, 1, 0, 2, n, 40, cols, alter=alter, offsets=np.array([0, n // 3, n], np.int32))


@pytest.mark.parametrize("act", [1, 3])
def test_activations_far_out(ctx, act):
    """Gates from far below to far above."""
    g = np.array([-6e4, -300, -200, -100, -89, -60, -20, -5, -1, -1e-3, -0.0, 0, 1e-4, 0.5, 1, 5, 20, 88, 300, 6e4], np.float16)
    w = np.zeros((1, 2, 8), np.float16)
    w[0, 0, 0] = w[0, 1, 1] = 1
    x = np.zeros((len(g), 8), np.float16)
    x[:, 0], x[:, 1] = g, 2
    h = ctx.weight_upload_half(1, 1, 2, 8, w, paired=True)
    try:
        got = ctx.MatMulGrouped(h, act, np.array([0, len(g)]), x)[:, 0]
    finally:
        ctx.weight_free(h)
    g = g.astype(np.float64)
    want = 2 * ref.act(act, g)
    tail = np.where(g < 0, np.minimum(np.abs(g) * (1 if act == 1 else 2 + g * g), 88), 1)
    assert (np.abs(got - want) <= (16 + 4 * tail) * 2.0 ** -24 * np.abs(want) + 1e-35).all()


@pytest.mark.parametrize("act", [1, 3])
def test_infinite_gates(ctx, act):
    """Gates that overflow to either infinity, beside a finite up; and a NaN."""
    big, small = ref.held(np.array([3e38, 1e-38]), 30)[0]
    w = np.zeros((1, 4, 8), np.uint16)
    w[0, :, 0] = big, big ^ 0x8000, small, small  # gate rows, up rows
    x = np.zeros((2, 8), np.uint16)
    x[0, 0], x[1] = big, 0x7FC0
    h = ctx.weight_upload_half(30, 1, 4, 8, w, paired=True)
    try:
        got = ctx.MatMulGrouped(h, act, np.array([0, 2]), x)
    finally:
        ctx.weight_free(h)
    assert got[0, 0] == np.inf and got[0, 1] == 0 and np.isnan(got[1]).all()


def test_fp16_subnormals(ctx):
    w = np.full((1, 4, 16), 2.0 ** -20, np.float16)
    x = np.full((3, 16), 2.0 ** -22, np.float16)
    x[1] = 1
    h = ctx.weight_upload_half(1, 1, 4, 16, w)
    try:
        got = ctx.MatMulGrouped(h, 0, np.array([0, 3]), x)
    finally:
        ctx.weight_free(h)
    np.testing.assert_array_equal(got, x.astype(F32) @ w[0].astype(F32).T)


def test_upload_from_device_and_unaligned(ctx):
    rng = np.random.default_rng(4)
    w = rng.standard_normal((3, 40, 24)).astype(np.float16)
    x = rng.standard_normal((30, 24)).astype(np.float16)
    at = np.array([0, 10, 11, 30])
    with Bufs(ctx) as B:
        odd = np.zeros(w.size + 1, np.float16)
        odd[1:] = w.ravel()
        hs = [ctx.weight_upload_half(1, 3, 40, 24, w), ctx.weight_upload_half(1, 3, 40, 24, B.of(w).ptr),
              ctx.weight_upload_half(1, 3, 40, 24, B.of(odd).ptr + 2)]
    got = [ctx.MatMulGrouped(h, 0, at, x) for h in hs]
    assert ctx.weight_shape(hs[0]) == (3, 40, 24)
    for h in hs:
        ctx.weight_free(h)
    np.testing.assert_array_equal(got[0], got[1])
    np.testing.assert_array_equal(got[0], got[2])


@pytest.mark.parametrize("n,paired", [(9, False), (16, True), (17, False), (70, False), (72, True), (73, False)])
def test_weights_past_the_caches(ctx, n, paired):
    """Matrices of more than 128 MB, few places a group: the row kernel's loads that pass the caches by, and the sizes beside them."""
    def alter(raw_x, x, raw_w, w):  # the same values from matrix to matrix, in other places
        for e in range(1, len(w)):
            raw_w[e], w[e] = np.roll(raw_w[0], e, 1), np.roll(w[0], e, 1)
    check(ctx, 30, 0, 9, n, 4096, 1800, act=1 if paired else 0, alter=alter)


@pytest.mark.parametrize("type_,paired", [(1, True), (30, False)])
@pytest.mark.parametrize("lengths", [(1, 32, 33, 64, 65, 96, 97, 128, 129), (0, 300, 5, 0, 128, 90, 257, 0, 31)])
def test_only_tiles_past_the_caches(ctx, lengths, type_, paired):
    """Matrices of more than 128 MB on the tile kernel: groups of one tile, whose weights pass the caches by, of each width, beside
    groups of several."""
    def alter(raw_x, x, raw_w, w):
        for e in range(1, len(w)):
            raw_w[e], w[e] = np.roll(raw_w[0], e, 1), np.roll(w[0], e, 1)
    offsets = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
    check(ctx, type_, 0, 9, int(offsets[-1]) + 3, 4096, 1800, act=3 if paired else 0, offsets=offsets, alter=alter)


def test_same_call_same_bits(ctx):
    """A call's result does not depend on timing, nor on the calls beside it."""
    rng = np.random.default_rng(5)
    w = rng.standard_normal((4, 200, 1024)).astype(np.float16)
    h = ctx.weight_upload_half(1, 4, 200, 1024, w)
    try:
        for n in (7, 100, 900):
            x = rng.standard_normal((n, 1024)).astype(np.float16)
            at = np.linspace(0, n, 5).astype(np.int32)
            first = ctx.MatMulGrouped(h, 0, at, x)
            for _ in range(3):
                np.testing.assert_array_equal(ctx.MatMulGrouped(h, 0, at, x), first)
    finally:
        ctx.weight_free(h)


# ---------------------------------------------------------------------------------------- experts
def expert_weights(rng, E, d, nf, type_):
    raw_g, wg = ref.held(rng.standard_normal((E, 2 * nf, d)) / np.sqrt(d), type_)
    raw_d, wd = ref.held(rng.standard_normal((E, d, nf)) / np.sqrt(nf), type_)
    return (raw_g, raw_d), (wg, wd)


def upload(ctx, type_, raw, E, d, nf):
    return ctx.weight_upload_half(type_, E, 2 * nf, d, raw[0], paired=True), ctx.weight_upload_half(type_, E, d, nf, raw[1])


def check_experts(ctx, type_, out_type, act, T, k, E, d, nf, seed=0, spoil=None):
    print(f"experts_half type {type_} out {out_type} act {act} T {T} k {k} E {E} d {d} nf {nf}", flush=True)
    rng = np.random.default_rng(seed + T + E + d + nf)
    raw, (wg, wd) = expert_weights(rng, E, d, nf, type_)
    raw_x, x = ref.held(rng.standard_normal((T, d)), type_)
    ids = rng.integers(0, E, (T, k)).astype(np.int32)
    if spoil:
        spoil(rng, ids)
    weights = rng.random((T, k)).astype(F32)
    hs = upload(ctx, type_, raw, E, d, nf)
    item = 4 if out_type == 0 else 2
    try:
        with Bufs(ctx) as B:
            pad = np.full(T * d * item + 64, 0x5A, np.uint8)
            out = B.of(pad)
            ctx.experts_half_device(*hs, act, T, k, B.of(raw_x).ptr, B.of(ids).ptr, B.of(weights).ptr, out_type, out.ptr)
            ctx.sync()
            got = ref.read(out, (T, d), out_type)
            assert (out.download(pad.shape, np.uint8)[T * d * item:] == 0x5A).all()
    finally:
        for h in hs:
            ctx.weight_free(h)
    want, bound = ref.experts(x, ids, weights, wg, wd, act, type_)
    bound = ref.rounded(want, bound, out_type)
    assert (np.abs(got - want) <= bound).all(), (np.abs(got - want) / bound).max()
    return got


@pytest.mark.parametrize("type_,out_type,act", [(1, 1, 1), (1, 0, 3), (30, 30, 1), (30, 0, 3)])
@pytest.mark.parametrize("size", [(1, 1, 1, 8, 8), (1, 8, 16, 72, 40), (3, 2, 4, 64, 32), (5, 4, 40, 96, 104), (40, 2, 4, 64, 72), (64, 8, 16, 136, 64),
                                  (300, 4, 5, 72, 40), (700, 2, 3, 64, 264), (33, 16, 256, 16, 8)])
def test_experts(ctx, size, type_, out_type, act):
    T, k, E, d, nf = size
    check_experts(ctx, type_, out_type, act, T, k, E, d, nf)


@pytest.mark.parametrize("T", [2, 50, 400])
def test_experts_skipped_and_repeated(ctx, T):
    def spoil(rng, ids):
        ids[rng.random(ids.shape) < 0.3] = -1
        ids[rng.random(ids.shape) < 0.1] = 6  # past the last
        ids[0] = -1
        ids[1] = 3
    got = check_experts(ctx, 30, 30, 1, T, 4, 6, 64, 40, spoil=spoil)
    assert (got[0] == 0).all()


def test_experts_all_rows_one_expert(ctx):
    check_experts(ctx, 1, 1, 3, 500, 2, 7, 64, 72, spoil=lambda rng, ids: ids.fill(5))


def test_experts_long_batch(ctx):
    """More assignments than one chunk of the workspace takes."""
    check_experts(ctx, 30, 30, 1, 9001, 8, 4, 16, 8)


def test_experts_in_bf16_match_the_run_by_hand(ctx, pkg):
    """A routing's experts by the grouped product, from the lists that the ids give, and by the one call."""
    rng = np.random.default_rng(8)
    E, d, nf, T, k = 12, 128, 64, 90, 3
    raw, (wg, wd) = expert_weights(rng, E, d, nf, 30)
    raw_x, x = ref.held(rng.standard_normal((T, d)), 30)
    logits = rng.standard_normal((T, E)).astype(F32)
    ids, weights = ctx.Route(pkg.RouteDesc(E, k), logits)
    hs = upload(ctx, 30, raw, E, d, nf)
    try:
        out = ctx.ExpertsHalf(*hs, 1, raw_x, ids, weights)
        order = np.argsort(ids.ravel(), kind="stable")
        at = np.searchsorted(ids.ravel()[order], np.arange(E + 1)).astype(np.int32)
        h = ctx.MatMulGrouped(hs[0], 1, at, raw_x, src=order // k)
        y = np.empty((T * k, d), F32)
        y[order] = ctx.MatMulGrouped(hs[1], 0, at, ref.held(h, 30)[0])
    finally:
        for h in hs:
            ctx.weight_free(h)
    by_hand = (y.reshape(T, k, d) * weights[:, :, None]).sum(1, dtype=np.float64)
    want, bound = ref.experts(x, ids, weights, wg, wd, 1, 30)
    assert (np.abs(out - want) <= ref.rounded(want, bound, 0)).all()
    assert (np.abs(by_hand - want) <= ref.rounded(want, bound, 0)).all()


# ---------------------------------------------------------------------------------------- refusals
def test_refusals(ctx, pkg):
    A, N = pkg.ArgumentError, pkg.NotSupportedError
    P = pkg.PHX
    w = np.zeros((2, 64, 64), np.float16)
    plain, paired = ctx.weight_upload_half(1, 2, 64, 64, w), ctx.weight_upload_half(1, 2, 64, 64, w, paired=True)
    down = ctx.weight_upload_half(1, 2, 64, 32, w[:, :, :32])
    bdown = ctx.weight_upload_half(30, 2, 64, 32, w[:, :, :32].view(np.uint16))
    int8 = ctx.weight_upload_i8(1, 64, 64, np.zeros((64, 64), np.int8), np.ones(64, F32))
    try:
        with Bufs(ctx) as B:
            off, x, y, src = B.of(np.zeros(3, np.int32)).ptr, B.empty(4096).ptr, B.empty(4096).ptr, B.of(np.zeros(8, np.int32)).ptr
            host = np.zeros(4096, np.uint8).ctypes.data

            def call(h=plain, act=0, n=4, off=off, x=x, n_x=4, src=None, y_type=0, y=y):
                ctx.matmul_grouped_device(h, act, n, off, x, n_x, src, y_type, y)
            call()
            for bad in (dict(h=None), dict(n=0), dict(n=P.MAX_ROWS_I8 + 1, n_x=P.MAX_ROWS_I8 + 1), dict(n_x=3), dict(n_x=0, src=src), dict(off=None),
                        dict(x=None), dict(y=None), dict(x=x + 2), dict(y=y + 4), dict(off=off + 1), dict(src=src + 2), dict(act=2), dict(act=7),
                        dict(x=host), dict(y=host), dict(off=host), dict(src=host), dict(y=x), dict(y=x + 16), dict(src=y)):
                with pytest.raises(A):
                    call(**bad)
            for bad in (dict(y_type=2), dict(y_type=8), dict(act=1), dict(h=paired), dict(h=int8)):
                with pytest.raises(N):
                    call(**bad)
            wide = ctx.weight_upload_half(1, 1, 1, 4096, np.zeros(4096, np.float16))
            with pytest.raises(A, match="2\\^32"):
                call(h=wide, n_x=1 << 19, src=src)
            ctx.weight_free(wide)

            def ffn(gu=paired, dn=down, act=1, T=2, k=2, x=x, ids=off, weights=src, out_type=0, out=y):
                ctx.experts_half_device(gu, dn, act, T, k, x, ids, weights, out_type, out)
            for bad in (dict(gu=None), dict(dn=None), dict(act=0), dict(act=2), dict(T=0), dict(k=0), dict(k=P.MAX_USED + 1), dict(T=P.MAX_ROWS_I8 + 1),
                        dict(x=None), dict(ids=None), dict(weights=None), dict(out=None), dict(x=host), dict(out=x), dict(out=y + 8)):
                with pytest.raises(A):
                    ffn(**bad)
            for bad in (dict(gu=plain), dict(dn=paired), dict(dn=bdown), dict(dn=int8), dict(out_type=2)):
                with pytest.raises(N):
                    ffn(**bad)
            with pytest.raises(A):
                ffn(dn=plain)  # sizes that do not fit
            for other in (ctx.matmul_device, ctx.matmul_k_device):
                with pytest.raises(N):
                    other(plain, 1, x, x, y)
            with pytest.raises(N):
                ctx.matmul_i8_device(plain, 1, x, x, 0, y)
            ctx.sync()
    finally:
        for h in (plain, paired, down, bdown, int8):
            ctx.weight_free(h)


def test_upload_refusals(ctx, pkg):
    at = np.zeros(64, np.float16).ctypes.data
    P = pkg.PHX
    for type_, n_mat, rows, cols, paired in ((1, 0, 8, 8, 0), (1, 257, 8, 8, 0), (1, 1, 0, 8, 0), (1, 1, 8, 4, 0), (1, 1, 8, 0, 0), (1, 1, 7, 8, 1),
                                             (1, 1, P.MAX_ROWS_I8 + 1, 8, 0), (1, 1, 8, P.MAX_COLS_I8 + 8, 0), (30, 1, 1 << 18, 1 << 16, 0)):
        with pytest.raises(pkg.ArgumentError):
            ctx.weight_upload_half(type_, n_mat, rows, cols, at, paired=bool(paired))
    for type_ in (0, 2, 24):
        with pytest.raises(pkg.NotSupportedError):
            ctx.weight_upload_half(type_, 1, 8, 8, at)
    for bad in (None, at + 1):
        with pytest.raises(pkg.ArgumentError):
            ctx.weight_upload_half(1, 1, 8, 8, bad)
    with pytest.raises(pkg.ArgumentError):
        ctx.weight_upload_half(30, 1, 8, 8, np.zeros((8, 8), np.float16))
    with pytest.raises(pkg.ArgumentError):
        ctx.weight_upload_half(1, 1, 8, 8, np.zeros((8, 7), np.float16))


def test_host_forms_refuse_sizes_that_are_not_the_handles(ctx, pkg):
    h = ctx.weight_upload_half(1, 2, 16, 8, np.zeros((2, 16, 8), np.float16))
    try:
        for at, x in (([0, 1], np.zeros((2, 8), np.float16)), ([0, 1, 2], np.zeros((2, 16), np.float16)), ([0, 1, 2], np.zeros((2, 8), F32)),
                      ([0, 1, 2.5], np.zeros((2, 8), np.float16))):
            with pytest.raises(pkg.ArgumentError):
                ctx.MatMulGrouped(h, 0, np.array(at), x)
    finally:
        ctx.weight_free(h)


def test_host_forms_refuse_rows_of_another_type(ctx, pkg):
    for type_, other in ((1, np.uint16), (30, np.float16)):
        w = np.zeros((1, 16, 8), np.float16 if type_ == 1 else np.uint16)
        h, d = ctx.weight_upload_half(type_, 1, 16, 8, w, paired=True), ctx.weight_upload_half(type_, 1, 8, 8, w[:, :8])
        try:
            for x in (np.zeros((2, 8), other), np.zeros((2, 8), np.int16)):
                with pytest.raises(pkg.ArgumentError):
                    ctx.MatMulGrouped(h, 1, np.array([0, 2]), x)
                with pytest.raises(pkg.ArgumentError):
                    ctx.ExpertsHalf(h, d, 1, x, np.zeros((2, 1), np.int32), np.ones((2, 1), F32))
            x = np.zeros((2, 8), w.dtype)
            assert (ctx.MatMulGrouped(h, 1, np.array([0, 2]), x) == 0).all()
            assert (ctx.ExpertsHalf(h, d, 1, x, np.zeros((2, 1), np.int32), np.ones((2, 1), F32)) == 0).all()
        finally:
            ctx.weight_free(h)
            ctx.weight_free(d)


def test_experts_past_the_caches(ctx):
    """One token's experts, and a decode step's, of matrices of more than 128 MB."""
    for T in (1, 12):
        check_experts(ctx, 30, 0, 1, T, 4, 20, 1024, 1704)


@pytest.mark.parametrize("n,what", enumerate(("the weight", "offsets", "x", "y", "src"), 1))
def test_memory_of_another_gpu(pkg, monkeypatch, n, what):
    monkeypatch.setenv("PHX_FAULT", f"device:{n}")
    with pkg.MoeContext(0) as c:
        h = c.weight_upload_half(1, 1, 8, 8, np.ones((8, 8), np.float16))  # host memory: nothing to check
        run = lambda: c.MatMulGrouped(h, 0, np.array([0, 2]), np.ones((2, 8), np.float16), src=np.array([0, 1]))  # noqa: E731
        with pytest.raises(pkg.ArgumentError, match=f"{what} is memory of device"):
            run()
        assert (run() == 8).all()
        c.weight_free(h)


@pytest.mark.parametrize("n,what", enumerate(("gate_up", "down", "x", "ids", "weights", "out"), 1))
def test_experts_memory_of_another_gpu(pkg, monkeypatch, n, what):
    monkeypatch.setenv("PHX_FAULT", f"device:{n}")
    with pkg.MoeContext(0) as c:
        hs = (c.weight_upload_half(1, 1, 16, 8, np.ones((16, 8), np.float16), paired=True),
              c.weight_upload_half(1, 1, 8, 8, np.ones((8, 8), np.float16)))
        run = lambda: c.ExpertsHalf(*hs, 1, np.ones((2, 8), np.float16), np.full((2, 1), -1), np.ones((2, 1), F32))  # noqa: E731
        with pytest.raises(pkg.ArgumentError, match=f"{what} is memory of device"):
            run()
        assert (run() == 0).all()
        for h in hs:
            c.weight_free(h)


def test_allocation_and_launch_faults(pkg, monkeypatch):
    """A failed allocation or launch inside the calls: an error, and the same call then gives the right result."""
    E, d, nf, k, T = 4, 64, 32, 2, 40
    rng = np.random.default_rng(3)
    raw, (wg, wd) = expert_weights(rng, E, d, nf, 1)
    raw_x, x = ref.held(rng.standard_normal((T, d)), 1)
    ids = rng.integers(0, E, (T, k)).astype(np.int32)
    weights = rng.random((T, k)).astype(F32)
    want, bound = ref.experts(x, ids, weights, wg, wd, 1, 1)
    seen = set()
    for spec in [f"malloc:{n}" for n in range(4, 22)] + [f"launch:{n}" for n in range(1, 13, 2)]:
        print("fault", spec, flush=True)
        monkeypatch.setenv("PHX_FAULT", spec)
        try:
            c = pkg.MoeContext(0)
        except pkg.OutOfDeviceMemoryError:
            continue
        finally:
            monkeypatch.delenv("PHX_FAULT")
        with c:
            for attempt in range(2):
                try:
                    hs = upload(c, 1, raw, E, d, nf)
                    out = c.ExpertsHalf(*hs, 1, raw_x, ids, weights)
                    break
                except (pkg.OutOfDeviceMemoryError, pkg.GpuDeviceLostError) as e:
                    seen.add(type(e).__name__)
                    assert attempt == 0
            assert (np.abs(out - want) <= ref.rounded(want, bound, 0)).all()
    assert seen == {"OutOfDeviceMemoryError", "GpuDeviceLostError"}
