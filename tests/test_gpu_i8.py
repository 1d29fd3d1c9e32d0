"""int8 rows, products and experts (phx_quant_i8, phx_weight_upload_i8, phx_matmul_i8, phx_experts_i8) against plain
implementations in 64 bits (tests/i8_ref.py): quants and scales equal, products within their stated roundings, at odd
sizes, every type and mode, empty rows and skipped places, and the whole run from a router's logits."""
import functools

import numpy as np
import pytest

import i8_ref as ref

pytestmark = pytest.mark.gpu

F32 = np.float32
STEP = {0: 2.0 ** -24, 1: 2.0 ** -11, 30: 2.0 ** -8}  # half a step, relative: float32, fp16, bf16
EPS = 1e-6


def act_of(pkg, orc, act):
    return orc.silu if act == pkg.PHX.QUANT_SILU_MUL else orc.gelu


def read(buf, shape, type_):
    """A buffer's rows as float64."""
    if type_ == 30:
        return ref.bf16_value(buf.download(shape, np.uint16)).astype(np.float64)
    return buf.download(shape, F32 if type_ == 0 else np.float16).astype(np.float64)


def held(v, type_):
    """float32 values in a call's type, and the values they then have."""
    if type_ == 1:
        h = v.astype(np.float16)
        return h, h.astype(F32)
    if type_ == 30:
        h = ref.bf16_bits(v)
        return h, ref.bf16_value(h)
    return v, v


class Bufs:
    """Device buffers of a test, freed at its end."""

    def __init__(self, ctx):
        self.ctx, self.all = ctx, []

    def __enter__(self):
        return self

    def __exit__(self, *a):
        self.ctx.sync()
        for b in self.all:
            b.free()

    def of(self, arr):
        b = self.empty(arr.nbytes)
        b.upload(arr)
        return b

    def empty(self, n):
        self.all.append(self.ctx.alloc(max(n, 16)))
        return self.all[-1]


# ---------------------------------------------------------------------------------------- rows
def transformed(orc, mode, x, aux):
    if mode == 0:
        return x
    if mode == 2:
        return ref.rms_norm(x, aux, EPS)
    return ((orc.silu(x) if mode == 1 else orc.gelu(x)) * aux).astype(F32)


@pytest.mark.parametrize("mode", [0, 1, 2, 3])
@pytest.mark.parametrize("type_", [0, 1, 30])
@pytest.mark.parametrize("n", [32, 96, 704, 2048, 2080, 8192, 8224, 20000])
def test_quant_rows(ctx, orc, n, type_, mode):
    """Rows apart by more than their length (gate and up in one buffer), ties, an empty row; equal bit for bit."""
    print(f"quant_i8 mode {mode} type {type_} n {n}", flush=True)
    rng = np.random.default_rng(n + 10 * mode + type_)
    rows, ld = 5, 2 * n + 8
    both = (2 * rng.standard_normal((rows, ld))).astype(F32)
    both[1, :n] = 0
    both[2, :n] = np.tile(np.array([127, -127, 2.5, -2.5, 0.5, -0.5, 1.5, 126.5], F32), n // 8)
    raw, both = held(both, type_)
    x, aux = both[:, :n], both[:, n:2 * n]
    with Bufs(ctx) as B:
        src = B.of(raw)
        weight = (1 + 0.2 * rng.standard_normal(n)).astype(F32)
        if mode == 2:
            aux, pa = weight, B.of(weight).ptr
        else:
            pa = None if mode == 0 else src.ptr + n * raw.itemsize
        qs, d = B.of(np.full((rows + 1, n), 99, np.int8)), B.of(np.full(rows + 1, 99, F32))
        ctx.quant_i8_device(mode, type_, src.ptr, pa, rows, n, ld, EPS, qs.ptr, d.ptr)
        ctx.sync()
        got, gd = qs.download((rows + 1, n), np.int8), d.download(rows + 1)
    rq, rd = ref.quant(transformed(orc, mode, x, aux))
    np.testing.assert_array_equal(gd[:rows].view(np.uint32), rd.view(np.uint32))
    np.testing.assert_array_equal(got[:rows], rq)
    assert (got[rows] == 99).all() and gd[rows] == 99  # behind the last row


def test_quant_edge_rows(ctx):
    """Scales at the ends of the type, and rows that hold a NaN or an infinity."""
    n = 64
    x = np.zeros((9, n), F32)
    x[0, 5] = 1e-44
    x[1, :] = 3e-38  # the scale would be under 2^-126
    x[2, 3] = 127 * 1.1754944e-38
    x[3, :] = np.linspace(-3.4e38, 3.4e38, n)
    x[4, :2] = 1.0, np.nan
    x[5, :2] = 1.0, np.inf
    x[6, :2] = -np.inf, np.nan
    x[7, :] = -0.0
    x[8, :2] = 1.0, 1e-30
    q, d = ctx.QuantI8(0, x)
    rq, rd = ref.quant(x)
    np.testing.assert_array_equal(q, rq)
    np.testing.assert_array_equal(d, rd)
    assert np.isnan(d[4:7]).all() and (q[4:7] == 0).all()


def test_quant_many_rows(ctx):
    """A grid of many rows."""
    x = np.random.default_rng(1).standard_normal((70001, 32)).astype(F32)
    q, d = ctx.QuantI8(0, x)
    rq, rd = ref.quant(x)
    np.testing.assert_array_equal(q, rq)
    np.testing.assert_array_equal(d, rd)


# ---------------------------------------------------------------------------------------- products
def check_product(ctx, T, rows, cols, type_, seed):
    print(f"matmul_i8 T {T} rows {rows} cols {cols} type {type_}", flush=True)
    rng = np.random.default_rng(seed)
    w, scale = ref.weights_of(rng, rows, cols)
    xq, xd = ref.rows_of(rng, T, cols)
    xq[0, :2] = -128, 127
    h = ctx.weight_upload_i8(1, rows, cols, w, scale)
    item = 4 if type_ == 0 else 2
    try:
        with Bufs(ctx) as B:
            pad = np.full(T * rows * item + 64, 0x5A, np.uint8)
            y = B.of(pad)
            ctx.matmul_i8_device(h, T, B.of(xq).ptr, B.of(xd).ptr, type_, y.ptr)
            ctx.sync()
            got = read(y, (T, rows), type_)
            assert (y.download(pad.shape, np.uint8)[T * rows * item:] == 0x5A).all()
    finally:
        ctx.weight_free(h)
    want = ref.product(xq, xd, w, scale)
    # the sum, the scales' product and the value, each rounded once; then the type
    bound = (3 * STEP[0] + (STEP[type_] if type_ else 0)) * 1.01 * np.abs(want)
    assert (np.abs(got - want) <= bound + (2.0 ** -25 if type_ == 1 else 0)).all()


@pytest.mark.parametrize("type_", [0, 1, 30])
@pytest.mark.parametrize("shape", [(1, 1, 32), (1, 33, 96), (2, 64, 128), (31, 31, 160), (32, 100, 256), (33, 257, 544), (64, 128, 2816),
                                   (77, 352, 704), (129, 96, 1024), (300, 260, 2080), (257, 513, 384)])
def test_matmul(ctx, shape, type_):
    check_product(ctx, *shape, type_, seed=sum(shape))


@pytest.mark.parametrize("shape", [(50, 8200, 96), (70, 8200, 64), (100, 16400, 64), (128, 16416, 160), (20, 8200, 32), (700, 8200, 96)])
def test_matmul_many_outputs(ctx, shape):
    """Outputs enough for the wider row tiles."""
    check_product(ctx, *shape, 30, seed=sum(shape))


def test_matmul_longest_rows(ctx):
    """65536 columns of the largest magnitudes: the sum's largest value, exact in int32."""
    T, rows, cols = 3, 40, 65536
    w = np.full((rows, cols), -128, np.int8)
    w[1::2] = 127
    scale = np.full(rows, 2.0 ** -20, F32)
    xq = np.full((T, cols), -128, np.int8)
    xq[1] = 127
    xd = np.full(T, 2.0 ** -10, F32)
    h = ctx.weight_upload_i8(1, rows, cols, w, scale)
    try:
        got = ctx.MatMulI8(h, rows, cols, xq, xd)
    finally:
        ctx.weight_free(h)
    want = ref.product(xq, xd, w, scale)
    assert (np.abs(got - want) <= STEP[0] * np.abs(want)).all()  # only the sum's rounding: the scales are powers of two


def test_matmul_many_rows(ctx):
    check_product(ctx, 70000, 33, 32, 0, seed=9)


def test_special_scales(ctx):
    """A NaN token scale (a row that held one) reaches its outputs and no others; zero rows give zeros."""
    rng = np.random.default_rng(2)
    w, scale = ref.weights_of(rng, 70, 96)
    xq, xd = ref.rows_of(rng, 40, 96)
    xd[7], xq[7], xd[9], xq[9] = np.nan, 0, 0, 0
    h = ctx.weight_upload_i8(1, 70, 96, w, scale)
    try:
        y = ctx.MatMulI8(h, 70, 96, xq, xd)
    finally:
        ctx.weight_free(h)
    assert np.isnan(y[7]).all() and (y[9] == 0).all() and np.isfinite(np.delete(y, 7, 0)).all()


def test_weights_from_device_memory(ctx):
    """The same handle from host arrays, from device buffers, and from an address no 16 bytes divide."""
    rng = np.random.default_rng(4)
    w, scale = ref.weights_of(rng, 65, 160)
    xq, xd = ref.rows_of(rng, 5, 160)
    with Bufs(ctx) as B:
        off = np.concatenate([np.zeros(3, np.int8), w.reshape(-1)])
        hs = [ctx.weight_upload_i8(1, 65, 160, w, scale), ctx.weight_upload_i8(1, 65, 160, B.of(w).ptr, B.of(scale).ptr),
              ctx.weight_upload_i8(1, 65, 160, B.of(off).ptr + 3, scale)]
        ys = [ctx.MatMulI8(h, 65, 160, xq, xd) for h in hs]
        for h in hs:
            ctx.weight_free(h)
    np.testing.assert_array_equal(ys[0], ys[1])
    np.testing.assert_array_equal(ys[0], ys[2])


# ---------------------------------------------------------------------------------------- activations
def test_activations_of_the_experts(ctx, orc):
    """The forms in the products' epilogues give the library's silu and gelu: gelu at every fp16 value and between them,
    silu over the whole range with the places where its quotient leaves the normal numbers."""
    every = np.arange(65536, dtype=np.uint16).view(np.float16).astype(F32)
    rng = np.random.default_rng(12)
    x = np.concatenate([every, (4 * rng.standard_normal(1 << 20)).astype(F32), rng.uniform(-110, 110, 1 << 18).astype(F32),
                        np.array([0.0, -0.0, 1e-40, -1e-40, 79.99999, -79.99999, 80, -80, -88.7, -88.8, -104, 3e38, -3e38, 10, -10,
                                  9.9999, -9.9999, 9.998, np.inf, -np.inf, np.nan], F32)])
    one = np.ones_like(x)
    with np.errstate(all="ignore"):
        np.testing.assert_array_equal(ctx.selftest(11, x, one), orc.silu(x))
        finite = x[~np.isnan(x)]
        np.testing.assert_array_equal(ctx.selftest(12, finite, np.ones_like(finite)), orc.gelu(finite))
    assert (ctx.selftest(12, np.full(64, np.nan, F32), np.ones(64, F32)) == 0).all()  # the table's value


# ---------------------------------------------------------------------------------------- experts
def expert_case(rng, E, d, nf):
    wg, sg = ref.weights_of(rng, E, 2 * nf, d)
    wd, sd = ref.weights_of(rng, E, d, nf)
    return wg, sg, wd, sd


@functools.lru_cache(maxsize=2)
def big_experts(E, d, nf):
    """Matrices of random bytes: quick to make where there are many."""
    rng = np.random.default_rng(E + nf)
    return (rng.integers(-90, 91, (E, 2 * nf, d), dtype=np.int8), (6e-4 * (1 + 0.3 * rng.random((E, 2 * nf)))).astype(F32),
            rng.integers(-90, 91, (E, d, nf), dtype=np.int8), (6e-4 * (1 + 0.3 * rng.random((E, d)))).astype(F32))


def upload(ctx, W):
    wg, sg, wd, sd = W
    E, n2, d = wg.shape
    return ctx.weight_upload_i8(E, n2, d, wg, sg, paired=True), ctx.weight_upload_i8(E, d, n2 // 2, wd, sd)


def check_experts(ctx, pkg, orc, W, xq, xd, ids, weights, act, types=(0,)):
    T, d = xq.shape
    k = ids.shape[1]
    hs = upload(ctx, W)
    try:
        with Bufs(ctx) as B:
            ins = [B.of(a).ptr for a in (xq, xd, ids, weights)]
            for type_ in types:
                print(f"experts_i8 T {T} d {d} E {W[0].shape[0]} k {k} nf {W[2].shape[2]} act {act} type {type_}", flush=True)
                out = B.of(np.full(T * d * (4 if type_ == 0 else 2) + 64, 0x5A, np.uint8))
                ctx.experts_i8_device(*hs, act, T, k, *ins, type_, out.ptr)
                ctx.sync()
                got = read(out, (T, d), type_)
                assert (out.download((out.nbytes,), np.uint8)[-64:] == 0x5A).all()
                want, size = ref.experts(xq, xd, ids, weights, *W, act_of(pkg, orc, act))
                # a term: three roundings of the product, one of its weight's; k - 1 additions; then the type
                bound = (4 + k) * STEP[0] * 1.01 * size + (STEP[type_] * 1.01 * np.abs(want) if type_ else 0)
                assert (np.abs(got - want) <= bound + (2.0 ** -25 if type_ == 1 else 0)).all()
                assert (got[(ids < 0).all(1) | (ids >= W[0].shape[0]).all(1)] == 0).all()
    finally:
        for h in hs:
            ctx.weight_free(h)


@pytest.mark.parametrize("act", [1, 3])
@pytest.mark.parametrize("T", [1, 2, 7, 33, 130, 400])
@pytest.mark.parametrize("dims", [(8, 64, 32, 2), (5, 96, 96, 5), (32, 512, 160, 4), (128, 256, 64, 8), (1, 32, 32, 1)])
def test_experts(ctx, pkg, orc, dims, T, act):
    E, d, nf, k = dims
    rng = np.random.default_rng(T + E)
    W = expert_case(rng, E, d, nf)
    xq, xd = ref.rows_of(rng, T, d)
    ids = np.argsort(rng.random((T, E)) ** 2, axis=1)[:, :k].astype(np.int32)
    weights = rng.random((T, k)).astype(F32)
    check_experts(ctx, pkg, orc, W, xq, xd, ids, weights, act, types=(0, 1, 30))


@pytest.mark.parametrize("T", [20, 100, 200, 300, 600])
def test_experts_past_the_caches(ctx, pkg, orc, T):
    """Experts of 138 MB: lists of every tile capacity, with weights that are read once, and the tile kernel both ways."""
    E, d, nf, k = 128, 1024, 352, 8
    W = big_experts(E, d, nf)
    rng = np.random.default_rng(T)
    xq, xd = ref.rows_of(rng, T, d)
    ids = np.argsort(rng.random((T, E)) ** 2, axis=1)[:, :k].astype(np.int32)
    ids[T // 2, 1] = -1
    check_experts(ctx, pkg, orc, W, xq, xd, ids, rng.random((T, k)).astype(F32), 1)


@pytest.mark.parametrize("case", [(64, 512, 1024, 4, 24), (32, 512, 672, 4, 60), (32, 512, 672, 4, 100), (32, 512, 672, 4, 130)])
def test_experts_in_the_caches(ctx, pkg, orc, case):
    """Lists of every tile capacity, and the tile kernel, over fewer bytes."""
    E, d, nf, k, T = case
    W = big_experts(E, d, nf)
    rng = np.random.default_rng(T)
    xq, xd = ref.rows_of(rng, T, d)
    ids = rng.integers(0, E, (T, k)).astype(np.int32)
    check_experts(ctx, pkg, orc, W, xq, xd, ids, rng.random((T, k)).astype(F32), 3, types=(0, 30))


@pytest.mark.parametrize("T", [1, 6, 150])
def test_experts_skipped_places(ctx, pkg, orc, T):
    """Places without an expert, tokens without any, ids out of range, the same expert twice, every token on one."""
    E, d, nf, k = 6, 128, 64, 3
    rng = np.random.default_rng(T)
    W = expert_case(rng, E, d, nf)
    xq, xd = ref.rows_of(rng, T, d)
    weights = rng.standard_normal((T, k)).astype(F32)
    for name in ("some", "none", "wild", "twice", "one"):
        ids = rng.integers(0, E, (T, k)).astype(np.int32)
        if name == "some":
            ids[rng.random((T, k)) < 0.5] = -1
        elif name == "none":
            ids[:] = -1
        elif name == "wild":
            ids[rng.random((T, k)) < 0.5] = [E, 1 << 30, -(1 << 31), -7][T % 4]
        elif name == "twice":
            ids[:] = ids[:, :1]
        else:
            ids[:] = 4
        check_experts(ctx, pkg, orc, W, xq, xd, ids, weights, 1)


def test_experts_chunks(ctx, pkg, orc):
    """More assignments than one chunk takes (65535 / k tokens)."""
    E, d, nf, k, T = 16, 32, 32, 4, 20011
    rng = np.random.default_rng(8)
    W = expert_case(rng, E, d, nf)
    xq, xd = ref.rows_of(rng, T, d)
    ids = rng.integers(-1, E, (T, k)).astype(np.int32)
    check_experts(ctx, pkg, orc, W, xq, xd, ids, rng.random((T, k)).astype(F32), 1, types=(0, 30))


def test_experts_row_with_nan(ctx, pkg):
    """A token whose row held a NaN: its output is NaN, its neighbours' are not."""
    E, d, nf, k, T = 4, 64, 32, 2, 9
    rng = np.random.default_rng(6)
    hs = upload(ctx, expert_case(rng, E, d, nf))
    x = rng.standard_normal((T, d)).astype(F32)
    x[4, 10] = np.nan
    xq, xd = ctx.QuantI8(0, x)
    ids = rng.integers(0, E, (T, k)).astype(np.int32)
    try:
        out = ctx.ExpertsI8(*hs, 1, xq, xd, ids, np.ones((T, k), F32))
    finally:
        for h in hs:
            ctx.weight_free(h)
    assert np.isnan(out[4]).all() and np.isfinite(np.delete(out, 4, 0)).all()


# ---------------------------------------------------------------------------------------- together
@pytest.mark.parametrize("T", [1, 19, 260])
def test_router_rows_experts_projection(ctx, pkg, orc, T):
    """A layer as a program runs it, on device buffers with no wait in between: the router's choice, the normed rows as
    int8, the experts, their output as int8 again, a dense projection."""
    E, d, nf, k, rows = 24, 256, 96, 4, 320
    rng = np.random.default_rng(T)
    W = expert_case(rng, E, d, nf)
    wp, sp = ref.weights_of(rng, rows, d)
    x = rng.standard_normal((T, d)).astype(F32)
    norm = (1 + 0.1 * rng.standard_normal(d)).astype(F32)
    logits = rng.standard_normal((T, E)).astype(F32)
    if T > 4:
        logits[T - 2:] = -np.inf  # the empty rows of a padded batch
    bias = (0.1 * rng.standard_normal(E)).astype(F32)
    D = pkg.RouteDesc(E, k, score=1, n_group=4, n_group_used=2, group_score=1, scale=2.5)
    hs = upload(ctx, W) + (ctx.weight_upload_i8(1, rows, d, wp, sp),)
    try:
        with Bufs(ctx) as B:
            bx, bn, bl, bb = (B.of(a) for a in (x, norm, logits, bias))
            ids, wt, q, s, o, q2, s2, y = (B.empty(n) for n in (T * k * 4, T * k * 4, T * d, T * 4, T * d * 4, T * d, T * 4,
                                                                T * rows * 4))
            ctx.route_device(D, T, bl.ptr, bb.ptr, ids.ptr, wt.ptr)
            ctx.quant_i8_device(2, 0, bx.ptr, bn.ptr, T, d, d, EPS, q.ptr, s.ptr)
            ctx.experts_i8_device(hs[0], hs[1], 1, T, k, q.ptr, s.ptr, ids.ptr, wt.ptr, 0, o.ptr)
            ctx.quant_i8_device(0, 0, o.ptr, None, T, d, d, EPS, q2.ptr, s2.ptr)
            ctx.matmul_i8_device(hs[2], T, q2.ptr, s2.ptr, 0, y.ptr)
            ctx.sync()
            got_ids, got_w = ids.download((T, k), np.int32), wt.download((T, k))
            got_o, got_y = o.download((T, d)), y.download((T, rows))
            got_q2, got_s2 = q2.download((T, d), np.int8), s2.download(T)
    finally:
        for h in hs:
            ctx.weight_free(h)
    rids, rw = ref.route(D, logits, bias)
    np.testing.assert_array_equal(got_ids, rids)
    xq, xd = ref.quant(ref.rms_norm(x, norm, EPS))
    want, size = ref.experts(xq, xd, rids, got_w, *W, orc.silu)
    assert (np.abs(got_o - want) <= (4 + k) * STEP[0] * 1.01 * size).all()
    if T > 4:
        assert (got_o[T - 2:] == 0).all()
    rq2, rs2 = ref.quant(got_o)
    np.testing.assert_array_equal(got_q2, rq2)
    want_y = ref.product(rq2, rs2, wp, sp)
    assert (np.abs(got_y - want_y) <= 3 * STEP[0] * 1.01 * np.abs(want_y)).all()


def test_two_contexts_and_a_captured_stack(pkg, ctx, orc):
    """Calls of two contexts in flight together, and a stack captured before the int8 calls that still runs after them."""
    E, d, nf, k, T = 8, 128, 64, 2, 50
    rng = np.random.default_rng(5)
    W = expert_case(rng, E, d, nf)
    xq, xd = ref.rows_of(rng, T, d)
    ids = rng.integers(0, E, (T, k)).astype(np.int32)
    weights = rng.random((T, k)).astype(F32)
    want, size = ref.experts(xq, xd, ids, weights, *W, orc.silu)
    L = pkg.synth.make_layer("c1_tiny")
    xs = pkg.synth.make_input("c1_tiny")
    with pkg.MoeContext(0) as other:
        other.upload(0, L)
        other.stack_capture(0, 1, xs.shape[0])
        before = other.stack_run(xs)
        hs = {c: upload(c, W) for c in (ctx, other)}
        with Bufs(ctx) as B:
            ins = [B.of(a).ptr for a in (xq, xd, ids, weights)]
            outs = {c: B.empty(T * d * 4) for c in hs}
            for _ in range(5):
                for c, h in hs.items():
                    c.experts_i8_device(*h, 1, T, k, *ins, 0, outs[c].ptr)
            for c in hs:
                c.sync()
            for o in outs.values():
                assert (np.abs(o.download((T, d)) - want) <= (4 + k) * STEP[0] * 1.01 * size).all()
        for c, h in hs.items():
            for x in h:
                c.weight_free(x)
        np.testing.assert_array_equal(other.stack_run(xs), before)


# ---------------------------------------------------------------------------------------- refusals
def test_refusals(ctx, pkg):
    rng = np.random.default_rng(0)
    w, scale = ref.weights_of(rng, 64, 64)
    plain = ctx.weight_upload_i8(1, 64, 64, w, scale)
    paired = ctx.weight_upload_i8(1, 64, 64, w, scale, paired=True)
    other = ctx.weight_upload_i8(1, 64, 32, w[:, :32], scale)
    q8 = ctx.weight_upload(pkg.PHX.Q8_0, np.zeros(64 * 2 * 34, np.uint8), 64, 64)
    host = np.zeros(4096, np.int8)
    arg, no = pkg.ArgumentError, pkg.NotSupportedError

    def refuse(call, ok, *changes):
        call(*ok)
        for at, value, error in changes:
            bad = list(ok)
            bad[at] = value
            with pytest.raises(error):
                call(*bad)
        call(*ok)
        ctx.sync()

    try:
        with Bufs(ctx) as B:
            a, b, c, o = (B.of(np.zeros(65536, np.uint8)).ptr for _ in range(4))
            refuse(ctx.quant_i8_device, (1, 0, a, b, 2, 64, 64, EPS, c, o),
                   (0, 4, arg), (0, -1, arg), (1, 2, no), (2, None, arg), (2, a + 4, arg), (3, None, arg), (3, b + 8, arg), (4, 0, arg),
                   (4, (1 << 20) + 1, arg), (5, 48, arg), (5, 0, arg), (5, 65568, arg), (6, 56, arg), (6, 68, arg), (8, None, arg),
                   (8, c + 4, arg), (8, a, arg), (9, None, arg), (9, o + 2, arg), (9, c, arg), (2, host.ctypes.data, arg))
            refuse(ctx.quant_i8_device, (2, 0, a, b, 2, 64, 64, EPS, c, o), (7, float("nan"), arg), (7, -1.0, arg))
            refuse(ctx.matmul_i8_device, (plain, 4, a, b, 0, o),
                   (0, None, arg), (0, paired, no), (0, q8, no), (1, 0, arg), (1, (1 << 20) + 1, arg), (2, None, arg), (2, a + 8, arg),
                   (3, b + 2, arg), (4, 8, no), (5, None, arg), (5, o + 8, arg), (5, a, arg), (5, host.ctypes.data, arg))
            down = ctx.weight_upload_i8(1, 64, 32, w[:, :32], scale)
            refuse(ctx.experts_i8_device, (paired, down, 1, 3, 2, a, b, c, c + 4096, 0, o),
                   (0, plain, no), (1, paired, no), (1, plain, arg), (0, q8, no), (1, None, arg), (2, 0, arg), (2, 2, arg), (3, 0, arg),
                   (4, 0, arg), (4, 17, arg), (5, None, arg), (5, a + 4, arg), (6, b + 1, arg), (7, None, arg), (8, None, arg), (9, 5, no),
                   (10, a, arg), (10, b, arg), (10, o + 4, arg), (7, host.ctypes.data, arg))
            ctx.weight_free(down)
        for call in (lambda: ctx.matmul_device(plain, 1, 0, 0, 0), lambda: ctx.lib.phx_matmul_i8(None, plain, 1, 0, 0, 0, 0)):
            try:
                assert call() == pkg.PHX.ERR_ARG
            except pkg.MoeError:
                pass
        for bad in ((0, 64, 64), (257, 64, 64), (1, 0, 64), (1, 64, 48), (1, 64, 0), (1, 64, 65568), (1, (1 << 20) + 1, 32)):
            with pytest.raises(arg):
                ctx.weight_upload_i8(*bad, w.ctypes.data, scale.ctypes.data)
        with pytest.raises(arg):
            ctx.weight_upload_i8(1, 32, 64, w[:32], scale[:32], paired=True)  # rows no multiple of 64
        with pytest.raises(arg):
            ctx.weight_upload_i8(1, 64, 64, w[:, :32], scale)
    finally:
        for h in (plain, paired, other, q8):
            ctx.weight_free(h)


def test_int8_handles_are_refused_by_the_other_products(ctx, pkg):
    w, scale = ref.weights_of(np.random.default_rng(0), 64, 256)
    h = ctx.weight_upload_i8(1, 64, 256, w, scale)
    try:
        with Bufs(ctx) as B:
            a, b, c = (B.empty(4096).ptr for _ in range(3))
            for call in (ctx.matmul_device, ctx.matmul_k_device):
                with pytest.raises(pkg.NotSupportedError):
                    call(h, 1, a, b, c)
    finally:
        ctx.weight_free(h)


def test_allocation_and_launch_faults(pkg, orc, monkeypatch):
    """A failed allocation or launch inside the calls: an error, and the same call then gives the right result."""
    E, d, nf, k, T = 4, 64, 32, 2, 10
    rng = np.random.default_rng(3)
    W = expert_case(rng, E, d, nf)
    xq, xd = ref.rows_of(rng, T, d)
    ids = rng.integers(0, E, (T, k)).astype(np.int32)
    weights = rng.random((T, k)).astype(F32)
    want, size = ref.experts(xq, xd, ids, weights, *W, orc.silu)
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
                    hs = upload(c, W)
                    out = c.ExpertsI8(*hs, 1, xq, xd, ids, weights)
                    break
                except (pkg.OutOfDeviceMemoryError, pkg.GpuDeviceLostError) as e:
                    seen.add(type(e).__name__)
                    assert attempt == 0
            assert (np.abs(out - want) <= (4 + k) * STEP[0] * 1.01 * size).all()
    assert seen == {"OutOfDeviceMemoryError", "GpuDeviceLostError"}
