"""Low-rank adapters of many requests (phx_lora_create, phx_lora_set, phx_lora_add) against their definition in 64 bits
(tests/half_ref.py): ranks from 1 to the most, slots set, replaced and emptied, rows without an adapter, sections of a wider
matrix, in place and apart, infinities that must not spread, and the run behind the norm and the int8 projection."""
import numpy as np
import pytest

import half_ref as ref
import i8_ref
from test_gpu_i8 import Bufs

pytestmark = pytest.mark.gpu

F32 = np.float32


def adapters(ctx, rng, type_, n_slot, max_rank, rows, cols, ranks):
    """A handle, and its slots as {number: (A, B, scale)} in float64."""
    h = ctx.lora_create(type_, n_slot, max_rank, rows, cols)
    slots = {}
    for s, rank in ranks.items():
        ra, a = ref.held(rng.standard_normal((rank, cols)) / np.sqrt(cols), type_)
        rb, b = ref.held(0.3 * rng.standard_normal((rows, rank)), type_)
        scale = float(F32(0.5 + s))
        ctx.lora_set(h, s, rank, ra, rb, scale)
        slots[s] = a, b, scale
    return h, slots


def run(ctx, h, T, raw_x, ids, y_type, ld, rows, before, in_place=False, col=0):
    """lora_add on rows of a matrix of ld values, from column col; the whole matrix's bytes afterwards."""
    item = 4 if y_type == 0 else 2
    with Bufs(ctx) as B:
        y_in = B.of(before)
        y = y_in if in_place else B.of(np.full(before.nbytes + 64, 0x3A, np.uint8))
        ctx.lora_add_device(h, T, B.of(raw_x).ptr, B.of(ids.astype(np.int32)).ptr, y_type, ld, y_in.ptr + col * item, y.ptr + col * item)
        ctx.sync()
        got, raw = ref.read(y, (T, ld), y_type), y.download((before.nbytes,) if in_place else (before.nbytes + 64,), np.uint8)
        if not in_place:
            assert (raw[before.nbytes:] == 0x3A).all()
            np.testing.assert_array_equal(y_in.download(before.shape, before.dtype), before)
    outside = np.ones(ld, bool)
    outside[col:col + rows] = False
    kept = raw[:before.nbytes].reshape(T, ld, item)[:, outside]
    assert (kept == (before.view(np.uint8).reshape(T, ld, item)[:, outside] if in_place else 0x3A)).all()
    return got[:, col:col + rows]


def check(ctx, type_, y_type, T, rows, cols, max_rank, ranks, ids, in_place=False, extra=0, col=0, seed=0):
    print(f"lora type {type_} y {y_type} T {T} {rows} x {cols} ranks {ranks} in place {in_place} ld +{extra}", flush=True)
    rng = np.random.default_rng(seed + T + rows + cols)
    n_slot = max(ranks, default=0) + 2
    h, slots = adapters(ctx, rng, type_, n_slot, max_rank, rows, cols, ranks)
    raw_x, x = ref.held(rng.standard_normal((T, cols)), type_)
    ld = rows + extra
    raw_y, y_in = ref.held(rng.standard_normal((T, ld)), y_type)
    try:
        got = run(ctx, h, T, raw_x, ids, y_type, ld, rows, raw_y, in_place, col)
    finally:
        ctx.lora_free(h)
    want, bound = ref.lora(x, ids, slots, y_in[:, col:col + rows].copy(), type_, y_type)
    bare = ~np.isin(ids, list(slots))
    np.testing.assert_array_equal(got[bare], y_in[bare][:, col:col + rows])
    bound = ref.rounded(want, bound, y_type)
    assert (np.abs(got - want) <= bound).all(), (np.abs(got - want) / bound).max()


@pytest.mark.parametrize("type_,y_type", [(1, 1), (1, 0), (30, 30), (30, 0), (30, 1)])
@pytest.mark.parametrize("T", [1, 5, 16, 17, 40, 300])
def test_mixed_slots(ctx, T, type_, y_type):
    """Ranks 1 to 40 in slots out of order, empty slots, ids without one."""
    ids = np.random.default_rng(T).integers(-2, 9, T)
    check(ctx, type_, y_type, T, 200, 264, 40, {0: 16, 3: 1, 4: 40, 5: 17, 6: 8}, ids)


@pytest.mark.parametrize("shape", [(1, 8), (7, 24), (63, 32), (64, 40), (65, 1000), (129, 4096), (1000, 8)])
@pytest.mark.parametrize("T", [1, 33])
def test_odd_sizes(ctx, T, shape):
    rows, cols = shape
    check(ctx, 30, 30, T, rows, cols, 20, {0: 20, 1: 5}, np.arange(T) % 3 - 1 if T > 1 else np.array([0]))
    check(ctx, 1, 0, T, rows, cols, 20, {0: 20, 1: 5}, np.arange(T) % 3 if T > 1 else np.array([1]), in_place=True)


@pytest.mark.parametrize("y_type", [0, 1, 30])
@pytest.mark.parametrize("extra,col", [(8, 8), (8, 0), (3, 1), (64, 24)])
def test_sections(ctx, extra, col, y_type):
    """Columns of a wider matrix, aligned or not; what lies beside them stays."""
    ids = np.arange(50) // 9 - 1
    for in_place in (False, True):
        check(ctx, 1, y_type, 50, 96, 64, 8, {0: 8, 2: 3}, ids, in_place=in_place, extra=extra, col=col)


@pytest.mark.parametrize("rank", [1, 15, 16, 31, 64, 127, 128])
def test_ranks(ctx, rank):
    for T in (1, 20):
        check(ctx, 30, 0, T, 70, 328, rank, {0: rank, 1: max(1, rank - 1)}, np.arange(T) % 2)


def test_prompts(ctx):
    """Rows of one request after another, lengths of no multiple, many rows."""
    ids = np.concatenate([np.full(n, s) for s, n in ((2, 1000), (0, 7), (-1, 33), (1, 1500), (2, 3), (0, 457))])
    check(ctx, 30, 30, len(ids), 264, 520, 32, {0: 32, 1: 16, 2: 9}, ids)


def test_many_slots(ctx):
    ids = np.random.default_rng(0).permutation(256)
    check(ctx, 1, 1, 256, 40, 64, 4, {s: 1 + s % 4 for s in range(0, 255)}, ids)


@pytest.mark.parametrize("type_,y_type", [(1, 0), (30, 30)])
@pytest.mark.parametrize("rank,T", [(16, 1023), (16, 1024), (16, 1025), (32, 1100), (33, 512), (40, 513), (128, 600)])
def test_many_rows_of_mixed_slots(ctx, rank, T, type_, y_type):
    """About the sizes where the slots of a tile go one after another in place of side by side; every tile of many slots."""
    ids = np.random.default_rng(rank + T).integers(-1, 5, T)
    check(ctx, type_, y_type, T, 136, 72, rank, {0: rank, 2: rank - 1, 3: 1, 4: min(rank, 17)}, ids, in_place=T % 2 == 0)


@pytest.mark.parametrize("T", [9, 700, 1100])
def test_same_call_same_bits(ctx, T):
    rng = np.random.default_rng(T)
    h, _ = adapters(ctx, rng, 30, 4, 24, 520, 1024, {0: 24, 1: 3, 2: 16})
    raw_x, _ = ref.held(rng.standard_normal((T, 1024)), 30)
    raw_y, _ = ref.held(rng.standard_normal((T, 520)), 30)
    ids = rng.integers(-1, 4, T)
    try:
        first = run(ctx, h, T, raw_x, ids, 30, 520, 520, raw_y)
        for _ in range(3):
            np.testing.assert_array_equal(run(ctx, h, T, raw_x, ids, 30, 520, 520, raw_y), first)
    finally:
        ctx.lora_free(h)


def test_long_batch(ctx):
    """More rows than one chunk of the workspace takes."""
    check(ctx, 30, 30, 70001, 8, 8, 3, {0: 3, 1: 2}, np.arange(70001) // 5 % 3)


def test_slots_are_replaced_and_emptied(ctx):
    """A slot takes an adapter of a lower rank, then none; calls already enqueued see it as it was."""
    rng = np.random.default_rng(3)
    rows, cols, T = 72, 64, 20
    h, slots = adapters(ctx, rng, 1, 2, 16, rows, cols, {0: 16, 1: 4})
    raw_x, x = ref.held(rng.standard_normal((T, cols)), 1)
    raw_y, y_in = ref.held(rng.standard_normal((T, rows)), 0)
    ids = np.arange(T) % 2
    try:
        with Bufs(ctx) as B:
            xb, ib, yb = B.of(raw_x), B.of(ids.astype(np.int32)), B.of(raw_y)
            outs = [B.empty(raw_y.nbytes) for _ in range(3)]
            expected = []
            for k, out in enumerate(outs):
                if k == 1:
                    ra, a = ref.held(rng.standard_normal((3, cols)), 1)
                    rb, b = ref.held(rng.standard_normal((rows, 3)), 1)
                    ctx.lora_set(h, 0, 3, ra, rb, -2.0)
                    slots[0] = a, b, -2.0
                if k == 2:
                    ctx.lora_set(h, 0, 0, None, None)
                    del slots[0]
                ctx.lora_add_device(h, T, xb.ptr, ib.ptr, 0, rows, yb.ptr, out.ptr)
                expected.append(ref.lora(x, ids, dict(slots), y_in, 1, 0))
            ctx.sync()
            for out, (want, bound) in zip(outs, expected):
                assert (np.abs(out.download((T, rows)) - want) <= ref.rounded(want, bound, 0)).all()
    finally:
        ctx.lora_free(h)


@pytest.mark.parametrize("type_", [1, 30])
def test_infinities_stay_in_their_row(ctx, type_):
    """Rows with an infinity or a NaN beside others of the same slot; a slot whose matrices hold NaNs that no row names; values of A x
    past fp16's range."""
    rng = np.random.default_rng(6)
    rows, cols, T = 40, 40, 18
    h, slots = adapters(ctx, rng, type_, 3, 5, rows, cols, {0: 5})
    bad = ref.held(np.full((5, cols), np.inf), 1)[0] if type_ == 1 else np.full((5, cols), 0x7FC0, np.uint16)
    ctx.lora_set(h, 1, 5, bad, bad.reshape(-1)[:rows * 5].reshape(rows, 5), 1.0)
    raw_x, x = ref.held(rng.standard_normal((T, cols)), type_)
    for row, v in ((2, np.inf), (5, -np.inf), (9, np.nan)):
        raw_x[row, cols - 1] = v if type_ == 1 else {np.inf: 0x7F80, -np.inf: 0xFF80}.get(v, 0x7FC0)
    big = 6e4 if type_ == 1 else 1e30
    raw_x[12], x[12] = (r[0] for r in ref.held(np.full((1, cols), big) * np.sign(slots[0][0][1]), type_))
    raw_y, y_in = ref.held(rng.standard_normal((T, rows)), 0)
    try:
        got = run(ctx, h, T, raw_x, np.zeros(T, int), 0, rows, rows, raw_y)
    finally:
        ctx.lora_free(h)
    fine = ~np.isin(np.arange(T), (2, 5, 9))
    want, bound = ref.lora(x[fine], np.zeros(fine.sum(), int), slots, y_in[fine], type_, 0)
    assert (np.abs(got[fine] - want) <= ref.rounded(want, bound, 0)).all()
    assert not np.isfinite(got[~fine]).any()


def test_norm_projection_adapters(ctx):
    """A layer's step as it is used: the residual's norm, the int8 projection of its rows, the adapters of its float rows, in one queue
    without a wait; each step against its definition of the step before's stored values."""
    rng = np.random.default_rng(11)
    T, n, rows = 37, 256, 160
    w, scale = i8_ref.weights_of(rng, rows, n)
    proj = ctx.weight_upload_i8(1, rows, n, w, scale)
    h, slots = adapters(ctx, rng, 30, 4, 16, rows, n, {0: 16, 2: 7})
    raw_x, x = ref.held(rng.standard_normal((T, n)), 30)
    raw_b, _ = ref.held(rng.standard_normal((T, n)), 30)
    norm = (1 + 0.1 * rng.standard_normal(n)).astype(F32)
    ids = rng.integers(-1, 4, T).astype(np.int32)
    try:
        with Bufs(ctx) as B:
            xb, out, qs, d, y, z = B.of(raw_x), B.empty(T * n * 2), B.empty(T * n), B.empty(T * 4), B.empty(T * rows * 4), B.empty(T * rows * 4)
            pb, pw, pi = B.of(raw_b).ptr, B.of(norm).ptr, B.of(ids).ptr
            ctx.add_norm_i8_device(30, xb.ptr, pb, pw, T, n, n, 1e-6, xb.ptr, 30, out.ptr, qs.ptr, d.ptr)
            ctx.matmul_i8_device(proj, T, qs.ptr, d.ptr, 0, y.ptr)
            ctx.lora_add_device(h, T, out.ptr, pi, 0, rows, y.ptr, z.ptr)
            ctx.sync()
            q, dv, v = qs.download((T, n), np.int8), d.download(T), ref.read(out, (T, n), 30)
            s, yv, zv = ref.read(xb, (T, n), 30), y.download((T, rows)), z.download((T, rows))
    finally:
        ctx.weight_free(proj)
        ctx.lora_free(h)
    np.testing.assert_array_equal(s, ref.held(x.astype(F32) + i8_ref.bf16_value(raw_b), 30)[1])
    normed = i8_ref.rms_norm(s, norm, 1e-6)
    rq, rd = i8_ref.quant(normed)
    np.testing.assert_array_equal(q, rq)
    np.testing.assert_array_equal(dv, rd)
    np.testing.assert_array_equal(v, ref.held(normed, 30)[1])
    np.testing.assert_array_equal(yv, i8_ref.product_f32(q, dv, w, scale))
    want, bound = ref.lora(v, ids, slots, yv.astype(np.float64), 30, 0)
    assert (np.abs(zv - want) <= ref.rounded(want, bound, 0)).all()


def test_refusals(ctx, pkg):
    A, N, P = pkg.ArgumentError, pkg.NotSupportedError, pkg.PHX
    for bad in ((1, 0, 4, 8, 8), (1, P.MAX_ADAPTERS + 1, 4, 8, 8), (1, 2, 0, 8, 8), (1, 2, P.MAX_RANK + 1, 8, 8), (1, 2, 4, 0, 8),
                (1, 2, 4, P.MAX_ROWS_I8 + 1, 8), (1, 2, 4, 8, 0), (1, 2, 4, 8, 12), (1, 2, 4, 8, P.MAX_COLS_I8 + 8)):
        with pytest.raises(A):
            ctx.lora_create(*bad)
    for type_ in (0, 8, 24):
        with pytest.raises(N):
            ctx.lora_create(type_, 2, 4, 8, 8)
    h = ctx.lora_create(1, 2, 4, 16, 16)
    try:
        m = np.zeros((16, 16), np.float16)
        at = m.ctypes.data
        for slot, rank, a, b, scale in ((-1, 4, at, at, 1.0), (2, 4, at, at, 1.0), (0, 5, at, at, 1.0), (0, -1, at, at, 1.0), (0, 4, None, at, 1.0),
                                        (0, 4, at, None, 1.0), (0, 4, at + 1, at, 1.0), (0, 4, at, at, np.inf), (0, 4, at, at, np.nan)):
            with pytest.raises(A):
                ctx.lora_set(h, slot, rank, a, b, scale)
        with pytest.raises(A):
            ctx.lora_set(None, 0, 4, at, at)
        with Bufs(ctx) as B:
            x, ids, y_in, y = B.empty(1024).ptr, B.of(np.zeros(8, np.int32)).ptr, B.empty(1024).ptr, B.empty(1024).ptr

            def call(h=h, T=2, x=x, ids=ids, y_type=0, ld=16, y_in=y_in, y=y):
                ctx.lora_add_device(h, T, x, ids, y_type, ld, y_in, y)
            call()
            call(y=y_in)
            for bad in (dict(h=None), dict(T=0), dict(T=P.MAX_ROWS_I8 + 1), dict(ld=15), dict(ld=(1 << 40) + 1), dict(x=None), dict(ids=None),
                        dict(y_in=None), dict(y=None), dict(x=x + 8), dict(ids=ids + 2), dict(y=y + 2), dict(y_in=y_in + 2), dict(x=at),
                        dict(y=at), dict(y=y_in + 16), dict(y=x), dict(y=ids), dict(y_in=at)):
                with pytest.raises(A):
                    call(**bad)
            with pytest.raises(N):
                call(y_type=2)
            ctx.sync()
    finally:
        ctx.lora_free(h)


@pytest.mark.parametrize("n,what", [(5, "the adapters"), (6, "x"), (7, "ids"), (8, "y"), (9, "y_in")])
def test_memory_of_another_gpu(pkg, monkeypatch, n, what):
    """The first five checks are those of a slot being set (its handle, a and b) twice over."""
    monkeypatch.setenv("PHX_FAULT", f"device:{n}")
    with pkg.MoeContext(0) as c:
        h = c.lora_create(1, 2, 4, 8, 8)
        with Bufs(c) as B:
            a = B.of(np.ones((4, 8), np.float16))
            c.lora_set(h, 0, 4, a.ptr, a.ptr)
            c.lora_set(h, 1, 1, np.ones((1, 8), np.float16), np.ones((8, 1), np.float16))  # host memory: the handle alone
            x, ids, y_in, y = B.of(np.ones((2, 8), np.float16)).ptr, B.of(np.ones(2, np.int32)).ptr, B.of(np.ones((2, 8), F32)).ptr, B.empty(64)
            run = lambda: c.lora_add_device(h, 2, x, ids, 0, 8, y_in, y.ptr)  # noqa: E731
            with pytest.raises(pkg.ArgumentError, match=f"{what} is memory of device"):
                run()
            run()
            c.sync()
            assert (y.download((2, 8)) == 9).all()
        c.lora_free(h)


@pytest.mark.parametrize("n,what", enumerate(("the adapters", "a", "b"), 1))
def test_set_memory_of_another_gpu(pkg, monkeypatch, n, what):
    monkeypatch.setenv("PHX_FAULT", f"device:{n}")
    with pkg.MoeContext(0) as c:
        h = c.lora_create(1, 1, 4, 8, 8)
        with Bufs(c) as B:
            a = B.of(np.ones((4, 8), np.float16))
            with pytest.raises(pkg.ArgumentError, match=f"{what} is memory of device"):
                c.lora_set(h, 0, 4, a.ptr, a.ptr)
            c.lora_set(h, 0, 4, a.ptr, a.ptr)
        c.lora_free(h)


def test_allocation_and_launch_faults(pkg, monkeypatch):
    rows, cols, T = 24, 16, 5
    seen = set()
    for spec in [f"malloc:{n}" for n in range(4, 16)] + [f"launch:{n}" for n in range(1, 4)]:
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
                bufs = []
                try:
                    h = c.lora_create(1, 1, 2, rows, cols)
                    c.lora_set(h, 0, 2, np.ones((2, cols), np.float16), np.ones((rows, 2), np.float16), 0.5)
                    for arr in (np.ones((T, cols), np.float16), np.zeros(T, np.int32), np.ones((T, rows), F32)):
                        bufs.append(c.alloc(arr.nbytes))
                        bufs[-1].upload(arr)
                    c.lora_add_device(h, T, bufs[0].ptr, bufs[1].ptr, 0, rows, bufs[2].ptr, bufs[2].ptr)
                    c.sync()
                    got = bufs[2].download((T, rows))
                    break
                except (pkg.OutOfDeviceMemoryError, pkg.GpuDeviceLostError) as e:
                    seen.add(type(e).__name__)
                    assert attempt == 0
            assert (got == 1 + cols).all()
    assert seen == {"OutOfDeviceMemoryError", "GpuDeviceLostError"}
