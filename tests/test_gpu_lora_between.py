"""phx_lora_add from one section of a wide matrix into another (rows of y between those of y_in), and what of it is refused."""
import numpy as np
import pytest

import half_ref as ref
from test_gpu_i8 import Bufs
from test_gpu_lora import adapters

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [1, 2, 37, 1100])
@pytest.mark.parametrize("rows,ld,start,to", [(64, 128, 0, 64), (64, 128, 64, 0), (70, 200, 3, 130), (70, 140, 70, 0), (96, 400, 304, 8)])
@pytest.mark.parametrize("y_type", [0, 1, 30])
def test_two_sections_of_one_matrix(ctx, y_type, rows, ld, start, to, T):
    print(f"lora between: y {y_type} T {T} rows {rows} ld {ld} from {start} to {to}", flush=True)
    rng = np.random.default_rng(T + rows + ld)
    type_ = 30 if y_type == 30 else 1
    item = 4 if y_type == 0 else 2
    h, slots = adapters(ctx, rng, type_, 4, 20, rows, 40, {0: 20, 2: 3})
    raw_x, x = ref.held(rng.standard_normal((T, 40)), type_)
    raw, whole = ref.held(rng.standard_normal((T, ld)), y_type)
    ids = rng.integers(-1, 4, T).astype(np.int32)
    try:
        with Bufs(ctx) as B:
            m = B.of(raw)
            ctx.lora_add_device(h, T, B.of(raw_x).ptr, B.of(ids).ptr, y_type, ld, m.ptr + start * item, m.ptr + to * item)
            ctx.sync()
            got = ref.read(m, (T, ld), y_type)
    finally:
        ctx.lora_free(h)
    beside = np.ones(ld, bool)
    beside[to:to + rows] = False
    np.testing.assert_array_equal(got[:, beside], whole[:, beside])
    want, bound = ref.lora(x, ids, slots, whole[:, start:start + rows].copy(), type_, y_type)
    bare = ~np.isin(ids, list(slots))
    np.testing.assert_array_equal(got[bare, to:to + rows], whole[bare, start:start + rows])
    assert (np.abs(got[:, to:to + rows] - want) <= ref.rounded(want, bound, y_type)).all()


def test_sections_that_meet_are_refused(ctx, pkg):
    rows, ld, T = 16, 48, 4
    h = ctx.lora_create(1, 1, 4, rows, 16)
    try:
        with Bufs(ctx) as B:
            m, x, ids = B.empty(2 * T * ld * 4), B.empty(T * 16 * 2), B.of(np.zeros(T, np.int32))
            base = m.ptr

            def call(start, to, ld=ld):
                ctx.lora_add_device(h, T, x.ptr, ids.ptr, 0, ld, base + 4 * start, base + 4 * to)
            for start, to in ((0, 15), (15, 0), (0, 33), (33, 0), (0, 1), (0, ld), (ld, 0), (0, ld + 15), (0, ld + 33), (2 * ld + 33, 0)):
                with pytest.raises(pkg.ArgumentError, match="overlaps"):
                    call(start, to)
            with pytest.raises(pkg.ArgumentError, match="overlaps"):
                call(0, 16, ld=31)
            for start, to in ((0, 16), (0, 32), (32, 0), (16, 32), (0, ld + 16), (2 * ld + 32, 0), (0, T * ld), (5, 5)):
                call(start, to)
            call(0, 16, ld=32)
            ctx.sync()
    finally:
        ctx.lora_free(h)


@pytest.mark.parametrize("n,what", [(2, "x"), (3, "ids"), (4, "y"), (5, "y_in")])
def test_memory_of_another_gpu(pkg, monkeypatch, n, what):
    """The first check is the handle's."""
    monkeypatch.setenv("PHX_FAULT", f"device:{n}")
    with pkg.MoeContext(0) as c:
        h = c.lora_create(1, 1, 4, 8, 8)
        with Bufs(c) as B:
            m, x, ids = B.empty(2 * 16 * 4), B.empty(32).ptr, B.of(np.zeros(2, np.int32)).ptr
            call = lambda: c.lora_add_device(h, 2, x, ids, 0, 16, m.ptr, m.ptr + 32)  # noqa: E731
            with pytest.raises(pkg.ArgumentError, match=f"{what} is memory of device"):
                call()
            call()
            c.sync()
        c.lora_free(h)
