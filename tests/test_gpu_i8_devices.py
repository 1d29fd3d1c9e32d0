"""The routing and int8 entry points refuse memory and weight handles of another GPU before anything is launched.  The
library's fault plan (PHX_FAULT=device:n, read when a context is created) has the n-th buffer or handle of a context that is
checked taken for another GPU's: that call raises, and the same call then runs."""
import numpy as np
import pytest

import i8_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture
def planned(pkg, monkeypatch):
    """planned(n): a context that takes the n-th checked buffer or handle for another GPU's."""
    made = []

    def make(n):
        monkeypatch.setenv("PHX_FAULT", f"device:{n}")
        made.append(pkg.MoeContext(0))
        monkeypatch.delenv("PHX_FAULT")
        return made[-1]
    yield make
    for c in made:
        c.close()


def refused_once(pkg, what, call):
    """call() raises, naming `what`, and then does not."""
    with pytest.raises(pkg.ArgumentError, match=f"{what} is memory of device"):
        call()
    return call()


@pytest.mark.parametrize("n,what", [(1, "w"), (2, "scale")])
def test_upload(pkg, planned, n, what):
    w, scale = ref.weights_of(np.random.default_rng(1), 64, 96)
    c = planned(n)
    bw, bs = c.alloc(w.nbytes), c.alloc(scale.nbytes)
    bw.upload(w)
    bs.upload(scale)
    c.weight_free(c.weight_upload_i8(1, 64, 96, w, scale))  # host memory: nothing to check
    h = refused_once(pkg, what, lambda: c.weight_upload_i8(1, 64, 96, bw.ptr, bs.ptr))
    xq, xd = ref.rows_of(np.random.default_rng(2), 3, 96)
    got = c.MatMulI8(h, 64, 96, xq, xd)
    np.testing.assert_array_equal(got, ref.product_f32(xq, xd, w, scale))
    c.weight_free(h)
    bw.free()
    bs.free()


@pytest.mark.parametrize("n,what", enumerate(("the weight", "xq", "xd", "y"), 1))
def test_product(pkg, planned, n, what):
    w, scale = ref.weights_of(np.random.default_rng(1), 64, 96)
    xq, xd = ref.rows_of(np.random.default_rng(2), 3, 96)
    c = planned(n)
    h = c.weight_upload_i8(1, 64, 96, w, scale)
    got = refused_once(pkg, what, lambda: c.MatMulI8(h, 64, 96, xq, xd))
    np.testing.assert_array_equal(got, ref.product_f32(xq, xd, w, scale))
    c.weight_free(h)


@pytest.mark.parametrize("n,what", enumerate(("gate_up", "down", "xq", "xd", "ids", "weights", "out"), 1))
def test_experts(pkg, planned, n, what):
    rng = np.random.default_rng(3)
    wg, sg = ref.weights_of(rng, 2, 64, 32)
    wd, sd = ref.weights_of(rng, 2, 32, 32)
    xq, xd = ref.rows_of(rng, 3, 32)
    ids, weights = np.full((3, 1), -1, np.int32), np.ones((3, 1), np.float32)
    c = planned(n)
    hs = c.weight_upload_i8(2, 64, 32, wg, sg, paired=True), c.weight_upload_i8(2, 32, 32, wd, sd)
    assert (refused_once(pkg, what, lambda: c.ExpertsI8(*hs, 1, xq, xd, ids, weights)) == 0).all()
    for h in hs:
        c.weight_free(h)


@pytest.mark.parametrize("n,what", enumerate(("logits", "ids", "weights", "bias"), 1))
def test_route(pkg, planned, n, what):
    D = pkg.RouteDesc(8, 2)
    logits, bias = np.random.default_rng(4).standard_normal((5, 8)).astype(np.float32), np.zeros(8, np.float32)
    c = planned(n)
    ids, _ = refused_once(pkg, what, lambda: c.Route(D, logits, bias))
    np.testing.assert_array_equal(ids, ref.route(D, logits, bias)[0])


@pytest.mark.parametrize("n,what", enumerate(("x", "qs", "d", "aux"), 1))
def test_rows(pkg, planned, n, what):
    x, aux = (np.random.default_rng(5).standard_normal((2, 64)).astype(np.float32) for _ in range(2))
    c = planned(n)
    q, d = refused_once(pkg, what, lambda: c.QuantI8(pkg.PHX.QUANT_SILU_MUL, x, aux))
    assert q.shape == (2, 64) and np.isfinite(d).all()
