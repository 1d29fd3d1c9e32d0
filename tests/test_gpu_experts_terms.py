"""The experts' h between the two products (phx_experts_half) is its float value in two terms of the weights' type: results against the
definition in 64 bits with a bound that leaves no room for one rounding of h to 16 bits, on each kernel that takes the terms."""
import numpy as np
import pytest

import half_ref as ref
from test_gpu_half import expert_weights, upload
from test_gpu_i8 import Bufs

pytestmark = pytest.mark.gpu

F32 = np.float32
TERMS = {1: (2.0 ** -22, 2.0 ** -25), 30: (2.0 ** -16, 2.0 ** -134)}  # half a step of the rest's type, twice; near zero


def experts(x, ids, weights, wg, wd, mode, type_):
    """half_ref.experts with h's two terms in place of its one rounding, the second product over twice as many terms."""
    T, d = x.shape
    out, size, err = np.zeros((T, d)), np.zeros((T, d)), np.zeros((T, d))
    rel, least = TERMS[type_]
    for e in range(len(wg)):
        t, j = np.nonzero(ids == e)
        if not len(t):
            continue
        h, dh = ref.gated(mode, x[t], wg[e])
        dh = dh + rel * (np.abs(h) + dh) + least
        size_e = np.abs(h) @ np.abs(wd[e]).T
        dy = ref.sums(2 * h.shape[1]) * size_e + dh @ np.abs(wd[e]).T * (1 + ref.sums(2 * h.shape[1]))
        y, w = h @ wd[e].T, weights[t, j].astype(np.float64)[:, None]
        np.add.at(out, t, y * w)
        np.add.at(size, t, np.abs(y * w))
        np.add.at(err, t, dy * np.abs(w))
    return out, err + (ids.shape[1] + 1) * 2.0 ** -24 * (size + err)


def call(ctx, hs, act, raw_x, ids, weights, out_type, d):
    T, k = ids.shape
    item = 4 if out_type == 0 else 2
    with Bufs(ctx) as B:
        out = B.of(np.full(T * d * item + 64, 0x5A, np.uint8))
        ctx.experts_half_device(*hs, act, T, k, B.of(raw_x).ptr, B.of(ids).ptr, B.of(weights).ptr, out_type, out.ptr)
        ctx.sync()
        assert (out.download((T * d * item + 64,), np.uint8)[T * d * item:] == 0x5A).all()
        return ref.read(out, (T, d), out_type)


# single assignments; lists on the row kernel; on the tile kernel with one tile an expert and several, odd nf and d
@pytest.mark.parametrize("type_,act", [(1, 1), (1, 3), (30, 1), (30, 3)])
@pytest.mark.parametrize("T,k,E,d,nf", [(1, 4, 8, 72, 40), (7, 2, 5, 64, 72), (150, 4, 16, 64, 64), (2000, 2, 3, 136, 104), (1500, 4, 8, 1032, 200), (3000, 8, 12, 520, 72), (4096, 2, 2, 64, 2048)])
def test_values(ctx, T, k, E, d, nf, type_, act):
    print(f"experts_half terms: type {type_} act {act} T {T} k {k} E {E} d {d} nf {nf}", flush=True)
    rng = np.random.default_rng(T + E + d + nf)
    raw, (wg, wd) = expert_weights(rng, E, d, nf, type_)
    raw_x, x = ref.held(rng.standard_normal((T, d)), type_)
    ids = rng.integers(-1, E, (T, k)).astype(np.int32)
    weights = rng.random((T, k)).astype(F32)
    hs = upload(ctx, type_, raw, E, d, nf)
    try:
        got = {t: call(ctx, hs, act, raw_x, ids, weights, t, d) for t in (0, type_)}
    finally:
        for h in hs:
            ctx.weight_free(h)
    want, bound = experts(x, ids, weights, wg, wd, act, type_)
    for t, g in got.items():
        b = ref.rounded(want, bound, t)
        assert (np.abs(g - want) <= b).all(), (np.abs(g - want) / b).max()


@pytest.mark.parametrize("type_", [1, 30])
@pytest.mark.parametrize("T,k,E,d,nf", [(3, 1, 4, 16, 8), (90, 1, 4, 16, 200), (2048, 1, 2, 64, 72), (4096, 1, 8, 512, 64)])
def test_bits_of_h(ctx, T, k, E, d, nf, type_):
    """One channel of h a row, act(g) * u with a gate so large that act(g) = g exactly and a product of 22 bits (16 with bf16), by a power of
    two in Wdown: the result is h's value itself, which the two terms hold whole."""
    rng = np.random.default_rng(T + d + nf)
    bits = 10 if type_ == 1 else 7
    mantissa = lambda *s: 1 + rng.integers(0, 1 << bits, s) * 2.0 ** -bits  # noqa: E731
    g, u = 2.0 ** 5 * mantissa(T), mantissa(T)  # silu(32) = 32 in float: exp(-32) is far under its half step
    e, ch = rng.integers(0, E, T), rng.integers(0, nf, E)
    wg, wd = np.zeros((E, 2 * nf, d)), np.zeros((E, d, nf))
    wg[np.arange(E), ch, 0] = 1
    wg[np.arange(E), nf + ch, d - 1] = 1
    wd[np.arange(E), :, ch] = 2.0 ** (np.arange(d) % 4 - 5)
    raw = ref.held(wg, type_)[0], ref.held(wd, type_)[0]
    x = np.zeros((T, d))
    x[:, 0], x[:, d - 1] = g, u
    raw_x, _ = ref.held(x, type_)
    hs = upload(ctx, type_, raw, E, d, nf)
    try:
        got = call(ctx, hs, 1, raw_x, e[:, None].astype(np.int32), np.ones((T, 1), F32), 0, d)
    finally:
        for h in hs:
            ctx.weight_free(h)
    np.testing.assert_allclose(got, (g * u)[:, None] * 2.0 ** (np.arange(d) % 4 - 5), rtol=2.0 ** -20 if type_ == 1 else 2.0 ** -16, atol=0)


@pytest.mark.parametrize("type_", [1, 30])
@pytest.mark.parametrize("T,E,d,nf", [(3, 4, 16, 40), (300, 4, 64, 72), (4096, 2, 512, 72), (4096, 2, 512, 8)])
def test_infinities_stay_in_their_row(ctx, type_, T, E, d, nf):
    """Rows whose h is infinite or NaN in its first or last channel, beside others of the same expert, where nf is no multiple of the
    kernels' steps."""
    rng = np.random.default_rng(T + nf)
    raw, (wg, wd) = expert_weights(rng, E, d, nf, type_)
    raw_x, x = ref.held(rng.standard_normal((T, d)), type_)
    ids = rng.integers(0, E, (T, 1)).astype(np.int32)
    weights = np.ones((T, 1), F32)
    bad = np.unique([0, 1, T // 2, T - 1])
    raw_x[bad, d - 1] = [{1: [np.inf, np.nan, -np.inf, np.nan], 30: [0x7F80, 0x7FC0, 0xFF80, 0x7FC0]}[type_][i] for i in range(len(bad))]
    hs = upload(ctx, type_, raw, E, d, nf)
    try:
        got = call(ctx, hs, 1, raw_x, ids, weights, 0, d)
    finally:
        for h in hs:
            ctx.weight_free(h)
    fine = np.delete(np.arange(T), bad)
    want, bound = experts(x[fine], ids[fine], weights[fine], wg, wd, 1, type_)
    assert (np.abs(got[fine] - want) <= ref.rounded(want, bound, 0)).all()
    assert not np.isfinite(got[bad]).any()


@pytest.mark.parametrize("type_", [1, 30])
@pytest.mark.parametrize("T,E,d,nf", [(3, 4, 16, 40), (300, 4, 64, 72), (4096, 2, 512, 72)])
def test_an_infinity_in_down_stays_in_its_output(ctx, type_, T, E, d, nf):
    """One value of one expert's Wdown: its output is no number in that expert's rows, everything else as it would be."""
    rng = np.random.default_rng(T + nf)
    raw, (wg, wd) = expert_weights(rng, E, d, nf, type_)
    raw[1][1, 5, nf - 1] = np.inf if type_ == 1 else 0x7F80
    raw_x, x = ref.held(rng.standard_normal((T, d)), type_)
    ids, weights = (np.arange(T) % E).astype(np.int32)[:, None], np.ones((T, 1), F32)
    hs = upload(ctx, type_, raw, E, d, nf)
    try:
        got = call(ctx, hs, 1, raw_x, ids, weights, 0, d)
    finally:
        for h in hs:
            ctx.weight_free(h)
    want, bound = experts(x, ids, weights, wg, wd, 1, type_)
    hit = np.zeros((T, d), bool)
    hit[ids[:, 0] == 1, 5] = True
    assert not np.isfinite(got[hit]).any()
    assert (np.abs(got - want)[~hit] <= ref.rounded(want, bound, 0)[~hit]).all()


def test_fp16_past_its_range(ctx):
    """An h past fp16's numbers is an infinity of its sign, without a NaN from its second term."""
    x = np.zeros((2, 8), np.float16)
    x[:, 0] = 1000
    w = np.zeros((1, 16, 8), np.float16)
    w[0, 0, 0], w[0, 8, 0] = 1, 1
    down = np.zeros((1, 8, 8), np.float16)
    down[0, :, 0] = [1, -1, 2, -2, 1, -1, 2, -2]
    hs = upload(ctx, 1, (w, down), 1, 8, 8)
    try:
        for T in (1, 2):
            got = call(ctx, hs, 1, x[:T], np.zeros((T, 1), np.int32), np.ones((T, 1), F32), 0, 8)
            np.testing.assert_array_equal(got, np.tile([np.inf, -np.inf], (T, 4)))
    finally:
        for h in hs:
            ctx.weight_free(h)
