"""Routing to experts (phx_route, phx_route_check): refusals and the descriptor's layout on the CPU; ids equal to the
plain implementation's in 64 bits (tests/i8_ref.py) and weights within one float32 rounding of it on the GPU, at the
ties, masks, empty rows and sizes where a selection goes wrong."""
import ctypes as C
import subprocess
from pathlib import Path

import numpy as np
import pytest

import i8_ref as ref

ROOT = Path(__file__).resolve().parent.parent
NINF = -np.inf


def desc(pkg, **kw):
    return pkg.RouteDesc(**{**dict(n_expert=128, n_used=8), **kw})


# ---------------------------------------------------------------------------------------- CPU
def test_desc_layout_matches_c(tmp_path, pkg):
    fields = [f for f, _ in pkg.RouteDesc._fields_]
    prog = ['#include <stdio.h>', '#include <stddef.h>', '#include "phx_moe.h"', "int main(void) {",
            '  printf("%zu\\n", sizeof(phx_route_desc));']
    prog += [f'  printf("%zu\\n", offsetof(phx_route_desc, {f}));' for f in fields]
    (tmp_path / "r.c").write_text("\n".join(prog + ["  return 0;", "}"]))
    exe = tmp_path / "r"
    subprocess.run(["gcc", "-std=c99", f"-I{ROOT / 'include'}", "-o", str(exe), str(tmp_path / "r.c")], check=True)
    vals = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert vals == [C.sizeof(pkg.RouteDesc)] + [getattr(pkg.RouteDesc, f).offset for f in fields]


def test_constants_match_header(pkg):
    text = (ROOT / "include" / "phx_moe.h").read_text()
    P = pkg.PHX
    for name, value in (("F16", P.F16), ("BF16", P.BF16), ("SCORE_SOFTMAX", P.SCORE_SOFTMAX),
                        ("SCORE_SIGMOID", P.SCORE_SIGMOID), ("GROUP_MAX", P.GROUP_MAX), ("GROUP_TOP2", P.GROUP_TOP2),
                        ("MAX_GROUPS", P.MAX_GROUPS)):
        assert f"#define PHX_{name} {value}" in text, name


@pytest.mark.parametrize("kw", [
    {}, dict(n_expert=1, n_used=1), dict(n_expert=256, n_used=16), dict(n_group=8, n_group_used=4, group_score=1),
    dict(n_expert=64, n_group=64, n_group_used=8), dict(score=1, renorm=0, logits_type=30, scale=2.5),
    dict(n_expert=250, n_group=25, n_group_used=1, n_used=10),
])
def test_check_accepts(pkg, kw):
    desc(pkg, **kw).check()


@pytest.mark.parametrize("kw,code", [
    (dict(n_expert=0), "ERR_ARG"), (dict(n_used=0), "ERR_ARG"), (dict(n_group=0), "ERR_ARG"), (dict(n_group_used=0), "ERR_ARG"),
    (dict(n_expert=257), "ERR_UNSUPPORTED"), (dict(n_used=17), "ERR_UNSUPPORTED"),
    (dict(n_group=128, n_group_used=64), "ERR_UNSUPPORTED"), (dict(n_expert=4, n_used=5), "ERR_ARG"),
    (dict(n_group=3), "ERR_ARG"), (dict(n_group=8, n_group_used=9), "ERR_ARG"),
    (dict(n_group=32, n_group_used=1), "ERR_ARG"),  # one group of four holds fewer than eight experts
    (dict(score=2), "ERR_ARG"), (dict(group_score=-1), "ERR_ARG"), (dict(renorm=2), "ERR_ARG"),
    (dict(logits_type=8), "ERR_UNSUPPORTED"), (dict(scale=float("nan")), "ERR_ARG"), (dict(scale=float("inf")), "ERR_ARG"),
])
def test_check_refuses(pkg, kw, code):
    with pytest.raises(pkg.MoeError) as e:
        desc(pkg, **kw).check()
    assert e.value.code == getattr(pkg.PHX, code)


def test_check_null(pkg):
    assert pkg.load_lib().phx_route_check(None) == pkg.PHX.ERR_ARG


# ---------------------------------------------------------------------------------------- GPU
def held(pkg, type_, v):
    """float32 logits in the type a call takes, and the values they then have."""
    if type_ == pkg.PHX.F16:
        h = v.astype(np.float16)
        return h, h.astype(np.float32)
    if type_ == pkg.PHX.BF16:
        h = ref.bf16_bits(v)
        return h, ref.bf16_value(h)
    return v, v


def agree(ctx, pkg, D, logits, bias=None):
    print("route:", {f: getattr(D, f) for f, _ in D._fields_}, logits.shape, bias is not None, flush=True)
    got, values = held(pkg, D.logits_type, logits)
    ids, w = ctx.Route(D, got, bias)
    rids, rw = ref.route(D, values, bias)
    np.testing.assert_array_equal(ids, rids)
    # doubles to within a few of their own steps, then one rounding to float32 (2^-24; half a step of the smallest
    # where the value is below the normal numbers)
    assert (np.abs(w - rw) <= np.maximum(1.001 * 2.0 ** -24 * np.abs(rw), 2.0 ** -150)).all()
    return ids, w


SHAPES = [(1, 1, 1), (3, 8, 2), (2, 20, 16), (5, 63, 7), (67, 64, 4), (4, 65, 8), (129, 128, 8), (6, 250, 10), (33, 256, 16)]


@pytest.mark.gpu
@pytest.mark.parametrize("score", [0, 1])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("type_", [0, 1, 30])
@pytest.mark.parametrize("shape", SHAPES)
def test_route(ctx, pkg, shape, type_, with_bias, score):
    T, E, k = shape
    rng = np.random.default_rng(T * 1000 + E + 7 * type_ + score)
    logits = (2 * rng.standard_normal((T, E))).astype(np.float32)
    bias = (0.2 * rng.standard_normal(E)).astype(np.float32) if with_bias else None
    for renorm in (0, 1):
        agree(ctx, pkg, desc(pkg, n_expert=E, n_used=k, score=score, logits_type=type_, renorm=renorm, scale=2.5), logits, bias)


@pytest.mark.gpu
@pytest.mark.parametrize("score", [0, 1])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("group_score", [0, 1])
@pytest.mark.parametrize("groups", [(256, 8, 4, 8), (256, 64, 7, 5), (60, 5, 2, 6), (250, 25, 3, 10), (64, 64, 9, 9), (96, 2, 1, 16),
                                    (24, 3, 1, 8)])
def test_groups(ctx, pkg, groups, group_score, with_bias, score):
    E, G, used, k = groups
    rng = np.random.default_rng(E + G + group_score)
    for type_ in (0, 30):  # bf16: many equal logits, so groups and experts tie
        logits = (1.5 * rng.standard_normal((37, E))).astype(np.float32)
        logits[3] = np.round(logits[3])
        logits[4] = 0.5
        logits[5, : E // 2] = NINF
        bias = (0.1 * rng.integers(-3, 4, E)).astype(np.float32) if with_bias else None
        agree(ctx, pkg, desc(pkg, n_expert=E, n_used=k, score=score, n_group=G, n_group_used=used, group_score=group_score,
                             logits_type=type_), logits, bias)


@pytest.mark.gpu
@pytest.mark.parametrize("score", [0, 1])
@pytest.mark.parametrize("groups", [(1, 1), (4, 2), (4, 4)])
@pytest.mark.parametrize("with_bias", [False, True])
def test_ties_and_masks(ctx, pkg, with_bias, groups, score):
    E, k = 32, 6
    rng = np.random.default_rng(11)
    rows = [np.zeros(E), np.tile([1.0, 2.0], E // 2), np.full(E, NINF), np.full(E, -3.4028235e38), np.full(E, 3.4028235e38),
            np.full(E, np.inf), np.full(E, np.nan), np.full(E, -200.0), np.full(E, 200.0)]
    for few in (0, 1, k - 1, k):  # candidates left
        r = np.full(E, NINF)
        r[rng.permutation(E)[:few]] = rng.standard_normal(few)
        rows.append(r)
    lowest = rng.standard_normal(E)
    lowest[3:] = -3.4028235e38  # masked by the type's lowest value: a candidate with no weight
    mixed = rng.standard_normal(E)
    mixed[[0, 5, 31]] = np.nan, np.inf, NINF
    zeros = np.where(np.arange(E) % 2, 0.0, -0.0)
    rows += [lowest, mixed, zeros, np.where(np.arange(E) % 3, 40.0, 41.0), np.where(np.arange(E) == 9, -np.inf, np.inf)]
    logits = np.array(rows, np.float32)
    bias = None
    if with_bias:
        bias = (0.5 * rng.integers(-2, 3, E)).astype(np.float32)
        bias[[1, 8, 17]] = NINF, np.nan, np.inf
    for renorm in (0, 1):
        for gs in (0, 1):
            D = desc(pkg, n_expert=E, n_used=k, score=score, n_group=groups[0], n_group_used=groups[1], group_score=gs, renorm=renorm)
            ids, w = agree(ctx, pkg, D, logits, bias)
            assert (w[ids < 0] == 0).all() and np.isfinite(w).all()
            assert (ids[2] == -1).all() and (ids[6] == -1).all()


@pytest.mark.gpu
def test_long_batch_and_all_experts(ctx, pkg):
    rng = np.random.default_rng(3)
    D = desc(pkg, n_expert=16, n_used=16)
    ids, w = agree(ctx, pkg, D, rng.standard_normal((4099, 16)).astype(np.float32))
    assert (np.sort(ids, 1) == np.arange(16)).all()
    np.testing.assert_allclose(w.astype(np.float64).sum(1), 1.0, atol=16 * 2.0 ** -24)


@pytest.mark.gpu
def test_rows_past_the_call_stay(ctx, pkg):
    """Buffers longer than T rows keep what is behind them."""
    D = desc(pkg, n_expert=40, n_used=3)
    lg = np.random.default_rng(5).standard_normal((8, 40)).astype(np.float32)
    bufs = [ctx.alloc(n) for n in (lg.nbytes, 8 * 12, 8 * 12)]
    try:
        bufs[0].upload(lg)
        for b in bufs[1:]:
            b.upload(np.full(24, 77, np.int32))
        ctx.route_device(D, 5, bufs[0].ptr, None, bufs[1].ptr, bufs[2].ptr)
        ctx.sync()
        ids = bufs[1].download((8, 3), np.int32)
        np.testing.assert_array_equal(ids[:5], ref.route(D, lg[:5])[0])
        assert (ids[5:] == 77).all() and (bufs[2].download((8, 3), np.int32)[5:] == 77).all()
    finally:
        for b in bufs:
            b.free()


@pytest.mark.gpu
def test_route_refuses(ctx, pkg):
    D = desc(pkg, n_expert=8, n_used=2)
    a, b = ctx.alloc(4096), ctx.alloc(4096)
    host = np.zeros(64, np.float32)
    try:
        ok = (D, 4, a.ptr, None, b.ptr, b.ptr + 1024)
        ctx.route_device(*ok)
        for i, v in ((1, 0), (1, -1), (1, (1 << 20) + 1), (2, None), (2, a.ptr + 2), (2, host.ctypes.data), (3, a.ptr + 1),
                     (4, None), (4, b.ptr + 1024), (4, a.ptr + 64), (5, b.ptr + 4), (5, host.ctypes.data)):
            bad = list(ok)
            bad[i] = v
            with pytest.raises(pkg.ArgumentError):
                ctx.route_device(*bad)
        with pytest.raises(pkg.NotSupportedError):
            ctx.route_device(desc(pkg, n_expert=300), *ok[1:])
        with pytest.raises(pkg.ArgumentError):
            ctx.Route(D, np.zeros((2, 9), np.float32))
        ctx.route_device(*ok)  # the context still works
        ctx.sync()
    finally:
        a.free()
        b.free()
