"""The bits that A x keeps on its way into B's product (phx_lora_add): ranks whose values lie far apart, each brought up again by its
column of B; and arrays that are views."""
import numpy as np
import pytest

import half_ref as ref
from test_gpu_lora import run

pytestmark = pytest.mark.gpu

F32 = np.float32
TYPES = {0: F32, 1: np.float16, 30: np.uint16}


def case(type_, ranks, T, seed):
    """Adapters whose A x takes one product a rank, 11 bits by 11 (8 by 8 with bf16), exact in a float, from 1 down to 2^-15 of
    a row's largest, and whose B brings rank r's value, times 2^(r % 16), to output r alone."""
    rng = np.random.default_rng(seed)
    bits = 10 if type_ == 1 else 7
    mantissa = lambda *s: (1 + rng.integers(0, 1 << bits, s) * 2.0 ** -bits) * rng.choice([-1, 1], s)  # noqa: E731
    order = np.arange(ranks) % 16
    raw_a, a = ref.held(mantissa(ranks, 8) * 2.0 ** -order[:, None], type_)
    raw_b, b = ref.held(np.diag(2.0 ** order), type_)
    x = np.zeros((T, 8))
    x[np.arange(T), np.arange(T) % 8] = mantissa(T)
    raw_x, x = ref.held(x, type_)
    return raw_a, raw_b, raw_x, x @ a.T * 2.0 ** order


@pytest.mark.parametrize("T", [1, 16, 40, 1100])
@pytest.mark.parametrize("ranks", [16, 21, 40])
@pytest.mark.parametrize("type_,y_type", [(1, 0), (1, 1), (1, 30), (30, 0)])
def test_ranks_far_apart(ctx, type_, y_type, ranks, T):
    """The values need 22 bits (16 with bf16), which the terms hold: two of fp16 22, four of bf16 32.  Each output then is one value by
    a power of two, exact in a float, and the result its one rounding."""
    raw_a, raw_b, raw_x, want = case(type_, ranks, T, ranks + T)
    for scale in (1.0, 2.0 ** -20, 2.0 ** 9):
        h = ctx.lora_create(type_, 1, ranks, ranks, 8)
        try:
            ctx.lora_set(h, 0, ranks, raw_a, raw_b, scale)
            y_in = np.zeros((T, ranks), TYPES[y_type])
            got = run(ctx, h, T, raw_x, np.zeros(T, int), y_type, ranks, ranks, y_in)
        finally:
            ctx.lora_free(h)
        np.testing.assert_array_equal(got, ref.held(want * scale, y_type)[1])


def test_values_next_to_the_ends_of_a_float(ctx):
    """A x near the largest and the smallest floats: the scaling leaves no number."""
    for type_, x0, a0, scale in ((1, 2.0 ** 15, 2.0 ** 15, 2.0 ** 97), (1, 2.0 ** -24, 2.0 ** -24, 2.0 ** -78), (1, 2.0 ** -20, 2.0 ** -20, 2.0 ** -100)):
        x, a = np.zeros((3, 8), np.float16), np.zeros((2, 8), np.float16)
        x[:, 0], a[:, 0] = x0, (a0, -a0)
        b = np.eye(2, dtype=np.float16)
        h = ctx.lora_create(type_, 1, 2, 2, 8)
        try:
            ctx.lora_set(h, 0, 2, a, b, scale)
            got = run(ctx, h, 3, x, np.zeros(3, int), 0, 2, 2, np.zeros((3, 2), F32))
        finally:
            ctx.lora_free(h)
        np.testing.assert_array_equal(got, np.tile([x0 * a0 * scale, -x0 * a0 * scale], (3, 1)))


@pytest.mark.parametrize("type_", [1, 30])
def test_views(ctx, type_):
    """Adapters set from transposed views and strided slices are those set from the arrays."""
    rng = np.random.default_rng(type_)
    raw_a, _ = ref.held(rng.standard_normal((12, 72)), type_)
    raw_b, _ = ref.held(rng.standard_normal((40, 12)), type_)
    raw_x, _ = ref.held(rng.standard_normal((5, 72)), type_)
    h = ctx.lora_create(type_, 1, 12, 40, 72)
    try:
        got = []
        for a, b in ((raw_a, raw_b), (np.ascontiguousarray(raw_a.T).T, np.ascontiguousarray(raw_b.T).T), (np.repeat(raw_a, 3, 1)[:, ::3], np.repeat(raw_b, 2, 0)[::2])):
            ctx.lora_set(h, 0, 12, a, b)
            got.append(run(ctx, h, 5, raw_x, np.zeros(5, int), 0, 40, 40, np.zeros((5, 40), F32)))
    finally:
        ctx.lora_free(h)
    for g in got[1:]:
        np.testing.assert_array_equal(g, got[0])
