"""The activations of the int8 experts' epilogues, bit for bit the library's silu and gelu, the signs of zeros among them.  The
library's gelu is its table (selftest 6): where fp16 rounds a value above -10 to -10 the table has 0, the formula -0."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

F32 = np.float32


def values():
    rng = np.random.default_rng(21)
    every = np.arange(65536, dtype=np.uint16).view(np.float16).astype(F32)
    bits = rng.integers(0, 1 << 32, 1 << 20, dtype=np.uint32).view(F32)  # every exponent, denormals too
    small = (2.0 ** rng.uniform(-149, -60, 1 << 14)).astype(F32)
    v = np.concatenate([every, bits, small, -small, rng.uniform(-90, 90, 1 << 18).astype(F32),
                        np.array([0.0, -0.0, 1e-45, -1e-45, 79.99999, -79.99999, -103.9, np.inf, -np.inf], F32)])
    return v[~np.isnan(v)]


def same_bits(got, want):
    nan = np.isnan(want)
    np.testing.assert_array_equal(np.isnan(got), nan)
    np.testing.assert_array_equal(got[~nan].view(np.uint32), want[~nan].view(np.uint32))


def test_silu_bits(ctx, orc):
    v = values()
    with np.errstate(all="ignore"):
        same_bits(ctx.selftest(11, v, np.ones_like(v)), orc.silu(v))


def test_gelu_bits(ctx, orc):
    v = values()
    one = np.ones_like(v)
    table = ctx.selftest(6, v, one)
    same_bits(ctx.selftest(12, v, one), table)
    np.testing.assert_array_equal(table, orc.gelu(v))
