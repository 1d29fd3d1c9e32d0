"""Products with fp16 / bf16 matrices, adapters and the residual's norm from their definitions (include/phx_moe.h), in numpy's
64 bits, each with a bound on what 32-bit sums and the named roundings may differ by."""
import numpy as np

import i8_ref as ref

F32 = np.float32
STEP = {0: 2.0 ** -24, 1: 2.0 ** -11, 30: 2.0 ** -8}  # half a step, relative: float32, fp16, bf16
TINY = {0: 2.0 ** -150, 1: 2.0 ** -25, 30: 2.0 ** -134}  # half a step of the subnormal numbers


def held(v, type_):
    """float32 values in a type as the library takes them, and the values they then have (float64)."""
    v = np.ascontiguousarray(v, F32)
    if type_ == 1:
        h = v.astype(np.float16)
        return h, h.astype(np.float64)
    if type_ == 30:
        h = ref.bf16_bits(v)
        return h, ref.bf16_value(h).astype(np.float64)
    return v, v.astype(np.float64)


def read(buf, shape, type_):
    if type_ == 30:
        return ref.bf16_value(buf.download(shape, np.uint16)).astype(np.float64)
    return buf.download(shape, F32 if type_ == 0 else np.float16).astype(np.float64)


def sums(K):
    """What a sum of K products in 32 bits may be off by, relative to the terms' magnitudes: a step (not half: the matrix cores
    need not round to nearest) for each addition."""
    return (K + 8) * 2.0 ** -23


def product(x, w):
    """x w^T and its bound."""
    return x @ w.T, sums(x.shape[1]) * (np.abs(x) @ np.abs(w).T)


def act(mode, g):
    with np.errstate(over="ignore", invalid="ignore"):
        z = g if mode == 1 else 2 * np.sqrt(2 / np.pi) * (g + 0.044715 * g ** 3)
        return np.where(z < -700, 0.0, g / (1 + np.exp(-np.maximum(z, -700))))


def gated(mode, x, w):
    """act(gate) * up of paired rows, and its bound: both activations' slopes are under 1.13; their own roundings (z's, the
    exponential's argument and value, the quotient, the product) under 16 half steps of the value, |z| <= 88 magnifying the
    argument's by itself (2^-24 of z in exp(z): 88 half steps where the value is that of a tail)."""
    nf = w.shape[0] // 2
    (g, dg), (u, du) = product(x, w[:nf]), product(x, w[nf:])
    a = act(mode, g)
    h = a * u
    tail = np.where(g < 0, np.minimum(np.abs(g) * (1 if mode == 1 else 2 + g * g), 88.0), 1.0)
    slope = np.where(np.isfinite(g), 1.13, 0.0)
    return h, slope * dg * (np.abs(u) + du) + np.abs(a) * du + (16 + 4 * tail) * 2.0 ** -24 * np.abs(h) + 1e-35 * (1 + np.abs(u))


def rounded(v, bound, type_):
    """The bound of a value known to `bound`, once rounded to a type."""
    return bound + STEP[type_] * (np.abs(v) + bound) + TINY[type_]


def experts(x, ids, weights, wg, wd, mode, type_):
    """The experts' FFN and its bound (before the output's rounding): h rounded to the weights' type, k float products and
    additions a row."""
    T, d = x.shape
    out, size, err = np.zeros((T, d)), np.zeros((T, d)), np.zeros((T, d))
    for e in range(len(wg)):
        t, j = np.nonzero(ids == e)
        if not len(t):
            continue
        h, dh = gated(mode, x[t], wg[e])
        dh = rounded(h, dh, type_)
        y, dy = product(h, wd[e])
        dy = dy + dh @ np.abs(wd[e]).T * (1 + sums(h.shape[1]))
        w = weights[t, j].astype(np.float64)[:, None]
        np.add.at(out, t, y * w)
        np.add.at(size, t, np.abs(y * w))
        np.add.at(err, t, dy * np.abs(w))
    return out, err + (ids.shape[1] + 1) * 2.0 ** -24 * (size + err)


def lora(x, ids, slots, y_in, type_, y_type):
    """y_in + scale B A x for slots {number: (A, B, scale)}, and its bound before the output's rounding: A's sums, the scale's
    product, the value's terms (two, or four where y is float, each a half step of the type of the rest; and under 2^-24
    of a row's largest), B's sums of at most eight times the ranks, the addition."""
    y, err = y_in.copy(), np.zeros_like(y_in)
    terms = STEP[type_] ** (4 if y_type == 0 else 2)
    for s, (a, b, scale) in slots.items():
        t = np.nonzero(ids == s)[0]
        if not len(t) or not len(a):
            continue
        low, dl = product(x[t], a)
        low, dl = low * scale, (dl + 8 * 2.0 ** -24 * np.abs(low)) * abs(scale) + 2.0 ** -24 * np.abs(low * scale)
        dl = dl + terms * (np.abs(low) + dl) + 2.0 ** -24 * np.abs(low).max(axis=1, keepdims=True)
        y[t] += low @ b.T
        err[t] = (dl + sums(8 * len(a)) * np.abs(low)) @ np.abs(b).T + 2.0 ** -24 * (np.abs(y_in[t]) + np.abs(low) @ np.abs(b).T)
    return y, err
