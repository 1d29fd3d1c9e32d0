"""Routing and int8 products from their definitions (include/phx_moe.h), in numpy: scores, sums and comparisons in 64
bits, the float32 roundings that a definition names taken where it names them."""
import numpy as np

F32 = np.float32
FLT_MAX, FLT_MIN = np.finfo(F32).max, np.finfo(F32).tiny


def bf16_bits(v):
    """float32 values as bf16 bits, to nearest even (no NaN)."""
    b = np.ascontiguousarray(v, F32).view(np.uint32)
    return ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)


def bf16_value(h):
    return (h.astype(np.uint32) << 16).view(F32)


def first_largest(v):
    """The lowest index of the largest value of a list without NaN."""
    return max(range(len(v)), key=lambda i: (v[i], -i))


def route(D, logits, bias=None):
    """ids and weights (float64) of float32 logits, token by token and place by place."""
    E, k, G = D.n_expert, D.n_used, D.n_group
    ids = np.full((len(logits), k), -1, np.int32)
    w = np.zeros((len(logits), k))
    for t, row in enumerate(np.asarray(logits, np.float64)):
        able = row > -np.inf
        l = np.where(able, np.minimum(row, float(FLT_MAX)), -np.inf)  # noqa: E741
        s = np.zeros(E)
        if able.any():
            with np.errstate(over="ignore"):
                if D.score == 0:
                    s[able] = np.exp(l[able] - l[able].max())
                    s /= s.sum()
                else:
                    s[able] = 1.0 / (1.0 + np.exp(-l[able]))
        c, key = s.copy(), l.copy()
        if bias is not None:
            b = np.asarray(bias, np.float64)
            able = able & (b > -np.inf)
            with np.errstate(invalid="ignore"):
                c = key = s + b
        c, key = np.where(able, c, -np.inf), np.where(able, key, -np.inf)
        if D.n_group_used < G:
            value = []
            for g in range(G):
                a = slice(g * (E // G), (g + 1) * (E // G))
                two = sorted(v for v in c[a] if v > -np.inf)[-2:]
                value.append(key[a].max() if D.group_score == 0 else sum(two) if two else -np.inf)
            kept = []
            for _ in range(D.n_group_used):
                kept.append(first_largest([-np.inf if g in kept else v for g, v in enumerate(value)])
                            if max(v for g, v in enumerate(value) if g not in kept) > -np.inf
                            else min(g for g in range(G) if g not in kept))
            for g in range(G):
                if g not in kept:
                    key[g * (E // G):(g + 1) * (E // G)] = -np.inf
        for j in range(k):
            e = first_largest(key)
            if key[e] == -np.inf:
                break
            ids[t, j], w[t, j] = e, s[e]
            key[e] = -np.inf
        if D.renorm:
            total = w[t].sum()
            w[t] = w[t] / total if total > 0 else 0.0
        w[t] *= float(F32(D.scale))
    return ids, w


def quant(v):
    """int8 rows and scales of float32 rows v."""
    v = np.asarray(v, F32)
    amax = np.abs(v).max(axis=1)
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        d = (amax / F32(127)).astype(F32)
        d = np.where(d >= FLT_MIN, d, F32(0))
        inv = np.where(d > 0, F32(1) / d, F32(0)).astype(F32)
        r = (v * inv[:, None]).astype(F32).astype(np.float64)
        q = np.clip(np.sign(r) * np.floor(np.abs(r) + 0.5), -127, 127)
    bad = ~np.isfinite(v).all(axis=1)
    q[bad], d[bad] = 0, np.nan
    return q.astype(np.int8), d


def rms_norm(x, w, eps):
    x = np.asarray(x, F32)
    mean = (x.astype(np.float64) ** 2).mean(axis=1).astype(F32)
    scale = (F32(1) / np.sqrt((mean + F32(eps)).astype(F32).astype(np.float64)).astype(F32)).astype(F32)
    return ((x * scale[:, None]).astype(F32) * np.asarray(w, F32)).astype(F32)


def sums(xq, w):
    """The whole-number sums, exact in float64."""
    return xq.astype(np.float64) @ w.astype(np.float64).T


def product(xq, xd, w, scale):
    """float64 of phx_matmul_i8's sum times the two scales."""
    return sums(xq, w) * xd.astype(np.float64)[:, None] * scale.astype(np.float64)


def product_f32(xq, xd, w, scale):
    """phx_matmul_i8's float value: one rounding of the sum, one of the scales' product, one of the value."""
    i = sums(xq, w).astype(F32)
    return (i * (xd.astype(F32)[:, None] * scale.astype(F32)).astype(F32)).astype(F32)


def experts(xq, xd, ids, weights, wg, sg, wd, sd, act):
    """(float64 sums, sums of the terms' magnitudes) of the experts' FFN; act maps float32 to float32."""
    T, d = xq.shape
    E, nf = wg.shape[0], wg.shape[1] // 2
    out, size = np.zeros((T, d)), np.zeros((T, d))
    for e in range(E):
        t, j = np.nonzero(ids == e)
        if not len(t):
            continue
        gu = product_f32(xq[t], xd[t], wg[e], sg[e])
        q, dh = quant((act(gu[:, :nf]) * gu[:, nf:]).astype(F32))
        y = product(q, dh, wd[e], sd[e]) * weights[t, j].astype(np.float64)[:, None]
        np.add.at(out, t, y)
        np.add.at(size, t, np.abs(y))
    return out, size


def weights_of(rng, *shape):
    """int8 matrices over the whole range, -128 among them, and their scales."""
    w = np.clip(np.rint(rng.standard_normal(shape) * 40), -128, 127).astype(np.int8)
    w[..., 0, :3] = -128, 127, -128
    return w, (6e-4 * (1 + 0.3 * rng.random(shape[:-1]))).astype(F32)


def rows_of(rng, T, cols):
    return quant(rng.standard_normal((T, cols)).astype(F32))
