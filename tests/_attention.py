"""Attention over a band in 64 bits with numpy, and how far a result in fewer may be from it.

``u`` is the largest relative error of one rounding to the panels' type.  The kernels round the
weights P (and dS) once for the second product and the result once at the end; everything between
is in 32 bits, whose share, ``c`` times the sum of magnitudes, counts some hundred roundings of
2^-24 and the error of a 32-bit score in the exponential."""
import numpy as np

U = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
# half of the type's smallest spacing: what one rounding may be off below its normal range
TINY = {"f32": 1e-30, "bf16": 1e-30, "f16": 2.0 ** -25}


def to_bits(x, dtype):
    """float32 / 64 array -> what a panel of that type is uploaded from (rounded to nearest even)."""
    x = np.ascontiguousarray(x, dtype=np.float32)
    if dtype == "f32":
        return x
    if dtype == "f16":
        return x.astype(np.float16)
    b = x.view(np.uint32)
    r = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def from_bits(b, dtype):
    if dtype == "bf16":
        return (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return b.astype(np.float64)


def visible(rows, cols, window, sinks):
    p = (cols - rows + np.arange(rows))[:, None]
    c = np.arange(cols)[None, :]
    see = c <= p
    if window:
        see &= (p - c < window) | (c < sinks)
    return see


def softmax(s, see):
    s = np.where(see, s, -np.inf)
    with np.errstate(divide="ignore"):
        top = np.max(s, axis=1, initial=-np.inf, keepdims=True)
        e = np.where(see, np.exp(s - np.where(np.isinf(top), 0.0, top)), 0.0)
        total = e.sum(1, keepdims=True)
        lse = np.where(np.isinf(top), 0.0, top) + np.log(total)
    return e / np.where(total == 0, 1.0, total), lse[:, 0]


def band(q, k, v, rows, cols, window, sinks, scale, dtype, d_o=None, o_in=None):
    """q [T, H, D], k / v [S, G, D], all float64 holding the panels' values.  Returns a dict of
    (value, bound) for o, lse and, with d_o (and the o that the gradient call was given), dq, dk, dv."""
    tiny = TINY[dtype]
    u, H, G, D = U[dtype], q.shape[1], k.shape[1], q.shape[2]
    z = {n: np.zeros_like(x) for n, x in (("o", q), ("dq", q), ("dk", k), ("dv", v))}
    e = {n: np.zeros_like(x) for n, x in z.items()}
    lse, lse_e = np.full((q.shape[0], H), -np.inf), np.zeros((q.shape[0], H))
    r0 = c0 = 0
    for n, m in zip(rows, cols):
        see = visible(n, m, window, sinks)
        for h in range(H):
            r, c, g = slice(r0, r0 + n), slice(c0, c0 + m), h // (H // G)
            Q, K, V = q[r, h], k[c, g], v[c, g]
            s = scale * (Q @ K.T)
            sabs = scale * (np.abs(Q) @ np.abs(K).T)
            P, l = softmax(s, see)
            lse[r, h] = l
            # 32 bits: a score's error times its weight, some roundings of the sums
            ce = np.where(see, 2.0 ** -24 * (D + 8) * sabs, 0.0).max(1, initial=0.0, keepdims=True)
            c32 = 2.0 ** -24 * 128 + 2.0 ** -24 * np.sqrt(m + 1.0) + 2 * ce
            lse_e[r, h] = (c32 * (1 + np.abs(np.where(np.isinf(l), 0, l))[:, None]))[:, 0]
            z["o"][r, h] = P @ V
            mass = P @ np.abs(V)
            e["o"][r, h] = u * np.abs(z["o"][r, h]) + (u + c32) * mass + tiny * (1 + np.abs(V).sum(0))
            if d_o is None:
                continue
            dO, O = d_o[r, h], o_in[r, h]
            dP, delta = dO @ V.T, (dO * (P @ V)).sum(1, keepdims=True)
            dS = P * (dP - delta)
            # delta comes from the rounded o; dP and delta carry 32-bit sums
            de = np.abs((dO * (O - P @ V)).sum(1, keepdims=True))
            dabs = np.abs(dO) @ np.abs(V).T + (np.abs(dO) * mass).sum(1, keepdims=True)
            dSe = tiny + u * np.abs(dS) + P * (de + 4 * c32 * dabs)
            z["dq"][r, h] = scale * (dS @ K)
            e["dq"][r, h] = u * np.abs(z["dq"][r, h]) + scale * (dSe @ np.abs(K)) + tiny
            z["dk"][c, g] += scale * (dS.T @ Q)
            e["dk"][c, g] += scale * (dSe.T @ np.abs(Q))
            z["dv"][c, g] += P.T @ dO
            e["dv"][c, g] += (tiny + (u + 4 * c32) * P).T @ np.abs(dO)
        r0, c0 = r0 + n, c0 + m
    for n in ("dk", "dv"):
        e[n] += u * np.abs(z[n]) + tiny
    out = {n: (z[n], e[n]) for n in z}
    out["lse"] = (lse, lse_e)
    return out


def worst(got, want):
    """Largest error over its bound (at most 1 passes); not-a-number counts as infinite."""
    value, bound = want
    same = (got == value) | (np.isnan(got) & np.isnan(value))  # infinities too
    with np.errstate(invalid="ignore"):
        x = np.where(same, 0.0, np.abs(got - value) / bound)
    return float(np.max(np.where(np.isnan(x), np.inf, x), initial=0.0))


# ---- 8 bits (e4m3) and the paged cache ------------------------------------------------------
def _f8_table():
    t = np.zeros(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        x = m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        t[c] = np.nan if (c & 127) == 127 else x
        if c & 128:
            t[c] = -t[c]
    return t


F8 = _f8_table()


def f8_codes(x):
    """To nearest, ties to the even code; beyond 448 that; NaN stays (any of its two codes)."""
    x = np.asarray(x, dtype=np.float64)
    up = F8[:127]  # ascending from 0 to 448
    a = np.minimum(np.where(np.isnan(x), 0.0, np.abs(x)), 448.0)
    hi = np.clip(np.searchsorted(up, a), 0, 126)
    lo = np.maximum(hi - 1, 0)
    dl, dh = a - up[lo], up[hi] - a
    code = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    code = np.where(np.isnan(x), 127, code)
    return (code + np.where(np.signbit(x), 128, 0)).astype(np.uint8)


def scale_for(most):
    """The smallest 2^e, -40 <= e <= 40, with most <= 448 * 2^e."""
    e = -40
    while e < 40 and float(most) > 448.0 * 2.0 ** e:
        e += 1
    return np.float32(2.0 ** e)


def rotate(x, table, pos):
    """x [rows, heads, dim] float32, rounded after every operation as the formula is written."""
    n = table.shape[1]
    h = n // 2
    y = x.astype(np.float32).copy()
    for r, p in enumerate(pos):
        if p < 0:
            continue
        c, s = table[p, :h], table[p, h:]
        a, b = x[r, :, :h].astype(np.float32), x[r, :, h:n].astype(np.float32)
        y[r, :, :h] = a * c - b * s
        y[r, :, h:n] = b * c + a * s
    return y


class HostCache:
    """The pages of a cache as the library lays them out, on the host."""

    def __init__(self, dtype, pages, page, heads, dim):
        self.dtype, self.pages, self.page, self.heads, self.dim = dtype, pages, page, heads, dim
        kind = {"f8": np.uint8, "f16": np.float16, "bf16": np.uint16}[dtype]
        garbage = {"f8": 0x7F, "f16": np.nan, "bf16": 0x7FC0}[dtype]  # not-a-number until written
        self.k = np.full((pages, heads, page, dim), garbage, kind)
        self.v = np.full((pages, heads, dim, page), garbage, kind)
        self.k_scale = np.full((pages, heads), np.nan, np.float32)
        self.v_scale = np.full((pages, heads), np.nan, np.float32)

    def append(self, pages_of, first, k, v):
        """Rows k / v [n, heads, dim] float32 (rotated) at positions first .. of one sequence."""
        for h in range(self.heads):
            for p in range(first // self.page, (first + len(k) - 1) // self.page + 1 if len(k) else 0):
                lo, hi = max(first - p * self.page, 0), min(first + len(k) - p * self.page, self.page)
                rows = slice(lo + p * self.page - first, hi + p * self.page - first)
                at = pages_of[p]
                if at >= self.pages:
                    continue
                for held, scales, x in ((self.k[at, h], self.k_scale, k[rows, h]),
                                        (self.v[at, h].T, self.v_scale, v[rows, h])):
                    if self.dtype != "f8":
                        held[lo:hi] = to_bits(x, self.dtype)
                        continue
                    with np.errstate(invalid="ignore"):
                        finite = np.where(np.isfinite(x), np.abs(x), 0)
                    scale, was = scale_for(finite.max()), scales[at, h]
                    if lo:
                        was = was if was > 0 else np.float32(0)
                        scale = max(scale, was)
                        if was != scale:
                            held[:lo] = f8_codes(F8[held[:lo]] * (was / scale))
                    scales[at, h] = scale
                    held[lo:hi] = f8_codes(x / scale)

    def values(self, pages_of, n):
        """Keys and values [n, heads, dim] in 64 bits of a sequence of n tokens."""
        k, v = np.zeros((n, self.heads, self.dim)), np.zeros((n, self.heads, self.dim))
        for p in range(-(-n // self.page)):
            at, hi = pages_of[p], min(self.page, n - p * self.page)
            if at >= self.pages:
                continue
            rows = slice(p * self.page, p * self.page + hi)
            for out, held, scales in ((k, self.k[at], self.k_scale), (v, self.v[at].transpose(0, 2, 1), self.v_scale)):
                x = held[:, :hi]
                x = F8[x] * scales[at].astype(np.float64)[:, None, None] if self.dtype == "f8" else from_bits(x, self.dtype)
                out[rows] = x.transpose(1, 0, 2)
        return k, v
