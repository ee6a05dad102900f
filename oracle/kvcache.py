"""The paged 8-bit key/value cache in numpy: appending with rotation, and attention over it in float64.

Layout and semantics are those of include/vybdq.h (vybdq_kv_append, vybdq_kv_attn). Appending follows the
definition in float32, one rounding per product and sum, so that codes and scales are reproducible bit for bit.
"""

import numpy as np

E_MIN, E_MAX, CODE_MAX = -60, 60, 448.0


def e4m3_decode(codes):
    """float64 values of e4m3 codes (uint8): sign, 4 exponent bits (bias 7), 3 mantissa bits; 0x7f is NaN."""
    c = np.asarray(codes, np.uint8).astype(np.int64)
    sign, e, m = np.where(c & 0x80, -1.0, 1.0), (c >> 3) & 15, c & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))
    return np.where((c & 0x7f) == 0x7f, np.nan, sign * v)


def e4m3_encode(x):
    """Codes of finite values held to +-448, to nearest, ties to even."""
    x = np.clip(np.asarray(x, np.float64), -CODE_MAX, CODE_MAX)
    a = np.abs(x)
    e = np.maximum(np.floor(np.log2(np.maximum(a, 2.0 ** -20))), -6)  # subnormals share the least exponent
    n = np.rint(a / 2.0 ** (e - 3)).astype(np.int64)                  # 8 .. 16, or 0 .. 8 below 2^-6
    code = np.where(e == -6, n, ((e + 7).astype(np.int64) << 3) + n - 8)  # a carry moves on into the exponent
    return (code | np.where(np.signbit(x), 0x80, 0)).astype(np.uint8)


def page_exponent(amax):
    """The least e with amax <= 448 * 2^e, within the allowed exponents; a zero has the least."""
    f, x = np.frexp(np.float64(amax))
    return int(np.clip(x - 9 if f <= 0.875 else x - 8, E_MIN, E_MAX)) if amax else E_MIN


def rotate(x, pos, cos, sin, interleaved):
    """x float32 [..., D] of one token at position pos."""
    if cos is None:
        return x.copy()
    half = cos.shape[1]
    c, s, y = cos[pos], sin[pos], x.copy()
    a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    with np.errstate(all="ignore"):
        y[..., a] = x[..., a] * c - x[..., b] * s
        y[..., b] = x[..., b] * c + x[..., a] * s
    return y


class Cache:
    """codes k, v uint8 and scales, laid out as the library's."""

    def __init__(self, k, v, k_scale, v_scale):
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.page = k.shape[2]

    def values(self, table, ctx, h):
        """float64 keys and values [ctx, D] of a sequence's head."""
        n = -(-ctx // self.page)
        D = self.k.shape[3]
        pages = [int(p) for p in table[:n]]
        k = np.concatenate([e4m3_decode(self.k[p, h]) * np.float64(self.k_scale[p, h]) for p in pages] or [np.zeros((0, D))])
        v = np.concatenate([e4m3_decode(self.v[p, h].transpose(0, 2, 1).reshape(-1, D)) * np.float64(self.v_scale[p, h])
                            for p in pages] or [np.zeros((0, D))])
        return k[:ctx], v[:ctx]

    def _write(self, codes, scale, pg, h, keep, new, bad, nan):
        """new float32 [n, D] into the slots behind the first `keep` of page pg."""
        D = new.shape[1]
        flat = codes[pg, h] if codes.ndim == 4 else codes[pg, h].transpose(0, 2, 1).reshape(-1, D).copy()
        e = page_exponent(np.max(np.where(np.isfinite(new), np.abs(new), 0), initial=0))
        if keep:
            old = int(np.log2(scale[pg, h]))
            if e > old:
                flat[:keep] = e4m3_encode(e4m3_decode(flat[:keep]) * 2.0 ** (old - e))
            e = max(e, old)
        scale[pg, h] = np.float32(2.0) ** e
        code = e4m3_encode(np.where(np.isfinite(new), new, 0).astype(np.float64) * 2.0 ** -e)
        code[bad] = nan
        flat[keep:keep + len(new)] = code
        codes[pg, h] = flat if codes.ndim == 4 else flat.reshape(-1, 4, D).transpose(0, 2, 1)

    def append(self, k, v, table, ctx, cos=None, sin=None, interleaved=False):
        """One sequence's rows k, v float32 [n, Hkv, D], the last of its ctx tokens."""
        n, p0 = len(k), ctx - len(k)
        k = np.stack([rotate(k[i], p0 + i, cos, sin, interleaved) for i in range(n)]) if n else k
        for i in range(p0 // self.page, (ctx - 1) // self.page + 1 if n else 0):
            lo, hi = max(p0, i * self.page), min(ctx, (i + 1) * self.page)
            for h in range(k.shape[1]):
                nk, nv = k[lo - p0:hi - p0, h], v[lo - p0:hi - p0, h]
                bad = ~(np.isfinite(nk).all(1) & np.isfinite(nv).all(1))
                self._write(self.k, self.k_scale, int(table[i]), h, lo - i * self.page, nk, bad, 0x7f)
                self._write(self.v, self.v_scale, int(table[i]), h, lo - i * self.page, nv, bad, 0)


def attention(q, k, v, p0, ctx, scale, causal=True, window=0):
    """q [n, D] at positions p0 ..., k, v [ctx, D], all float64: out [n, D], lse [n], and for a bound on a computation's
    error sum_j p_j |v_j| [n, D] and max_j |scale| sum_d |q_d k_jd| [n]."""
    pos, j = p0 + np.arange(len(q))[:, None], np.arange(ctx)[None, :]
    seen = np.ones((len(q), ctx), bool)
    if causal:
        seen &= j <= pos
    if window:
        seen &= j > pos - window
    out, lse = np.zeros_like(q), np.full(len(q), -np.inf)
    weight, reach = np.zeros_like(q), np.zeros(len(q))
    for i in range(len(q)):
        at = seen[i]
        if not at.any():
            continue
        t = (k[at] @ q[i]) * scale
        m = t.max()
        if np.isnan(t).any():
            out[i], lse[i] = np.nan, np.nan
            continue
        p = np.exp(t - m)
        lse[i] = m + np.log(p.sum())
        p /= p.sum()
        out[i], weight[i] = p @ v[at], p @ np.abs(v[at])
        reach[i] = (np.abs(k[at]) @ np.abs(q[i])).max() * abs(scale)
    return out, lse, weight, reach
