"""Codes that the e4m3 matrix instruction loses most of: for tests of its bound."""

import numpy as np

from oracle import fp8


def hard_codes(rng, M, N, K, kind):
    """xc [M, K], wc [N, K]. large: every eight k hold one product of 2^16 (of alternating sign from eight to eight) and seven just
    below 2^-13 of it, all of one sign, so that blocks sum to what is dropped; subnormal: the same beside a large weight that meets
    a subnormal code; spread: random exponents; normal: as quantizing normal data leaves them."""
    j, first = np.arange(K) // 8, np.arange(K) % 8 == 0
    if kind == "large":
        x = np.where(first, 256.0, 1.875 * 2.0 ** rng.integers(0, 2, (M, K)))
        w = np.where(first, np.where(j % 2, -256.0, 256.0), 1.875 * 2.0 ** rng.integers(-1, 1, (N, K)))
    elif kind == "subnormal":
        x = np.where(first, 2.0 ** -9 * rng.integers(1, 8, (M, K)), 2.0 ** -6 * rng.integers(8, 16, (M, K)) / 8)
        w = np.where(first, np.where(j % 2, -256.0, 256.0), 2.0 ** -7 * rng.integers(1, 8, (N, K)) / 4)
    elif kind == "spread":
        x, w = (rng.uniform(-1.9, 1.9, (n, K)) * 2.0 ** rng.integers(-9, 9, (n, K)) for n in (M, N))
        x, w = np.clip(x, -448, 448), np.clip(w, -448, 448)
    else:
        x, w = (np.clip(rng.standard_normal((n, K)) * 110, -448, 448) for n in (M, N))
    return fp8.e4m3_encode(x), fp8.e4m3_encode(w)
