"""The numpy oracle of the 8-bit key/value cache: its e4m3 against torch's, its scales and rotation against
plain formulas. CPU only."""

import numpy as np
import pytest
import torch

from oracle import kvcache


def test_e4m3_decode_matches_torch():
    codes = np.arange(256, dtype=np.uint8)
    want = torch.from_numpy(codes).view(torch.float8_e4m3fn).double().numpy()
    np.testing.assert_array_equal(kvcache.e4m3_decode(codes), want)


def test_e4m3_encode_matches_torch(rng):
    x = np.concatenate([rng.standard_normal(4000) * 2.0 ** rng.integers(-14, 9, 4000), [0.0, -0.0, 448, -448, 2.0 ** -10],
                        kvcache.e4m3_decode(np.arange(0x7f, dtype=np.uint8))]).astype(np.float32)
    a = kvcache.e4m3_decode(np.arange(0x7e, dtype=np.uint8))
    x = np.concatenate([x, ((a[1:] + a[:-1]) / 2).astype(np.float32)])  # ties
    x = np.clip(x, -448, 448)
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    np.testing.assert_array_equal(kvcache.e4m3_encode(x), want)


@pytest.mark.parametrize("e", [-60, -9, 0, 13, 60])
def test_page_exponent(e):
    top = np.float32(448.0) * np.float32(2.0) ** e
    assert kvcache.page_exponent(top) == e
    assert kvcache.page_exponent(np.nextafter(top, np.float32(np.inf))) == min(e + 1, 60)
    assert kvcache.page_exponent(0.0) == -60


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotation_is_a_rotation(rng, interleaved):
    x = rng.standard_normal((3, 64)).astype(np.float32)
    ang = rng.standard_normal((5, 16))
    c, s = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)
    y = kvcache.rotate(x, 4, c, s, interleaved)
    pick = (lambda t: t[:, 0:32:2] + 1j * t[:, 1:32:2]) if interleaved else (lambda t: t[:, :16] + 1j * t[:, 16:32])
    # two products and a sum in float32: at most 3 half steps of the larger pair member
    np.testing.assert_allclose(pick(y), pick(x.astype(np.float64)) * np.exp(1j * ang[4]), atol=8 * 2.0 ** -22)
    np.testing.assert_array_equal(y[:, 32:], x[:, 32:])


def test_attention_oracle_against_torch(rng):
    q, k, v = rng.standard_normal((5, 64)), rng.standard_normal((9, 64)), rng.standard_normal((9, 64))
    out, lse, _, _ = kvcache.attention(q, k, v, 4, 9, 0.125)
    t = torch.from_numpy(q @ k.T * 0.125).masked_fill(torch.arange(9)[None] > 4 + torch.arange(5)[:, None], -torch.inf)
    np.testing.assert_allclose(out, (t.softmax(-1) @ torch.from_numpy(v)).numpy(), rtol=1e-12, atol=1e-13)
    np.testing.assert_allclose(lse, t.logsumexp(-1).numpy(), rtol=1e-12)
    out, lse, _, _ = kvcache.attention(q, k[:0], v[:0], -5, 0, 0.125)
    assert (out == 0).all() and np.isneginf(lse).all()


def test_append_keeps_and_rounds_anew(rng):
    """Tokens added one at a time, each larger than the ones before: every stored value within half a step of its
    code, and where it falls among the subnormals within the half steps 2^-10 scale (1 + 1/2 + ...) of every growth."""
    P, D = 16, 64
    c = kvcache.Cache(np.zeros((1, 1, P, D), np.uint8), np.zeros((1, 1, P // 4, D, 4), np.uint8),
                      np.ones((1, 1), np.float32), np.ones((1, 1), np.float32))
    x = (rng.standard_normal((P, 1, D)) * 1.7 ** np.arange(P)[:, None, None]).astype(np.float32)
    for t in range(P):
        c.append(x[t:t + 1], -x[t:t + 1], [0], t + 1)
    k, v = c.values([0], P, 0)
    step = np.abs(x[:, 0]) * 2.0 ** -4 + 2 * 2.0 ** -10 * c.k_scale[0, 0]
    assert (np.abs(k - x[:, 0]) <= step).all() and (np.abs(v + x[:, 0]) <= step).all()
