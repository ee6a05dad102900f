"""8-bit floating-point weights on the GPU, form by form, on data whose result is known to the last bit or bounded by arithmetic: what
may lie beside what."""

import numpy as np
import pytest
import torch

from oracle import fp8
from vybforge_amd import _lib, ops

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn


def stream():
    return torch.cuda.current_stream().cuda_stream


# ---- whole numbers: every sum is exact in float32, in any order and on both instructions ----------

def whole(rng, rows, K, top, dev):
    """e4m3 codes [rows, K] of the whole numbers -top .. top, on the GPU."""
    table = torch.from_numpy(fp8.e4m3_encode(np.arange(-top, top + 1).astype(np.float64))).to(dev)
    g = torch.Generator(device=dev)
    g.manual_seed(int(rng.integers(1 << 30)))
    return table[torch.randint(0, 2 * top + 1, (rows, K), generator=g, device=dev)].view(E4M3)


def powers(rng, shape, dev):
    """Scales 1/2, 1, 2."""
    return torch.from_numpy(2.0 ** rng.integers(-1, 2, shape)).float().to(dev)


def values(codes, scales, per):
    """float32 values: a scale for `per` rows (1: activations, 128: weights) and 128 columns."""
    return codes.float() * scales.repeat_interleave(per, 0)[:len(codes)].repeat_interleave(128, 1)[:, :codes.shape[1]]


def whole_product(rng, M, N, K, dev):
    """W, Ws, Xq, Xs and the product, exact in float32: whole numbers up to 6 in quarters, below 2^24 quarters for K < 2^17."""
    W, Ws = whole(rng, N, K, 2, dev), powers(rng, (fp8.blocks(N), fp8.blocks(K)), dev)
    X, Xs = whole(rng, M, K, 3, dev), powers(rng, (M, fp8.blocks(K)), dev)
    return W, Ws, X, Xs, (values(X, Xs, 1).double() @ values(W, Ws, 128).double().t())


# ---- buffers side by side -------------------------------------------------------------------------

@pytest.mark.parametrize("M", [1, 3, 40, 300])
def test_columns_of_one_matrix(dev, rng, M):
    """X, Y, the residual and, in a gap between rows, the codes and scales of X: columns of one wider matrix overlap nowhere."""
    N, K = 192, 256
    W, Ws, Xq, Xs, want = whole_product(rng, M, N, K, dev)
    x = values(Xq, torch.ones_like(Xs), 1)
    want = (x.double() @ values(W, Ws, 128).double().t())
    wide = torch.zeros(M, 1024, device=dev)
    wide[:, :K], wide[:, K + N:K + 2 * N] = x, 5.0
    wide[:, K + 2 * N:] = 7.0
    p, ld = wide.data_ptr(), 1024
    n = _lib.lib.vybdq_linear_fp8_workspace_size(M, N, K)
    ws = torch.empty(n + 256, dtype=torch.uint8, device=dev)
    ops.call("vybdq_linear_fp8", W.data_ptr(), Ws.data_ptr(), p, _lib.F32, ld, p + 4 * K, M, N, K, _lib.F32, ld, p + 4 * (K + N),
             (ws.data_ptr() + 255) // 256 * 256, n, stream())
    assert torch.equal(wide[:, K:K + N].double(), want + 5) and torch.equal(wide[:, :K], x)
    assert (wide[:, K + N:K + 2 * N] == 5).all() and (wide[:, K + 2 * N:] == 7).all()
    # the residual is the output itself
    ops.call("vybdq_linear_fp8", W.data_ptr(), Ws.data_ptr(), p, _lib.F32, ld, p + 4 * K, M, N, K, _lib.F32, ld, p + 4 * K,
             (ws.data_ptr() + 255) // 256 * 256, n, stream())
    assert torch.equal(wide[:, K:K + N].double(), 2 * want + 5)
    if M == 3:  # 768 codes and 6 scales between two rows of X
        codes, scales = p + 4 * 256, p + 4 * 512
        ops.call("vybdq_quant_fp8", p, _lib.F32, ld, codes, scales, M, K, stream())
        q, s = fp8.quant(x.cpu().numpy())
        np.testing.assert_array_equal(wide[0, 256:448].view(torch.uint8).cpu().numpy(), q.reshape(-1))
        np.testing.assert_array_equal(wide[0, 512:518].cpu().numpy(), s.reshape(-1))


def test_layer_output_over_its_input(dev, rng):
    """out may be x."""
    E, H, I = 8, 256, 128
    pairs = [(whole(rng, E * n, k, 2, dev).view(E, n, k), torch.ones(E, n // 128, k // 128, device=dev)) for n, k in ((I, H), (I, H), (H, I))]
    layer = ops.MoeFp8Layer(*pairs, topk=2)
    for T in (2, 70):
        x, logits = torch.randn(T, H, device=dev), torch.randn(T, E, device=dev)
        want, v = layer(x, logits), x.clone()
        assert layer(v, logits, out=v) is v and torch.equal(v, want)
