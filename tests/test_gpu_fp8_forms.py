"""8-bit floating-point weights on the GPU, form by form, on data whose result is known to the last bit or bounded by arithmetic: what
may lie beside what, and what the e4m3 instruction drops."""

import numpy as np
import pytest
import torch

from oracle import fp8
from oracle.kvcache import e4m3_decode
from tests.e4m3_cases import hard_codes
from vybforge_amd import _lib, ops

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "f64": torch.float64}
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f64": 2.0 ** -24}  # half a step of the last rounding, relative


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


# ---- the e4m3 instruction ---------------------------------------------------------------------------

# (rows, K, forced tile): few rows, the tiles for short K, every tile of the pipeline with whole and short last blocks
FORMS = [(1, 640, None), (12, 1040, None), (40, 384, None), (100, 400, None), (520, 256, None), (40, 640, "64,1"), (40, 528, "64,1"),
         (60, 1152, "64,2"), (130, 640, "128,1"), (130, 528, "128,1"), (200, 640, "192,1"), (270, 640, "256,1"), (270, 528, "256,1")]


@pytest.mark.parametrize("kind", ["large", "subnormal", "spread", "normal"])
@pytest.mark.parametrize("y", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("M,K,tile", FORMS)
def test_what_the_instruction_drops(dev, rng, monkeypatch, M, K, tile, y, kind):
    """16-bit outputs are the instruction's sums to float32, so within the bound of what it drops; float32 outputs drop nothing. What
    float32 adds: each of a block's 128 products and of the KB blocks rounds, or is cut, by 2^-23 of the partial sums at most, with
    two for the scales' products (as everywhere here); the codes' scales are 1, and float16 is kept off its border by 2^-12."""
    if tile:
        monkeypatch.setenv("VYBDQ_FP8_TILE", tile)
    N, KB = 300, fp8.blocks(K)
    some = np.unique(np.r_[0, M - 1, rng.integers(0, M, 10)])  # (the oracle's rows)
    xc, wc = hard_codes(rng, M, N, K, kind)
    f = np.float32(2.0 ** -12)
    work = ops.Fp8Workspace([(M, N, K)], dev)
    got = ops.gemm_fp8(torch.from_numpy(wc).to(dev).view(E4M3), torch.full((fp8.blocks(N), KB), float(f), device=dev),
                       torch.from_numpy(xc).to(dev).view(E4M3), torch.ones(M, KB, device=dev), y_dtype=DT[y], workspace=work)
    got, xs = got.double().cpu().numpy()[some], xc[some]
    X, W = e4m3_decode(xs), e4m3_decode(wc)
    exact, size = f * (X @ W.T), f * (np.abs(X) @ np.abs(W).T)
    want = exact if y == "f32" else f * fp8.e4m3_instruction(xs, wc).sum(-1)
    tol = (130 + KB) * 2.0 ** -23 * size
    last = lambda v, t: HALF[y] * (np.abs(v) + t) + (2.0 ** -25 if y == "f16" else 0)
    assert (np.abs(got - want) <= tol + last(want, tol)).all(), np.abs(got - want).max()
    tol += 0 if y == "f32" else f * fp8.e4m3_loss(xs, wc)
    assert (np.abs(got - exact) <= tol + last(exact, tol)).all()
