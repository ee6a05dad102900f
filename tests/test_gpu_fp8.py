"""8-bit floating-point weights on the GPU: the quantizer and the router against the oracle bit for bit, the product against float64 with
a bound from the arithmetic, the layer where every code is certain and where it is not, and all of them as a host runs them."""

import math

import numpy as np
import pytest
import torch

from oracle import fp8
from oracle.kvcache import e4m3_decode
from vybforge_amd import _lib, ops

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "f64": torch.float64}
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f64": 2.0 ** -24}  # half a step of the last rounding, relative


def to(dev, a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(dev)


def codes_to(dev, a):
    return to(dev, a).view(torch.float8_e4m3fn)


def matrix(rng, N, K, lead=()):
    """Codes of any magnitude (no NaN), scales of every size about 1 / sqrt(K)."""
    c = rng.integers(0, 256, lead + (N, K), dtype=np.uint8)
    c[(c & 0x7f) == 0x7f] ^= 1
    s = np.exp(rng.standard_normal(lead + (fp8.blocks(N), fp8.blocks(K)))) / (100 * math.sqrt(K))
    return c, s.astype(np.float32)


def normal_matrix(rng, N, K, lead=()):
    """Codes and scales as quantizing N(0, 1 / K) weights leaves them."""
    c = fp8.e4m3_encode(rng.standard_normal(lead + (N, K)) * 110)
    s = rng.uniform(0.5, 1.5, lead + (fp8.blocks(N), fp8.blocks(K))) / (110 * math.sqrt(K))
    return c, s.astype(np.float32)


def on(dev, m):
    return codes_to(dev, m[0]), to(dev, m[1])


def bits(t):
    return t.view(torch.uint8).cpu().numpy()


# ---- quantizer ------------------------------------------------------------------------------------

def check_quant(dev, x):
    """x a tensor on the GPU, rows of any stride."""
    want = fp8.quant(x.detach().float().cpu().numpy())
    q, s = ops.quant_fp8(x)
    np.testing.assert_array_equal(bits(q), want[0])
    np.testing.assert_array_equal(s.cpu().numpy(), want[1])


@pytest.mark.parametrize("x", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("M,K", [(1, 16), (1, 128), (3, 144), (17, 2576), (2, 6144), (200, 272), (5, 17408)])
def test_quantizer(dev, rng, x, M, K):
    v = rng.standard_normal((M, K)) * np.exp(rng.standard_normal((M, 1)) * 3)
    check_quant(dev, torch.from_numpy(v).to(DT[x]).to(dev))


@pytest.mark.parametrize("scale", [0.0, 1e-45, 1e-38, 2.0 ** -101, 2.0 ** -92, 1e-6, 448.0, 449.0, 1e10, 3e38])
def test_quantizer_magnitudes(dev, rng, scale):
    v = rng.uniform(-1, 1, (6, 256)).astype(np.float32) * np.float32(scale)
    v[:, 7] = scale
    check_quant(dev, torch.from_numpy(v).to(dev))


def test_quantizer_ties_and_borders(dev):
    # every midpoint of two codes below a block's largest value, at scales on both sides of a power of two's border
    values = e4m3_decode(np.arange(127).astype(np.uint8))
    mids = (values[1:] + values[:-1]) / 2
    rows = [np.concatenate([[top], mids * top / 448, [0.0]])[:128] for top in (448.0, 447.999, 448.0001, 7.0, 3.5, 1.0)]
    check_quant(dev, torch.from_numpy(np.stack(rows).astype(np.float32)).to(dev))


def test_quantizer_infinities_and_nan_stay_in_their_block(dev, rng):
    v = rng.standard_normal((5, 384)).astype(np.float32)
    v[0, 3], v[1, 200], v[2, 383], v[3, :] = np.inf, -np.inf, np.nan, np.nan
    check_quant(dev, torch.from_numpy(v).to(dev))
    assert np.isnan(fp8.quant(v)[1]).tolist() == [[True, False, False], [False, True, False], [False, False, True], [True] * 3,
                                                  [False] * 3]


def test_quantizer_slices_and_given_outputs(dev, rng):
    wide = torch.from_numpy(rng.standard_normal((9, 1024)).astype(np.float32)).to(dev).half()
    check_quant(dev, wide[:, 128:528])
    check_quant(dev, wide[::2, 64:320])
    check_quant(dev, wide[3:4])
    q = torch.full((9 * 1024 + 64,), 85, dtype=torch.uint8, device=dev)
    s = torch.full((9 * 8 + 8,), 85.0, device=dev)
    ops.quant_fp8(wide, out=(q[:9 * 1024].view(torch.float8_e4m3fn), s[:72]))
    assert (q[9 * 1024:] == 85).all() and (s[72:] == 85).all()
    np.testing.assert_array_equal(q[:9 * 1024].cpu().numpy(), fp8.quant(wide.float().cpu().numpy())[0].reshape(-1))
    assert ops.quant_fp8(wide[:0])[0].shape == (0, 1024)


# ---- product --------------------------------------------------------------------------------------

def product_bound(xc, xs, wc, ws, y):
    """float64 product and what separates the kernel from it: every block sum and the outer sum in float32 (each of 128 + KB
    terms rounds, or is cut, by 2^-23 of the partial sums, which sum |x w| bounds); for 16-bit outputs the e4m3 instruction
    loses up to 2^-10 of each block's largest product; the last rounding is half a step, or the least subnormal's."""
    X, W = e4m3_decode(xc), e4m3_decode(wc)
    out, err = np.zeros((X.shape[0], W.shape[0])), np.zeros((X.shape[0], W.shape[0]))
    KB, rows = xs.shape[1], np.arange(W.shape[0]) // 128
    for b in range(KB):
        at = slice(128 * b, 128 * (b + 1))
        f = xs[:, b, None].astype(np.float64) * ws[rows, b][None].astype(np.float64)
        out += f * (X[:, at] @ W[:, at].T)
        err += np.abs(f) * (np.abs(X[:, at]) @ np.abs(W[:, at]).T) * (130 + KB) * 2.0 ** -23
        if y in ("f16", "bf16"):
            err += np.abs(f) * np.abs(X[:, None, at] * W[None, :, at]).max(-1) * 2.0 ** -10
    return out, err + HALF[y] * (np.abs(out) + err) + (2.0 ** -25 if y == "f16" else 2.0 ** -140)


def check_product(dev, rng, M, N, K, y, rs=False, make=matrix, split=False):
    (wc, ws), x = make(rng, N, K), rng.standard_normal((M, K)) * np.exp(rng.standard_normal((M, fp8.blocks(K)))).repeat(128, 1)[:, :K]
    xc, xs = fp8.quant(x.astype(np.float32))
    want, tol = product_bound(xc, xs, wc, ws, y)
    r = None
    if rs:
        r = torch.from_numpy(rng.standard_normal((M, N))).to(DT[y]).to(dev)
        want = want + r.double().cpu().numpy()
        tol = tol + HALF[y] * np.abs(r.double().cpu().numpy())
    work = ops.Fp8Workspace([(M, N, K)], dev) if split else None
    if split:
        work.buf.fill_(0x7f)  # any contents (NaN, as float32)
    out = ops.gemm_fp8(*on(dev, (wc, ws)), *on(dev, (xc, xs)), y_dtype=DT[y], residual=r, workspace=work)
    got = out.double().cpu().numpy()
    assert out.shape == (M, N) and (np.abs(got - want) <= tol).all(), np.abs((got - want) / tol).max()
    return out


@pytest.mark.parametrize("y", ["f32", "bf16"])
@pytest.mark.parametrize("K", [16, 112, 128, 144, 1024, 2576])
@pytest.mark.parametrize("M,N", [(1, 1), (1, 16), (2, 129), (16, 100), (17, 128), (33, 257), (64, 64), (65, 130), (129, 300)])
def test_product(dev, rng, M, N, K, y):
    check_product(dev, rng, M, N, K, y)


@pytest.mark.parametrize("y", ["f32", "f16", "bf16", "f64"])
@pytest.mark.parametrize("M,N,K", [(1, 640, 512), (12, 1003, 528), (70, 96, 640), (300, 520, 384), (513, 260, 256)])
def test_product_types_and_residuals(dev, rng, M, N, K, y):
    check_product(dev, rng, M, N, K, y, rs=True, make=normal_matrix)


@pytest.mark.parametrize("M,N,K", [(1, 4000, 8192), (7, 200, 17408), (40, 300, 12288), (530, 700, 1536), (1030, 520, 640)])
def test_product_long(dev, rng, M, N, K):
    check_product(dev, rng, M, N, K, "bf16", make=normal_matrix)


@pytest.mark.parametrize("y", ["f32", "bf16"])
@pytest.mark.parametrize("tile", ["64,1", "64,3", "128,1", "128,4", "192,1", "192,3", "256,1", "256,2"])
@pytest.mark.parametrize("M,N,K", [(17, 1000, 2048), (64, 37, 2176), (130, 520, 2048), (300, 1300, 1152), (33, 300, 2064), (200, 290, 1648)])
def test_product_tiles_and_splits(dev, rng, monkeypatch, M, N, K, tile, y):
    """Every tile of the pipeline, whole and with K split, more tiles than one to a workgroup or fewer, ragged in every way."""
    monkeypatch.setenv("VYBDQ_FP8_TILE", tile)
    check_product(dev, rng, M, N, K, y, rs=True, make=normal_matrix, split=True)


def test_product_many_tiles_to_a_workgroup(dev, rng):
    """More tiles than workgroups: each goes on from tile to tile (17 x 23 tiles of 256 x 256, 64 x 33 of 64 x 256)."""
    for M, N, K in ((4200, 5700, 512), (64, 90000, 512)):
        (wc, ws), (xc, xs) = normal_matrix(rng, N, K), fp8.quant(rng.standard_normal((M, K)).astype(np.float32))
        W, X = on(dev, (wc, ws)), on(dev, (xc, xs))
        got = ops.gemm_fp8(*W, *X)
        rows, cols = rng.choice(M, min(M, 40), replace=False), rng.choice(N, 300, replace=False)
        want = (fp8.activations(xc[rows], xs[rows]) @ (e4m3_decode(wc[cols]) * ws[cols // 128].repeat(128, 1)[:, :K]).T)
        # (the bound of product_bound with the largest |x w| sum: values of rms 1 over K = 512 terms)
        np.testing.assert_allclose(got.cpu().numpy()[np.ix_(rows, cols)], want, rtol=0, atol=134 * 2.0 ** -23 * 40)
        again = torch.empty_like(got)
        for i in range(0, M, 1000):
            ops.gemm_fp8(*W, X[0][i:i + 1000], X[1][i:i + 1000], out=again[i:i + 1000])
        assert (got - again).abs().max() < 1e-4  # (tiles of other sizes sum in the same order, block by block)


@pytest.mark.parametrize("M", [1, 16, 40, 100, 600])
@pytest.mark.parametrize("y", ["f32", "bf16"])
def test_product_is_exact_where_float32_is(dev, rng, M, y):
    """Small whole numbers: every sum is one float32 holds, in any order and for both instructions."""
    N, K = 200, 272
    x, w = rng.integers(-3, 4, (M, K)).astype(np.float32), rng.integers(-2, 3, (N, K)).astype(np.float32)
    wc, ws = fp8.e4m3_encode(w), np.ones((2, 3), np.float32)
    ws[1] = 0.25
    xc, xs = fp8.quant(x)
    want = (x @ fp8.weights(wc, ws).T.astype(np.float32))
    got = ops.gemm_fp8(*on(dev, (wc, ws)), *on(dev, (xc, xs)), y_dtype=DT[y])
    assert torch.equal(got.cpu(), torch.from_numpy(want).to(DT[y]))


@pytest.mark.parametrize("y", ["f32", "bf16"])
@pytest.mark.parametrize("K", [1040, 1136, 2032])
@pytest.mark.parametrize("M", [1, 16, 40, 200])
def test_product_short_last_block_beside_nan(dev, rng, M, K, y):
    """Rows end inside a block: what follows them in memory (the next row's first codes, all NaN) takes no part."""
    N = 140
    x, w = rng.integers(-3, 4, (M, K)).astype(np.float32), rng.integers(-2, 3, (N, K)).astype(np.float32)
    wc, (xc, xs) = fp8.e4m3_encode(w), fp8.quant(x)
    wc[1::2, :128], xc[1::2, :128] = 0x7f, 0x7f
    got = ops.gemm_fp8(codes_to(dev, wc), torch.ones(2, fp8.blocks(K), device=dev), *on(dev, (xc, xs)), y_dtype=DT[y]).float().cpu()
    want = torch.from_numpy(x @ w.T).to(DT[y]).float()
    want[1::2], want[:, 1::2] = math.nan, math.nan
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())


@pytest.mark.parametrize("M", [1, 20, 130])
def test_product_nan_stays_in_its_row_and_column(dev, rng, M):
    N, K = 150, 400
    wc, ws = normal_matrix(rng, N, K)
    x = rng.standard_normal((M, K)).astype(np.float32)
    x[M // 2, 130] = np.inf
    wc[33, 399] = 0x7f
    ws[1, 2] = np.inf  # (rows 128 .. of W)
    got = ops.gemm_fp8(*on(dev, (wc, ws)), *on(dev, fp8.quant(x))).cpu().numpy()
    bad = np.zeros((M, N), bool)
    bad[M // 2], bad[:, 33] = True, True
    assert np.isnan(got[bad]).all() and np.isfinite(got[~bad][got[~bad] < np.inf][:1]).all()
    assert np.isfinite(got[:, :128][~bad[:, :128]]).all() and not np.isfinite(got[:, 128:]).any()


def test_product_writes_nothing_else(dev, rng):
    for M, N, K in ((1, 37, 144), (16, 130, 128), (50, 65, 256), (100, 129, 272), (600, 257, 128)):
        W, X = on(dev, matrix(rng, N, K)), on(dev, fp8.quant(rng.standard_normal((M, K)).astype(np.float32)))
        buf = torch.full((M * N + 512,), 7.0, device=dev)
        ops.gemm_fp8(*W, *X, out=buf[256:256 + M * N].view(M, N))
        assert (buf[:256] == 7).all() and (buf[256 + M * N:] == 7).all()


def test_rows_do_not_depend_on_their_neighbours_values(dev, rng):
    """A row's result is the same whatever the other rows hold (NaN included)."""
    N, K = 300, 640
    W = on(dev, normal_matrix(rng, N, K))
    for M in (5, 40, 100, 600):
        x = rng.standard_normal((M, K)).astype(np.float32)
        a = ops.gemm_fp8(*W, *on(dev, fp8.quant(x)))
        x[:M // 2] = np.nan
        b = ops.gemm_fp8(*W, *on(dev, fp8.quant(x)))
        assert torch.equal(a[M // 2:], b[M // 2:]) and b[:M // 2].isnan().all()


# ---- linear ---------------------------------------------------------------------------------------

@pytest.mark.parametrize("x", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("y", ["bf16", "f32"])
@pytest.mark.parametrize("M,N,K", [(1, 9, 144), (1, 1000, 2560), (3, 130, 1040), (16, 257, 2576), (17, 64, 272), (64, 300, 512), (130, 140, 384)])
def test_linear(dev, rng, M, N, K, x, y):
    """The quantizer and the product, from slices of a wider matrix as from whole rows."""
    wc, ws = normal_matrix(rng, N, K)
    layer = ops.Fp8Linear(*on(dev, (wc, ws)), max_rows=M + 3)
    wide = torch.from_numpy(rng.standard_normal((M, K + 64)).astype(np.float32)).to(DT[x]).to(dev)
    X = wide[:, 32:32 + K]
    want, tol = product_bound(*fp8.quant(X.float().cpu().numpy()), wc, ws, y)
    for v in (X, X.contiguous()):
        got = layer(v, y_dtype=DT[y]).double().cpu().numpy()
        assert (np.abs(got - want) <= tol).all()
    if M == 1:
        assert torch.equal(layer(X[0], y_dtype=DT[y]), layer(X, y_dtype=DT[y]))


def test_linear_same_as_its_parts(dev, rng):
    for M in (1, 2, 16, 30, 64, 200):
        W = on(dev, normal_matrix(rng, 520, 1296))
        X = torch.randn(M, 1296, device=dev, dtype=torch.bfloat16)
        r = torch.randn(M, 520, device=dev)
        layer = ops.Fp8Linear(*W, max_rows=200)
        a, b = layer(X, residual=r), ops.gemm_fp8(*W, *ops.quant_fp8(X), residual=r)
        assert (a - b).abs().max() <= 2e-5  # (K may be split in another way: 1296 terms below 4 rms, 2^-24 each)
        out = torch.empty(M, 520, device=dev)
        assert layer(X, residual=r, out=out) is out and torch.equal(out, a)


def test_linear_refuses(dev, rng):
    layer = ops.Fp8Linear(*on(dev, matrix(rng, 20, 128)), max_rows=4)
    X = torch.randn(5, 128, device=dev)
    with pytest.raises(ValueError, match="5 rows"):
        layer(X)
    with pytest.raises(ValueError, match="consecutive"):
        layer(torch.randn(128, 4, device=dev).t())
    with pytest.raises(_lib.VybdqError, match="x_dt"):
        layer(X[:2].double())
    with pytest.raises(ValueError, match="residual"):
        layer(X[:2], residual=torch.zeros(2, 20, device=dev, dtype=torch.half))
    with pytest.raises(_lib.VybdqError, match="16-byte"):
        layer(torch.randn(4, 130, device=dev)[:, 1:129])
    assert layer(X[:0]).shape == (0, 20)


def test_linear_on_a_stream_of_its_own_and_in_a_graph(dev, rng):
    layers = [ops.Fp8Linear(*on(dev, normal_matrix(rng, K, K)), max_rows=40) for K in (512, 512)]
    x = torch.randn(40, 512, device=dev, dtype=torch.bfloat16)

    def step(v):
        return layers[1](layers[0](v, y_dtype=torch.bfloat16), y_dtype=torch.bfloat16, residual=v)

    for M in (1, 40):
        want = [step(x[:M] * i) for i in (1, 2, 3)]
        torch.cuda.synchronize()
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            got = step(x[:M])
        s.synchronize()
        assert torch.equal(got, want[0])
        v = x[:M].clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = step(v)
        for i in (1, 2, 3):
            v.copy_(x[:M] * i)
            g.replay()
            assert torch.equal(y, want[i - 1])
            assert torch.equal(step(x[:M]), want[0])


# ---- router ---------------------------------------------------------------------------------------

def check_route(dev, logits, k, bias=None, dt=torch.float32, **kw):
    l = torch.from_numpy(np.asarray(logits)).to(dt)
    b = None if bias is None else to(dev, np.asarray(bias, np.float32))
    idx, w = ops.moe_route(l.to(dev), k, bias=b, **kw)
    kw = dict(kw)
    want = fp8.route(l.double().numpy(), k, None if bias is None else np.asarray(bias, np.float32), softmax=kw.pop("score", "sigmoid") == "softmax", **kw)
    np.testing.assert_array_equal(idx.cpu().numpy(), want[0])
    # float64 throughout and one rounding: half a step of float32, and float64's own noise
    np.testing.assert_allclose(w.cpu().numpy(), want[1], rtol=2.0 ** -24 * 1.001, atol=1e-44)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("E,groups,top,per,k", [(256, 8, 4, 2, 8), (256, 1, 1, 2, 8), (160, 8, 3, 1, 6), (64, 64, 5, 2, 5), (1, 1, 1, 2, 1),
                                                (63, 9, 4, 2, 28), (1023, 33, 7, 2, 64), (1024, 2, 1, 1, 64), (7, 7, 7, 1, 7),
                                                (100, 50, 50, 2, 64), (330, 3, 2, 2, 16)])
def test_route(dev, rng, score, renorm, E, groups, top, per, k):
    for T, bias in ((1, None), (13, rng.standard_normal(E) * 0.1), (70, None)):
        check_route(dev, rng.standard_normal((T, E)) * 2, k, bias, score=score, renorm=renorm, groups=groups, top_groups=top,
                    group_top=per, scale=1.7)


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16, torch.float64])
def test_route_types_with_ties(dev, rng, dt):
    # few distinct values: ties between experts and between groups everywhere
    logits = rng.integers(-2, 3, (40, 96)).astype(np.float64)
    for score in ("sigmoid", "softmax"):
        check_route(dev, logits, 9, dt=dt, score=score, groups=8, top_groups=3, group_top=1)
        check_route(dev, logits, 9, dt=dt, score=score, groups=1, renorm=False)
        check_route(dev, logits, 9, np.zeros(96), dt=dt, score=score, groups=12, top_groups=5)


@pytest.mark.parametrize("E,groups,top,k", [(300, 1, 1, 64), (512, 1, 1, 9), (400, 2, 1, 40), (1000, 4, 2, 64), (600, 1, 1, 20)])
def test_route_ties_among_a_lanes_entries(dev, rng, E, groups, top, k):
    # (5 to 8 entries to a lane, then more: equal values in one lane, in several, and NaN, which come last)
    logits = rng.integers(-1, 2, (20, E)).astype(np.float64)
    logits[10:, ::2] = -np.inf
    check_route(dev, logits, k, dt=torch.bfloat16, score="softmax", groups=groups, top_groups=top, group_top=1)
    logits[15:, 1::3] = np.nan
    check_route(dev, logits, k, dt=torch.float16, groups=groups, top_groups=top, group_top=1)
    check_route(dev, logits[:15], k, np.zeros(E), dt=torch.float32, groups=groups, top_groups=top)


def test_route_masked_and_saturated(dev, rng):
    logits = rng.standard_normal((12, 64)).astype(np.float32)
    logits[0] = -np.inf                     # nothing left: weights 0
    logits[1, 8:] = -np.inf                 # one group left
    logits[2] = 80.0                        # sigmoid is 1 everywhere
    logits[3] = np.linspace(700, 900, 64)   # saturated, still in order
    logits[4] = -np.linspace(700, 900, 64)
    logits[5, ::2] = -np.inf
    logits[6] = 3e38
    logits[7, 5] = np.nan
    masked = np.where(rng.random(64) < 0.5, -np.inf, 0.1).astype(np.float32)
    for score in ("sigmoid", "softmax"):
        for renorm in (True, False):
            for rows in (logits[:7], logits[7:8] if score == "sigmoid" else logits[8:]):
                for bias in (None, masked):
                    kw = dict(score=score, renorm=renorm, scale=1.0)
                    check_route(dev, rows, 6, bias, **kw)
                    check_route(dev, rows, 6, bias, groups=8, top_groups=2, group_top=1, **kw)
    idx, w = ops.moe_route(to(dev, logits[7:8]), 4, score="softmax", renorm=False)
    assert w.isnan().all() and 5 not in idx.tolist()[0]


def test_route_default_arguments_are_the_plain_router(dev, rng):
    logits = to(dev, rng.standard_normal((30, 128)).astype(np.float32))
    bias = to(dev, (rng.standard_normal(128) * 0.1).astype(np.float32))
    for b in (None, bias):
        a, c = ops.moe_route(logits, 8, bias=b), ops.moe_route(logits, 8, bias=b, groups=4, top_groups=4)
        assert torch.equal(a[0], c[0]) and torch.equal(a[1], c[1])


def test_route_of_many_tokens(dev, rng):
    check_route(dev, rng.standard_normal((2500, 64)), 4, groups=4, top_groups=2, dt=torch.bfloat16)
    assert ops.moe_route(torch.zeros(0, 64, device=dev), 4, groups=4, top_groups=2)[0].shape == (0, 4)


# ---- layer ----------------------------------------------------------------------------------------

def certain_experts(rng, E, H, I):
    """Gate and up of three entries -1 or 1 to a row: with whole-number x up to 3 their products are whole numbers up to 9, exact in
    float32 on both instructions, and the activation has few values, all away from the borders between codes."""
    def sparse(n, k):
        w = np.zeros((E, n, k))
        for e in range(E):
            for r in range(n):
                w[e, r, rng.choice(k, 3, replace=False)] = rng.choice([-1.0, 1.0], 3)
        return fp8.e4m3_encode(w), np.ones((E, fp8.blocks(n), fp8.blocks(k)), np.float32)
    return sparse(I, H), sparse(I, H), normal_matrix(rng, H, I, (E,))


def near_a_border(gate, up, x, limit):
    """Whether some activation lies so near the border between two codes that float32 could go either way."""
    xq = fp8.activations(*fp8.quant(x))
    for e in range(gate[0].shape[0]):
        g, u = xq @ fp8.weights(gate[0][e], gate[1][e]).T, xq @ fp8.weights(up[0][e], up[1][e]).T
        g, u = np.minimum(g, limit), np.clip(u, -limit, limit)
        a = g / (1 + np.exp(-g)) * u
        lo, hi = fp8.quant(a * (1 - 4e-6)), fp8.quant(a * (1 + 4e-6))
        if (lo[0] != hi[0]).any() or (lo[1] != hi[1]).any():
            return True
    return False


def one(pair, e=0):
    return pair[0][e], pair[1][e]


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("T,E,k,H,I,shared", [(1, 6, 3, 256, 128, True), (2, 4, 2, 384, 256, False), (5, 8, 8, 128, 128, True),
                                              (33, 5, 2, 640, 384, True), (300, 4, 3, 256, 256, True), (150, 1, 1, 128, 128, False),
                                              (700, 3, 2, 256, 128, True)])
def test_layer_where_codes_are_certain(dev, rng, T, E, k, H, I, shared, out):
    gate, up, down = certain_experts(rng, E + 1, H, I)
    x = rng.integers(-3, 4, (T, H)).astype(np.float32)
    for limit in (7.0, 2.5, math.inf):
        assert not near_a_border(gate, up, x, limit)
        logits = rng.standard_normal((T, E)).astype(np.float32)
        idx, w = fp8.route(logits, k, scale=1.5)
        cut = [(c[:E], s[:E]) for c, s in (gate, up, down)]
        last = [one(m, E) for m in (gate, up, down)] if shared else None
        want = fp8.moe(x, idx, w.astype(np.float32), *cut, shared=last, limit=limit)
        layer = ops.MoeFp8Layer(*[on(dev, m) for m in cut], topk=k, shared=[on(dev, m) for m in last] if shared else None, scale=1.5,
                                limit=limit)
        got, gi, gw = layer(to(dev, x), to(dev, logits), out_dtype=DT[out], routing=True)
        np.testing.assert_array_equal(gi.cpu().numpy(), idx)
        # down: the product's bound per row, summed with the weights; then k + 1 float32 terms
        tol, size = np.zeros((T, H)), np.zeros((T, H))
        xq = fp8.activations(*fp8.quant(x))
        for e in range(E + 1 if shared else E):
            g, u = xq @ fp8.weights(*one(gate, e)).T, xq @ fp8.weights(*one(up, e)).T
            a = np.minimum(g, limit) / (1 + np.exp(-np.minimum(g, limit))) * np.clip(u, -limit, limit)
            we = (w * (idx == e)).sum(1) if e < E else np.ones(T)
            hit = np.nonzero(we)[0]
            for r0 in range(0, len(hit), 64):
                r = hit[r0:r0 + 64]
                y, t = product_bound(*fp8.quant(a[r]), *one(down, e), "f32" if out == "f32" else "bf16")
                t -= HALF["f32" if out == "f32" else "bf16"] * np.abs(y) * 0.99  # (rows are kept in float32)
                tol[r] += we[r, None] * t
                size[r] += we[r, None] * np.abs(y)
        tol += (k + 3) * 2.0 ** -24 * size + HALF[out] * (np.abs(want) + tol)
        err = np.abs(got.double().cpu().numpy() - want)
        assert (err <= tol).all(), (err / tol).max()


@pytest.mark.parametrize("x", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("T,E,k,H,I", [(1, 16, 4, 1024, 512), (9, 16, 4, 1024, 512), (64, 8, 2, 768, 256), (400, 8, 3, 512, 384),
                                       (1200, 4, 2, 512, 256)])
def test_layer(dev, rng, T, E, k, H, I, x):
    """Float32 noise of gate and up moves an activation to the next code with a probability of its size over a code's step:
    2^-16 (the e4m3 instruction, of the row's rms) over about 1 / 11 of the value, about 2e-4 of all, each by 1 / 11: 1.3e-3 of
    the rms. Held to 4e-3 with the bf16 rounding (1.1e-3), and the worst of a row to 10 times that."""
    gate, up, down = (normal_matrix(rng, n, m, (E,)) for n, m in ((I, H), (I, H), (H, I)))
    shared = [one(normal_matrix(rng, n, m, (1,))) for n, m in ((I, H), (I, H), (H, I))]
    X = torch.from_numpy(rng.standard_normal((T, H)).astype(np.float32)).to(DT[x])
    logits, bias = rng.standard_normal((T, E)).astype(np.float32), (rng.standard_normal(E) * 0.05).astype(np.float32)
    kw = dict(groups=4, top_groups=max(2, -(-k * 4 // E)), group_top=min(2, E // 4))
    layer = ops.MoeFp8Layer(*[on(dev, m) for m in (gate, up, down)], topk=k, shared=[on(dev, m) for m in shared], bias=to(dev, bias),
                            score="softmax", renorm=False, scale=2.0, **kw)
    idx, w = fp8.route(logits, k, bias, 2.0, softmax=True, renorm=False, **kw)
    want = fp8.moe(X.float().numpy(), idx, w, gate, up, down, shared)
    got, gi, gw = layer(X.to(dev), to(dev, logits), out_dtype=torch.bfloat16, routing=True)
    np.testing.assert_array_equal(gi.cpu().numpy(), idx)
    np.testing.assert_allclose(gw.cpu().numpy(), w, rtol=2.0 ** -24 * 1.001)
    err, rms = got.double().cpu().numpy() - want, np.sqrt((want ** 2).mean())
    assert np.sqrt((err ** 2).mean()) <= 4e-3 * rms and np.abs(err).max() <= 4e-2 * rms


def small_layer(dev, rng, E=8, H=256, I=256, **kw):
    pairs = [on(dev, normal_matrix(rng, n, m, (E,))) for n, m in ((I, H), (I, H), (H, I))]
    return ops.MoeFp8Layer(*pairs, topk=2, shared=[(c[0], s[0]) for c, s in pairs], **kw)


def test_layer_tokens_are_their_own(dev, rng):
    """A token's output does not depend on its neighbours, on the batch's order or on a NaN in another token; all tokens at one
    expert; the same call twice gives the same bits."""
    layer = small_layer(dev, rng)
    for T in (3, 20, 200):
        x, logits = torch.randn(T, 256, device=dev), torch.randn(T, 8, device=dev)
        a = layer(x, logits)
        assert torch.equal(a, layer(x, logits))
        p = torch.randperm(T, device=dev)
        assert torch.equal(layer(x[p].contiguous(), logits[p].contiguous()), a[p])
        y = x.clone()
        y[1, 5] = math.nan
        b = layer(y, logits)
        assert b[1].isnan().all() and torch.equal(b[0], a[0]) and torch.equal(b[2:], a[2:])
        same = logits.clone()
        same[:, 3], same[:, 6] = 9.0, 8.0
        c = layer(x, same)
        assert torch.isfinite(c).all()
        assert torch.equal(c[:1], layer(x[:1], same[:1])) or T > 3  # (another T may take other tiles)


def test_layer_empty_batch_outputs_and_refusals(dev, rng):
    layer = small_layer(dev, rng)
    x, logits = torch.randn(6, 256, device=dev), torch.randn(6, 8, device=dev)
    assert layer(x[:0], logits[:0]).shape == (0, 256)
    buf = torch.full((6 * 256 + 512,), 3.0, device=dev)
    layer(x, logits, out=buf[256:-256].view(6, 256))
    assert (buf[:256] == 3).all() and (buf[-256:] == 3).all()
    with pytest.raises(ValueError, match="x must"):
        layer(x[:, :128].contiguous(), logits)
    with pytest.raises(ValueError, match="logits must"):
        layer(x, logits[:5])
    with pytest.raises(_lib.VybdqError, match="x_dt"):
        layer(x.double(), logits)
    with pytest.raises(_lib.VybdqError, match="topk"):
        small_layer(dev, rng, groups=8, top_groups=1)(x, logits)


def test_layer_in_graphs_whose_workspace_outgrew_them(dev, rng):
    """A captured call of few tokens replays rightly after eager calls of more tokens have replaced the workspace, beside
    another graph of the same layer, with eager work between."""
    layer = small_layer(dev, rng)
    x, logits = torch.randn(300, 256, device=dev), torch.randn(300, 8, device=dev)
    ops.MoeFp8Layer.__call__(layer, x[:2], logits[:2])  # (the library is loaded before a capture)
    graphs = []
    for T in (4, 60):
        v, l = x[:T].clone(), logits[:T].clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = layer(v, l)
        graphs.append((T, v, l, g, y))
    for i in range(3):
        big = layer(x, logits)
        for T, v, l, g, y in graphs:
            v.copy_(x[i:T + i])
            l.copy_(logits[i:T + i])
            g.replay()
            assert torch.equal(y, layer(x[i:T + i].contiguous(), logits[i:T + i].contiguous()))
        assert torch.equal(big, layer(x, logits))


def test_a_block_as_a_host_runs_it(dev, rng):
    """Projection, router logits, router and experts in one stream, as a decode step and as a prompt, against the same in float64."""
    H, I, E, k = 512, 256, 16, 4
    proj = normal_matrix(rng, H, H)
    gate_w = (rng.standard_normal((E, H)) / math.sqrt(H)).astype(np.float32)
    gate, up, down = (normal_matrix(rng, n, m, (E,)) for n, m in ((I, H), (I, H), (H, I)))
    lin = ops.Fp8Linear(*on(dev, proj), max_rows=300)
    layer = ops.MoeFp8Layer(*[on(dev, m) for m in (gate, up, down)], topk=k, groups=4, top_groups=2)
    router = to(dev, gate_w)
    for T in (1, 17, 300):
        x = torch.from_numpy(rng.standard_normal((T, H)).astype(np.float32)).bfloat16().to(dev)
        h = lin(x, y_dtype=torch.bfloat16, residual=x)
        logits = ops.router_logits(h, router)
        y, idx, w = layer(h, logits, out_dtype=torch.bfloat16, routing=True)
        hx = h.double().cpu().numpy()
        want_h, tol = product_bound(*fp8.quant(x.float().cpu().numpy()), *proj, "bf16")
        r = x.double().cpu().numpy()
        assert (np.abs(hx - want_h - r) <= tol + HALF["bf16"] * np.abs(r)).all()
        wi, ww = fp8.route(hx @ gate_w.astype(np.float64).T, k, groups=4, top_groups=2)
        np.testing.assert_array_equal(idx.cpu().numpy(), wi)
        want = fp8.moe(hx, wi, ww, gate, up, down)
        err, rms = y.double().cpu().numpy() - want, np.sqrt((want ** 2).mean())
        assert np.sqrt((err ** 2).mean()) <= 4e-3 * rms and np.abs(err).max() <= 4e-2 * rms
