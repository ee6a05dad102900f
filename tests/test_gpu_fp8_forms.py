"""8-bit floating-point weights on the GPU, form by form, on data whose result is known to the last bit or bounded by arithmetic: what
may lie beside what, what the e4m3 instruction drops, and every kernel of the pipeline going on from tile to tile."""

import math

import numpy as np
import pytest
import torch

from oracle import fp8
from oracle.kvcache import e4m3_decode
from tests import st_writer
from tests.e4m3_cases import hard_codes
from vybforge_amd import _lib, ops
from vybforge_amd.safetensors import Checkpoint

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


# ---- from tile to tile ------------------------------------------------------------------------------

CUS = 256  # a tile of the pipeline fills a CU's LDS, so this many workgroups take all tiles in turn


def force(monkeypatch, rows, splits, M, N, K, y, more=1.0):
    """Force tiles of `rows` x 256 and splits of K, and see that the product takes them, more than `more` to a workgroup."""
    nk = -(-K // 128)
    assert nk // splits >= 4 and (rows < 192 or y in ("f16", "bf16")) and (rows != 192 or K % 128 == 0)
    assert splits == 1 or (M <= 1024 and splits <= min(nk // 4, 16) and splits * M * N * 4 <= 1 << 26)
    assert -(-M // rows) * -(-N // 256) * splits > more * CUS
    monkeypatch.setenv("VYBDQ_FP8_TILE", f"{rows},{splits}")


TILES = [(64, 1, 512, "bf16"), (64, 1, 528, "bf16"), (64, 1, 640, "f32"), (64, 1, 656, "f32"), (128, 1, 640, "bf16"), (128, 1, 624, "f16"),
         (128, 1, 512, "f32"), (128, 1, 528, "f64"), (192, 1, 512, "f16"), (192, 1, 640, "bf16"), (192, 1, 896, "bf16"),
         (256, 1, 512, "bf16"), (256, 1, 528, "bf16"), (256, 1, 640, "f16"), (256, 1, 1008, "bf16")]


@pytest.mark.parametrize("N", [17988, 17989])
@pytest.mark.parametrize("rows,splits,K,y", TILES)
def test_product_from_tile_to_tile(dev, rng, monkeypatch, rows, splits, K, y, N):
    M = 9 * rows + 5
    force(monkeypatch, rows, splits, M, N, K, y, more=2.5)
    W, Ws, X, Xs, want = whole_product(rng, M, N, K, dev)
    r = torch.randint(-99, 100, (M, N), device=dev).to(DT[y])
    got = ops.gemm_fp8(W, Ws, X, Xs, y_dtype=DT[y], residual=r)
    assert torch.equal(got, (want + r.double()).to(DT[y]))
    assert ops.gemm_fp8(W, Ws, X, Xs, y_dtype=DT[y], residual=r, out=r) is r and torch.equal(r, got)


@pytest.mark.parametrize("N", [8988, 8990])
@pytest.mark.parametrize("K", [1776, 1792])  # 14 blocks, 4, 5 and 5 to a split
@pytest.mark.parametrize("rows,y", [(64, "bf16"), (64, "f32"), (128, "f16"), (128, "f64"), (192, "bf16"), (256, "bf16")])
def test_split_product_from_tile_to_tile(dev, rng, monkeypatch, rows, y, K, N):
    if rows == 192 and K % 128:
        K = 1920  # (that tile takes whole blocks: 5 to each split)
    M = 600
    force(monkeypatch, rows, 3, M, N, K, y)
    W, Ws, X, Xs, want = whole_product(rng, M, N, K, dev)
    r = torch.randint(-99, 100, (M, N), device=dev).to(DT[y])
    work = ops.Fp8Workspace([(M, N, K)], dev)
    work.buf.fill_(0x7f)
    got = ops.gemm_fp8(W, Ws, X, Xs, y_dtype=DT[y], residual=r, workspace=work)
    assert torch.equal(got, (want + r.double()).to(DT[y]))


def test_scales_far_apart(dev, rng):
    """The scales' products are formed before they meet a sum: 2^100 and 2^-100 leave nothing behind."""
    for M, N, K in ((1, 50, 640), (70, 300, 640), (300, 300, 256)):
        W, Ws, X, Xs, want = whole_product(rng, M, N, K, dev)
        for e in (100, -100):
            for y in ("f32", "bf16"):
                got = ops.gemm_fp8(W, Ws * 2.0 ** e, X, Xs * 2.0 ** -e, y_dtype=DT[y])
                assert torch.equal(got, want.to(DT[y]))


def test_products_of_one_workspace_in_a_graph(dev, rng, monkeypatch):
    """Split products of two layers, one after the other through one workspace, captured and replayed with eager work between."""
    M, K = 200, 2048
    layers, wants = [], []
    work = ops.Fp8Workspace([(M, K, K)], dev)
    for _ in range(2):
        W, Ws = whole(rng, K, K, 2, dev), powers(rng, (K // 128, K // 128), dev)
        layers.append(ops.Fp8Linear(W, Ws, max_rows=M, workspace=work))
    step = lambda v: layers[1](layers[0](v, y_dtype=torch.bfloat16), y_dtype=torch.bfloat16, residual=v)
    x = torch.randn(3, M, K, device=dev).bfloat16()
    for tile in ("64,3", "128,4"):
        monkeypatch.setenv("VYBDQ_FP8_TILE", tile)
        wants, v = [step(x[i]) for i in range(3)], x[0].clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = step(v)
        for i in (0, 1, 2, 1):
            v.copy_(x[i])
            g.replay()
            assert torch.equal(y, wants[i])
            assert torch.equal(step(x[0]), wants[0])


# ---- the experts' layer -----------------------------------------------------------------------------

def sparse(rng, E, n, k):
    """Codes [E, n, k] with three entries -1 or 1 to a row: products with whole numbers up to 3 are whole numbers up to 9."""
    c = np.zeros((E * n, k), np.uint8)
    first, step = rng.integers(0, k, E * n), rng.integers(1, k // 3, (2, E * n))
    for at in (first, first + step[0], first + step[0] + step[1]):
        c[np.arange(E * n), at % k] = np.where(rng.random(E * n) < 0.5, 0x38, 0xb8)
    return c.reshape(E, n, k), np.ones((E, fp8.blocks(n), fp8.blocks(k)), np.float32)


def normal(rng, E, n, k):
    c = np.stack([fp8.e4m3_encode(np.clip(rng.standard_normal((n, k)) * 110, -448, 448)) for _ in range(E)])
    return c, (rng.uniform(0.5, 1.5, (E, fp8.blocks(n), fp8.blocks(k))) / (110 * math.sqrt(k))).astype(np.float32)


def on(dev, pair):
    return torch.from_numpy(pair[0]).to(dev).view(E4M3), torch.from_numpy(pair[1]).to(dev)


def weights64(pair, e, dev):
    return torch.from_numpy(fp8.weights(pair[0][e], pair[1][e])).to(dev)


def expert(x, gate, up, down, e, limit, out, dev):
    """float64 output rows [t, H] of expert e, what separates the kernel's float32 rows from them, and their magnitude. No activation
    may lie so near the border between two codes (4e-6 of it) that float32 could go either way."""
    g, u = (x @ weights64(p, e, dev).t() for p in (gate, up))
    g, u = g.clamp(max=limit), u.clamp(-limit, limit)
    a = (g / (1 + torch.exp(-g)) * u).cpu().numpy()
    codes, scales = fp8.quant(a)
    for f in (1 - 4e-6, 1 + 4e-6):
        c, s = fp8.quant(a * f)
        assert (c == codes).all() and (s == scales).all()
    a, w = torch.from_numpy(fp8.activations(codes, scales)).to(dev), weights64(down, e, dev)
    tol = (130 + scales.shape[1]) * 2.0 ** -23 * (a.abs() @ w.abs().t())
    if out != "f32":  # the instruction's loss: 2^-10 of the sum of magnitudes, subnormal codes counted as 2^-6
        size = lambda c, s: np.where(c & 0x7f, np.maximum(np.abs(e4m3_decode(c)), 2.0 ** -6), 0) * s
        sa = torch.from_numpy(size(codes, scales.astype(np.float64).repeat(128, 1))).to(dev)
        sw = torch.from_numpy(size(down[0][e], down[1][e].astype(np.float64).repeat(128, 0).repeat(128, 1))).to(dev)
        tol += 2.0 ** -10 * (sa @ sw.t())
    y = a @ w.t()
    return y, tol, y.abs()


# tiles of 128 and of 64 rows, three blocks of K (the pipeline's least) and more, experts of a few rows and of many; `one`: all tokens
# at the same experts
LAYERS = [(6000, 4, 2, 384, 384, True, 128, ""), (5000, 5, 2, 896, 640, False, 128, ""), (2000, 64, 2, 384, 384, True, 64, ""),
          (1500, 64, 2, 896, 640, False, 64, ""), (1500, 64, 2, 896, 640, True, 64, "one"), (200, 8, 2, 384, 384, False, 64, "one"),
          (20, 8, 2, 640, 384, True, 16, "one")]


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("T,E,k,H,I,shared,rows,where", LAYERS)
def test_layer_from_tile_to_tile(dev, rng, T, E, k, H, I, shared, rows, where, out):
    n, hit, limit = T * k, min(E, T * k), 7.0
    assert rows == (16 if n <= 8 * hit else 64 if n <= 64 * hit else 128)
    logits = rng.standard_normal((T, E)).astype(np.float32) + np.linspace(-1.5, 1.5, E, dtype=np.float32)[rng.permutation(E)]
    if where == "one":
        logits[:, 3], logits[:, 6] = 9.0, 8.0
    idx, w = fp8.route(logits, k, scale=1.5)
    count = np.bincount(idx.reshape(-1), minlength=E)
    if where == "" and T > 1000:
        tiles = (-(-count // rows)).sum() + (-(-T // rows) if shared else 0)
        assert tiles * (I // 128) > CUS and tiles * -(-H // 256) > CUS
        assert count.max() > 128 and (rows == 128 or count[count > 0].min() < 32)
    gate, up, down = sparse(rng, E + 1, I, H), sparse(rng, E + 1, I, H), normal(rng, E + 1, H, I)
    x = rng.integers(-3, 4, (T, H)).astype(np.float32)
    cut = [on(dev, (c[:E], s[:E])) for c, s in (gate, up, down)]
    layer = ops.MoeFp8Layer(*cut, topk=k, shared=[on(dev, (c[E], s[E])) for c, s in (gate, up, down)] if shared else None, scale=1.5,
                            limit=limit)
    xd, ld = torch.from_numpy(x).to(dev), torch.from_numpy(logits).to(dev)
    got, gi, gw = layer(xd, ld, out_dtype=DT[out], routing=True)
    np.testing.assert_array_equal(gi.cpu().numpy(), idx)
    np.testing.assert_allclose(gw.cpu().numpy(), w, rtol=2.0 ** -24 * 1.001)
    want, tol, size = (torch.zeros(T, H, dtype=torch.float64, device=dev) for _ in range(3))
    wd = gw.double().cpu().numpy()
    for e in range(E + 1 if shared else E):
        share = (wd * (idx == e)).sum(1) if e < E else np.ones(T)
        t = torch.from_numpy(np.nonzero(share)[0]).to(dev)
        if len(t):
            f = torch.from_numpy(share).to(dev)[t, None]
            for total, part in zip((want, tol, size), expert(xd[t].double(), gate, up, down, e, limit, out, dev)):
                total[t] += f * part
    tol += (k + 3) * 2.0 ** -24 * size  # the weighted sum, in float32
    tol += HALF[out] * (want.abs() + tol)
    err = (got.double() - want).abs()
    assert (err <= tol).all(), (err / tol).max()
    assert torch.equal(layer(xd, ld, out_dtype=DT[out]), got)  # whichever workgroup is the faster one


@pytest.mark.parametrize("T,times", [(8, 10), (64, 4), (400, 1)])
def test_activations_of_gate_and_up_keep_their_codes(dev, rng, T, times):
    """Down is the identity and the one expert's weight 1, so the float32 output is the quantized activation itself. Gate and up on fp16
    instructions are off by 1e-7 of their rms, exponential, division and products by 3e-7: an activation moves to the next code with
    a probability of 4e-7 over a step of 1/8 to 1/16 of it, about 1 in 200000 (1 in 5000 had the e4m3 instruction taken the sums).
    10 of 200000 are allowed, each by one code."""
    H = I = 512
    eye = np.zeros((1, H, I), np.uint8)
    eye[0, np.arange(H), np.arange(H)] = 0x38
    moved = total = 0
    for _ in range(times):
        gate, up = normal(rng, 1, I, H), normal(rng, 1, I, H)
        layer = ops.MoeFp8Layer(on(dev, gate), on(dev, up), on(dev, (eye, np.ones((1, 4, 4), np.float32))), topk=1, scale=1.0)
        x = rng.standard_normal((T, H)).astype(np.float32)
        got, _, w = layer(torch.from_numpy(x).to(dev), torch.zeros(T, 1, device=dev), routing=True)
        assert (w == 1).all()
        xq = fp8.activations(*fp8.quant(x))
        g, u = (xq @ fp8.weights(p[0][0], p[1][0]).T for p in (gate, up))
        g, u = np.minimum(g, 10.0), np.clip(u, -10.0, 10.0)
        codes, scales = fp8.quant(g / (1 + np.exp(-g)) * u)
        scales = scales.astype(np.float64).repeat(128, 1)
        have = fp8.e4m3_encode(got.double().cpu().numpy() / scales)
        np.testing.assert_array_equal(e4m3_decode(have) * scales, got.double().cpu().numpy())
        other = e4m3_decode(have) != e4m3_decode(codes)
        assert (np.abs((have & 0x7f).astype(int) - (codes & 0x7f).astype(int))[other] == 1).all()
        moved, total = moved + other.sum(), total + other.size
    assert moved <= max(1, 10 * total // 200000), (moved, total)


def small_layer(dev, rng, E, H, I, k, shared=True, **kw):
    """A layer, its host pairs (E + 1 experts, the last one shared) and whole-number tokens for it."""
    pairs = sparse(rng, E + 1, I, H), sparse(rng, E + 1, I, H), normal(rng, E + 1, H, I)
    layer = ops.MoeFp8Layer(*[on(dev, (c[:E], s[:E])) for c, s in pairs], topk=k, limit=7.0,
                            shared=[on(dev, (c[E], s[E])) for c, s in pairs] if shared else None, **kw)
    return layer, pairs, lambda T: torch.from_numpy(rng.integers(-3, 4, (T, H)).astype(np.float32)).to(dev)


@pytest.mark.parametrize("T", [2, 30, 200])
def test_layer_inputs_of_every_type(dev, rng, T):
    """Tokens and logits that every type holds give the same bits in every type; 16-bit outputs are one sum, rounded to each."""
    layer, _, tokens = small_layer(dev, rng, 8, 384, 256, 3)
    x, logits = tokens(T), torch.randn(T, 8, device=dev).bfloat16()
    for out in ("f32", "f16", "bf16"):
        want = layer(x, logits.float(), out_dtype=DT[out])
        for a in (torch.float32, torch.float16, torch.bfloat16):
            for b in (torch.float64, torch.float32, torch.float16, torch.bfloat16):
                if b != torch.float16 or (logits.to(b).bfloat16() == logits).all():
                    assert torch.equal(layer(x.to(a), logits.to(b), out_dtype=DT[out]), want), (a, b)
    h, b = (layer(x, logits, out_dtype=DT[d]).double() for d in ("f16", "bf16"))
    assert ((h - b).abs() <= (2.0 ** -8 + 2.0 ** -10) * b.abs() + 2.0 ** -24).all()


@pytest.mark.parametrize("T", [1, 5, 40])
def test_layer_gives_either_part_of_its_routing(dev, rng, T):
    layer, _, tokens = small_layer(dev, rng, 8, 256, 128, 2, shared=False, scale=1.5)
    x, logits = tokens(T), torch.randn(T, 8, device=dev)
    want, idx, w = layer(x, logits, routing=True)
    ws, n = layer._workspace(T)
    for give_idx, give_w in ((True, False), (False, True), (False, False)):
        out, i, v = torch.empty_like(want), torch.full_like(idx, -7), torch.full_like(w, -7)
        ops.call("vybdq_moe_forward_fp8", x.data_ptr(), _lib.F32, logits.data_ptr(), _lib.F32, 0, *layer._w, out.data_ptr(), _lib.F32,
                 i.data_ptr() if give_idx else 0, v.data_ptr() if give_w else 0, T, 256, 128, 8, 2, 1.5, 7.0, 0, 1, 1, 1, 2, ws, n, stream())
        assert torch.equal(out, want)
        assert torch.equal(i, idx if give_idx else torch.full_like(idx, -7))
        assert torch.equal(v, w if give_w else torch.full_like(w, -7))


@pytest.mark.parametrize("E,k,kw", [(1024, 64, {}), (1000, 8, dict(groups=8, top_groups=3)), (96, 1, {}), (1024, 1, dict(groups=64, top_groups=9))])
@pytest.mark.parametrize("T", [1, 2, 9])
def test_layer_of_many_experts(dev, rng, E, k, kw, T):
    layer, pairs, tokens = small_layer(dev, rng, E, 128, 128, k, score="softmax", renorm=False, scale=2.0, **kw)
    x, logits = tokens(T), rng.standard_normal((T, E)).astype(np.float32)
    idx, w = fp8.route(logits, k, None, 2.0, softmax=True, renorm=False, **kw)
    got, gi, gw = layer(x, torch.from_numpy(logits).to(dev), routing=True)
    np.testing.assert_array_equal(gi.cpu().numpy(), idx)
    np.testing.assert_allclose(gw.cpu().numpy(), w, rtol=2.0 ** -24 * 1.001)
    want, tol, size = expert(x.double(), *pairs, E, 7.0, "f32", dev)
    for t in range(T):
        for s in range(k):
            parts = expert(x[t:t + 1].double(), *pairs, int(idx[t, s]), 7.0, "f32", dev)
            for total, part in zip((want, tol, size), parts):
                total[t] += float(gw[t, s]) * part[0]
    tol = tol + (k + 3) * 2.0 ** -24 * size
    assert ((got.double() - want).abs() <= tol + HALF["f32"] * (want.abs() + tol)).all()


def test_layers_on_two_streams_at_once(dev, rng):
    """Two layers with workspaces of their own, call by call beside each other; then one of them moves to the other's stream and
    grows there."""
    made = [small_layer(dev, rng, 8, 512, 384, 2) for _ in range(2)]
    xs = [[(tokens(T), torch.randn(T, 8, device=dev)) for T in (3, 100, 700, 50)] for _, _, tokens in made]
    wants = [[layer(*a) for a in x] for (layer, _, _), x in zip(made, xs)]
    fresh = [ops.MoeFp8Layer(*zip(layer.tensors[0:6:2], layer.tensors[1:6:2]), topk=2, limit=7.0,
                             shared=list(zip(layer.tensors[6::2], layer.tensors[7::2]))) for layer, _, _ in made]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for j in range(4):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(fresh[i](*xs[i][j]))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g, w in zip(got, wants) for a, b in zip(g, w))
    layer = ops.MoeFp8Layer(*zip(made[0][0].tensors[0:6:2], made[0][0].tensors[1:6:2]), topk=2, limit=7.0,
                            shared=list(zip(made[0][0].tensors[6::2], made[0][0].tensors[7::2])))
    for j, s in ((1, streams[0]), (2, streams[1]), (3, streams[0])):
        for other in streams:
            s.wait_stream(other)
        with torch.cuda.stream(s):
            y = layer(*xs[0][j])
            torch.empty(layer._ws.numel() // 2, dtype=torch.uint8, device=dev).fill_(0x7f)  # (where a freed workspace may have been)
        s.synchronize()
        assert torch.equal(y, wants[0][j])


@pytest.mark.parametrize("M", [1, 3, 30, 140])
def test_linear_with_every_output(dev, rng, M):
    """Float64 outputs and residuals, one row of a wider matrix, an output in place of the residual."""
    N, K = 201, 656
    W, Ws, Xq, Xs, _ = whole_product(rng, M, N, K, dev)
    x = values(Xq, torch.ones_like(Xs), 1)
    want = x.double() @ values(W, Ws, 128).double().t()
    layer = ops.Fp8Linear(W, Ws, max_rows=M)
    wide = torch.full((M, 1024), 77.0, device=dev)
    wide[:, 16:16 + K] = x
    for y in ("f64", "f32", "f16", "bf16"):
        r = torch.randint(-9, 10, (M, N), device=dev).to(DT[y])
        for v in (wide[:, 16:16 + K], wide[:, 16:16 + K].half(), wide[M - 1:, 16:16 + K]):
            rows = slice(M - len(v), M)
            out = r[rows].clone()
            assert layer(v, y_dtype=DT[y], residual=out, out=out) is out
            assert torch.equal(out, (want[rows] + r[rows].double()).to(DT[y]))


def test_layer_from_a_checkpoint(dev, rng, tmp_path):
    """Experts that a checkpoint holds one tensor each, copied into stacked arrays."""
    E, H, I = 4, 256, 128
    pairs = [normal(rng, E, n, m) for n, m in ((I, H), (I, H), (H, I))]
    tensors = []
    for (c, s), proj in zip(pairs, ("gate_proj", "up_proj", "down_proj")):
        for e in range(E):
            tensors.append((f"mlp.experts.{e}.{proj}.weight", "F8_E4M3", list(c[e].shape), c[e].tobytes()))
            tensors.append((f"mlp.experts.{e}.{proj}.scale", s[e]))
    st_writer.write(tmp_path / "model.safetensors", tensors)
    ckpt = Checkpoint(tmp_path)

    def stacked(proj, N, K):
        codes = torch.empty(E, N, K, dtype=E4M3, device=dev)
        scales = torch.empty(E, N // 128, K // 128, device=dev)
        for e in range(E):
            codes[e].copy_(ckpt.to_device(f"mlp.experts.{e}.{proj}.weight", dev))
            scales[e].copy_(ckpt.to_device(f"mlp.experts.{e}.{proj}.scale", dev))
        return codes, scales

    layer = ops.MoeFp8Layer(stacked("gate_proj", I, H), stacked("up_proj", I, H), stacked("down_proj", H, I), topk=2)
    x, logits = torch.randn(9, H, device=dev), torch.randn(9, E, device=dev)
    assert torch.equal(layer(x, logits), ops.MoeFp8Layer(*[on(dev, p) for p in pairs], topk=2)(x, logits))
