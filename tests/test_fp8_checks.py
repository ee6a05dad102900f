"""Refusals of the 8-bit floating-point entry points (return codes before any launch, and the wrappers' checks), workspace sizes,
and the oracle's quantizer and router against plain statements of them. CPU only: no call here reaches the GPU."""

import re

import numpy as np
import pytest
import torch

from oracle import fp8, moe
from oracle.kvcache import e4m3_decode
from vybforge_amd import _lib, ops

QUANT = dict(X=16, x_dt=0, ldx=256, Xq=1 << 44, Xs=4, M=3, K=256, stream=0)
GEMM = dict(W=16, Ws=4, Xq=1 << 50, Xs=1 << 51, Y=4, M=3, N=5, K=256, y_dt=0, ldy=0, RS=0, ws=0, ws_bytes=0, stream=0)
LINEAR = dict(W=16, Ws=4, X=1 << 50, x_dt=0, ldx=256, Y=4, M=3, N=5, K=256, y_dt=0, ldy=0, RS=0, ws=256, ws_bytes=1 << 20, stream=0)
ROUTE = dict(logits=8, logits_dt=0, bias=4, idx=4, w=4, T=3, E=64, topk=4, scale=1.0, softmax=0, renorm=1, groups=8, top_groups=2,
             group_top=2, stream=0)
MOE = dict(x=16, x_dt=0, logits=8, logits_dt=0, bias=4, gate=16, gate_s=4, up=16, up_s=4, down=16, down_s=4, sg=16, sgs=4, su=16,
           sus=4, sd=16, sds=4, out=16, out_dt=0, idx=0, w=0, T=3, H=256, I=128, E=64, topk=4, scale=1.0, limit=10.0, softmax=0,
           renorm=1, groups=8, top_groups=2, group_top=2, ws=256, ws_bytes=1 << 30, stream=0)
PRODUCT = [(dict(K=250), _lib.ERR_SHAPE, "K must"), (dict(K=0), _lib.ERR_SHAPE, "K must"), (dict(K=2 ** 23), _lib.ERR_SHAPE, "K must"),
           (dict(N=0), _lib.ERR_SHAPE, "N must"), (dict(N=2 ** 24), _lib.ERR_SHAPE, "N must"), (dict(M=-1), _lib.ERR_SHAPE, "M below"),
           (dict(M=2 ** 23, N=2 ** 20), _lib.ERR_SHAPE, "2\\^22"), (dict(ldy=4), _lib.ERR_SHAPE, "ldy"), (dict(y_dt=4), _lib.ERR_ARG, "y_dt"),
           (dict(W=0), _lib.ERR_ARG, "null"), (dict(Y=0), _lib.ERR_ARG, "null"), (dict(W=24), _lib.ERR_ALIGN, "W must"),
           (dict(Y=6), _lib.ERR_ALIGN, "aligned"), (dict(Ws=6), _lib.ERR_ALIGN, "aligned"), (dict(RS=6), _lib.ERR_ALIGN, "aligned")]


def refused(name, args, change, code, text):
    assert getattr(_lib.lib, name)(*(args | change).values()) == code
    assert re.search(text, _lib.last_error()) and _lib.last_error().startswith(name)


@pytest.mark.parametrize("change,code,text", [
    (dict(x_dt=3), _lib.ERR_ARG, "x_dt"), (dict(K=24), _lib.ERR_SHAPE, "K must"), (dict(K=0), _lib.ERR_SHAPE, "K must"),
    (dict(M=-1), _lib.ERR_SHAPE, "M must"), (dict(M=2 ** 28), _lib.ERR_SHAPE, "2\\^28"), (dict(X=0), _lib.ERR_ARG, "null"),
    (dict(M=2 ** 27), _lib.ERR_SHAPE, "2\\^28"), (dict(Xs=0), _lib.ERR_ARG, "null"), (dict(ldx=255), _lib.ERR_SHAPE, "ldx"),
    (dict(ldx=257), _lib.ERR_ALIGN, "16-byte"), (dict(X=8), _lib.ERR_ALIGN, "16-byte"), (dict(Xq=8), _lib.ERR_ALIGN, "16-byte"),
    (dict(Xs=2), _lib.ERR_ALIGN, "4-byte"), (dict(x_dt=1, ldx=260), _lib.ERR_ALIGN, "16-byte"),
    (dict(Xq=16), _lib.ERR_ARG, "overlap"), (dict(X=32, Xq=16), _lib.ERR_ARG, "overlap"), (dict(Xq=16 + 2944), _lib.ERR_ARG, "overlap")])
def test_quantizer_refuses(change, code, text):
    refused("vybdq_quant_fp8", QUANT, change, code, text)


@pytest.mark.parametrize("change,code,text", PRODUCT + [
    (dict(Xq=0), _lib.ERR_ARG, "null"), (dict(Xq=24), _lib.ERR_ALIGN, "Xq"), (dict(Xs=2), _lib.ERR_ALIGN, "Xs"),
    (dict(ws=128), _lib.ERR_WORKSPACE, "workspace"), (dict(ws_bytes=-1), _lib.ERR_WORKSPACE, "workspace"),
    (dict(Xq=16, Y=16), _lib.ERR_ARG, "overlap"), (dict(Xs=60, Y=16), _lib.ERR_ARG, "overlap")])
def test_product_refuses(change, code, text):
    refused("vybdq_gemm_fp8", GEMM, change, code, text)


@pytest.mark.parametrize("change,code,text", PRODUCT + [
    (dict(x_dt=3), _lib.ERR_ARG, "x_dt"), (dict(X=0), _lib.ERR_ARG, "null"), (dict(ldx=255), _lib.ERR_SHAPE, "ldx"),
    (dict(X=8), _lib.ERR_ALIGN, "16-byte"), (dict(ldx=257), _lib.ERR_ALIGN, "16-byte"), (dict(ws=0), _lib.ERR_WORKSPACE, "workspace"),
    (dict(ws=128), _lib.ERR_WORKSPACE, "workspace"), (dict(ws_bytes=1000), _lib.ERR_WORKSPACE, "workspace"),
    (dict(M=2 ** 23, N=1, K=2 ** 16, ldx=2 ** 16), _lib.ERR_SHAPE, "2\\^28"), (dict(X=16, Y=3000), _lib.ERR_ARG, "overlap")])
def test_linear_refuses(change, code, text):
    refused("vybdq_linear_fp8", LINEAR, change, code, text)


ROUTING = [(dict(logits_dt=4), _lib.ERR_ARG, "logits_dt"), (dict(E=0), _lib.ERR_SHAPE, "E <= 1024"), (dict(groups=0), _lib.ERR_SHAPE, "groups"),
           (dict(groups=7), _lib.ERR_SHAPE, "divide E"), (dict(top_groups=0), _lib.ERR_SHAPE, "top_groups"),
           (dict(top_groups=9), _lib.ERR_SHAPE, "top_groups"), (dict(group_top=0), _lib.ERR_ARG, "group_top"),
           (dict(group_top=3), _lib.ERR_ARG, "group_top"), (dict(topk=17), _lib.ERR_SHAPE, "topk"), (dict(logits=0), _lib.ERR_ARG, "null"),
           (dict(logits=10), _lib.ERR_ALIGN, "aligned"), (dict(bias=6), _lib.ERR_ALIGN, "aligned")]


@pytest.mark.parametrize("change,code,text", ROUTING + [
    (dict(E=1025, groups=1, top_groups=1), _lib.ERR_SHAPE, "E <= 1024"), (dict(E=512, groups=128), _lib.ERR_SHAPE, "groups"), (dict(topk=0), _lib.ERR_SHAPE, "topk"),
    (dict(T=-1), _lib.ERR_SHAPE, "T below"), (dict(T=2 ** 24), _lib.ERR_SHAPE, "T below"), (dict(topk=65, E=1024), _lib.ERR_SHAPE, "topk"),
    (dict(idx=0), _lib.ERR_ARG, "null"), (dict(w=0), _lib.ERR_ARG, "null"), (dict(idx=6), _lib.ERR_ALIGN, "aligned")])
def test_router_refuses(change, code, text):
    refused("vybdq_moe_route_groups", ROUTE, change, code, text)


@pytest.mark.parametrize("change,code,text", [c for c in ROUTING if c[0] != dict(E=0)] + [
    (dict(x_dt=3), _lib.ERR_ARG, "x_dt"), (dict(out_dt=3), _lib.ERR_ARG, "out_dt"), (dict(H=192), _lib.ERR_SHAPE, "H and I"),
    (dict(I=64), _lib.ERR_SHAPE, "H and I"), (dict(T=2 ** 20), _lib.ERR_SHAPE, "tokens"), (dict(T=-1), _lib.ERR_SHAPE, "tokens"), (dict(E=1025), _lib.ERR_SHAPE, "E up"),
    (dict(sds=0), _lib.ERR_ARG, "shared"), (dict(sg=0), _lib.ERR_ARG, "shared"), (dict(x=0), _lib.ERR_ARG, "null"), (dict(gate=0), _lib.ERR_ARG, "null"),
    (dict(down_s=0), _lib.ERR_ARG, "null"), (dict(out=0), _lib.ERR_ARG, "null"), (dict(limit=0.0), _lib.ERR_ARG, "limit"),
    (dict(limit=float("nan")), _lib.ERR_ARG, "limit"), (dict(x=24), _lib.ERR_ALIGN, "16-byte"), (dict(up=24), _lib.ERR_ALIGN, "16-byte"),
    (dict(sus=6), _lib.ERR_ALIGN, "4-byte"), (dict(out=24), _lib.ERR_ALIGN, "16-byte"), (dict(ws=0), _lib.ERR_WORKSPACE, "workspace"),
    (dict(ws=128), _lib.ERR_WORKSPACE, "workspace"), (dict(ws_bytes=100), _lib.ERR_WORKSPACE, "workspace")])
def test_layer_refuses(change, code, text):
    refused("vybdq_moe_forward_fp8", MOE, change, code, text)


def test_nothing_to_do_is_no_launch():
    assert _lib.lib.vybdq_quant_fp8(*(QUANT | dict(M=0, X=0, Xq=0, Xs=0)).values()) == _lib.OK
    assert _lib.lib.vybdq_gemm_fp8(*(GEMM | dict(M=0, Xq=0, Y=0)).values()) == _lib.OK
    assert _lib.lib.vybdq_linear_fp8(*(LINEAR | dict(M=0, X=0, Y=0, ws=0)).values()) == _lib.OK
    assert _lib.lib.vybdq_moe_route_groups(*(ROUTE | dict(T=0, logits=0, idx=0, w=0)).values()) == _lib.OK
    assert _lib.lib.vybdq_moe_forward_fp8(*(MOE | dict(T=0, x=0, logits=0, out=0, ws=0)).values()) == _lib.OK


def test_workspace_sizes():
    part, size = _lib.lib.vybdq_gemm_fp8_workspace_size, _lib.lib.vybdq_linear_fp8_workspace_size
    for bad in ((-1, 16, 128), (1, 0, 128), (1, 16, 120), (1, 16, 0), (2 ** 24, 16, 128)):
        assert size(*bad) == part(*bad) == -1
    for N, K in ((1, 16), (1000, 2576), (17408, 5120), (300, 17408), (5, 1024)):
        rest = [part(M, N, K) for M in (0, 1, 2, 5, 16, 17, 33, 64, 65, 100, 256, 257, 600, 1024, 1025, 4096)]
        assert rest == sorted(rest) and max(rest) <= 1 << 26
        got = [size(M, N, K) for M in (0, 1, 2, 5, 16, 17, 33, 64, 65, 100, 256, 257, 600, 4096)]
        assert got == sorted(got) and got[1] >= K
    size = _lib.lib.vybdq_moe_fp8_workspace_size
    for bad in ((-1, 256, 128, 8, 2), (1, 200, 128, 8, 2), (1, 256, 64, 8, 2), (1, 256, 128, 0, 1), (1, 256, 128, 8, 9), (1, 256, 128, 1025, 8)):
        assert size(*bad) == -1
    for E, k in ((8, 2), (256, 8), (1, 1)):
        got = [size(T, 1024, 512, E, k) for T in (0, 1, 2, 7, 8, 9, 31, 32, 33, 64, 65, 200, 512, 513, 4000)]
        assert got == sorted(got)


def cpu(*shape, dtype=torch.float32):
    return torch.zeros(shape).to(dtype)


def test_wrappers_refuse():
    e = torch.float8_e4m3fn
    W, Ws = cpu(5, 256, dtype=e), cpu(1, 2)
    with pytest.raises(ValueError, match="float8"):
        ops.Fp8Linear(cpu(5, 256), Ws)
    with pytest.raises(ValueError, match="scales must be"):
        ops.Fp8Linear(W, cpu(2, 2))
    with pytest.raises(ValueError, match="scales must be"):
        ops.Fp8Linear(W, cpu(1, 2, dtype=torch.float64))
    with pytest.raises(ValueError, match="multiple of 16"):
        ops.Fp8Linear(cpu(5, 40, dtype=e), cpu(1, 1))
    with pytest.raises(ValueError, match="contiguous"):
        ops.Fp8Linear(cpu(256, 16, dtype=e).t(), cpu(1, 2))
    with pytest.raises(ValueError, match="unsupported"):
        ops.Fp8Linear(W, Ws, max_rows=-1)
    with pytest.raises(ValueError, match="Xq must"):
        ops.gemm_fp8(W, Ws, cpu(3, 128, dtype=e), cpu(3, 2))
    with pytest.raises(ValueError, match="Xs must"):
        ops.gemm_fp8(W, Ws, cpu(3, 256, dtype=e), cpu(2, 3))
    with pytest.raises(ValueError, match="GPU"):
        ops.quant_fp8(cpu(3, 256))
    layer = ops.Fp8Linear(W, Ws)
    with pytest.raises(ValueError, match="X must be"):
        layer(cpu(3, 128))
    with pytest.raises(ValueError, match="GPU"):
        layer(cpu(3, 256))
    with pytest.raises(ValueError, match="score"):
        ops.moe_route(cpu(3, 8), 2, score="relu")
    gate, up = ((cpu(4, 128, 256, dtype=e), cpu(4, 1, 2)) for _ in range(2))
    down = (cpu(4, 256, 128, dtype=e), cpu(4, 2, 1))
    with pytest.raises(ValueError, match="down must"):
        ops.MoeFp8Layer(gate, up, gate)
    with pytest.raises(ValueError, match="scales must"):
        ops.MoeFp8Layer(gate, (up[0], cpu(4, 2, 1)), down)
    with pytest.raises(ValueError, match="shared down"):
        ops.MoeFp8Layer(gate, up, down, shared=[(cpu(128, 256, dtype=e), cpu(1, 2))] * 3)
    with pytest.raises(ValueError, match="bias"):
        ops.MoeFp8Layer(gate, up, down, bias=cpu(5))


# ---- the oracle ---------------------------------------------------------------------------------

def test_oracle_quantizer_rounds_once_to_the_nearest_code(rng):
    x = (rng.standard_normal((40, 300)) * 2.0 ** rng.integers(-30, 30, (40, 1))).astype(np.float32)
    codes, scales = fp8.quant(x)
    values = np.sort(e4m3_decode(np.delete(np.arange(256), (0x7f, 0xff)).astype(np.uint8)))
    for m in range(40):
        for b in range(3):
            part, s = x[m, 128 * b:128 * (b + 1)].astype(np.float64), float(scales[m, b])
            assert np.frexp(s)[0] == 0.5 and np.abs(part).max() <= 448 * s and np.abs(part).max() > 224 * s
            near = np.abs(part[:, None] / s - values[None]).min(1)
            np.testing.assert_allclose(np.abs(part / s - e4m3_decode(codes[m, 128 * b:128 * (b + 1)])), near, rtol=0, atol=0)


def test_oracle_router_is_the_plain_one_without_groups(rng):
    logits, bias = rng.standard_normal((50, 37)), rng.standard_normal(37) * 0.1
    for b in (None, bias):
        want, got = moe.route_logits(logits, 5, b, 2.5), fp8.route(logits, 5, b, 2.5)
        np.testing.assert_array_equal(want[0], got[0])
        np.testing.assert_allclose(want[1], got[1], rtol=1e-14)
    i, w = fp8.route(logits, 5, None, 1.0, softmax=True, renorm=False)
    p = np.exp(logits) / np.exp(logits).sum(1, keepdims=True)
    np.testing.assert_allclose(w, np.take_along_axis(p, i, 1), rtol=1e-13)
    np.testing.assert_array_equal(i, moe.route_logits(logits, 5)[0])
