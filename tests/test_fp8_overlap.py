"""Which buffers of the 8-bit floating-point entry points may share bytes: refusals, before any launch. CPU only: no call here
reaches the GPU (tests/test_gpu_fp8_forms.py holds the calls that are accepted)."""

import re

import pytest

from vybforge_amd import _lib

A = 1 << 40  # (an address of its own for every buffer: A, 2 A, ..)
QUANT = dict(X=A, x_dt=0, ldx=256, Xq=2 * A, Xs=3 * A, M=3, K=256, stream=0)
GEMM = dict(W=A, Ws=2 * A, Xq=3 * A, Xs=4 * A, Y=5 * A, M=40, N=500, K=2048, y_dt=0, ldy=0, RS=6 * A, ws=7 * A, ws_bytes=1 << 26,
            stream=0)
LINEAR = dict(W=A, Ws=2 * A, X=3 * A, x_dt=0, ldx=2048, Y=5 * A, M=40, N=500, K=2048, y_dt=0, ldy=0, RS=6 * A, ws=7 * A,
              ws_bytes=1 << 26, stream=0)
ROUTE = dict(logits=A, logits_dt=0, bias=2 * A, idx=3 * A, w=4 * A, T=3, E=64, topk=4, scale=1.0, softmax=0, renorm=1, groups=8,
             top_groups=2, group_top=2, stream=0)
MOE = dict(x=A, x_dt=0, logits=2 * A, logits_dt=0, bias=3 * A, gate=4 * A, gate_s=5 * A, up=6 * A, up_s=7 * A, down=8 * A,
           down_s=9 * A, sg=10 * A, sgs=11 * A, su=12 * A, sus=13 * A, sd=14 * A, sds=15 * A, out=16 * A, out_dt=0, idx=17 * A,
           w=18 * A, T=3, H=256, I=128, E=64, topk=4, scale=1.0, limit=10.0, softmax=0, renorm=1, groups=8, top_groups=2,
           group_top=2, ws=19 * A, ws_bytes=1 << 30, stream=0)


def refused(name, args, change, text):
    assert getattr(_lib.lib, name)(*(args | change).values()) == _lib.ERR_ARG
    assert re.search(text, _lib.last_error()) and _lib.last_error().startswith(name)


@pytest.mark.parametrize("change", [
    dict(Xs=A), dict(Xs=A + 4 * 768 - 4), dict(Xs=A - 4 * 5), dict(Xs=2 * A), dict(Xs=2 * A + 764), dict(Xs=2 * A - 4 * 5),
    dict(Xq=A + 3 * 256 * 4 - 16), dict(Xq=A - 752), dict(ldx=512, Xs=A + 4 * 512), dict(ldx=512, Xs=A + 4 * 1023),
    dict(ldx=512, Xq=A + 4 * 256 - 16), dict(ldx=512, Xq=A + 4 * 256 + 512), dict(x_dt=1, M=1, Xs=A + 508)])
def test_quantizer(change):
    refused("vybdq_quant_fp8", QUANT, change, "overlap")


PRODUCT = [(dict(Y=A), "W or Ws"), (dict(Y=A + 500 * 2048 - 4), "W or Ws"), (dict(Y=2 * A + 4 * 63), "W or Ws"),
           (dict(Y=2 * A - 4), "W or Ws"), (dict(RS=5 * A + 4), "RS must"), (dict(RS=5 * A - 4), "RS must"),
           (dict(RS=5 * A + 4 * 500), "RS must"), (dict(ldy=1000, RS=5 * A + 4 * 499), "RS must"),
           (dict(ldy=1000, RS=5 * A + 4 * 501), "RS must"), (dict(ldy=1000, RS=5 * A - 4 * 499), "RS must"),
           (dict(ldy=1000, RS=5 * A + 4 * 39000), "RS must"), (dict(Y=7 * A), "workspace"), (dict(W=7 * A + 256), "workspace"),
           (dict(Ws=7 * A), "workspace"), (dict(RS=7 * A + 4), "workspace")]


@pytest.mark.parametrize("change,text", PRODUCT + [
    (dict(Y=3 * A), "overlap X"), (dict(Y=3 * A + 40 * 2048 - 4), "overlap X"), (dict(Y=4 * A), "overlap X"),
    (dict(Y=4 * A + 4 * 40 * 16 - 4), "overlap X"), (dict(Xq=7 * A), "workspace"), (dict(Xs=7 * A), "workspace"),
    (dict(ldy=100000, Xq=5 * A + 4 * 100000 * 39), "overlap X")])
def test_product(change, text):
    refused("vybdq_gemm_fp8", GEMM, change, text)


@pytest.mark.parametrize("change,text", PRODUCT + [
    (dict(Y=3 * A), "overlap X"), (dict(Y=3 * A + 4 * 40 * 2048 - 4), "overlap X"), (dict(X=7 * A), "workspace"),
    (dict(ldx=4096, ldy=4096, Y=3 * A + 4 * 2044), "overlap X"), (dict(ldx=4096, ldy=4096, Y=3 * A + 4 * 4000), "overlap X"),
    (dict(ldx=4096, ldy=4096, Y=3 * A - 4 * 400), "overlap X"), (dict(ldx=4096, ldy=1000, Y=3 * A + 4 * 2048), "overlap X")])
def test_linear(change, text):
    refused("vybdq_linear_fp8", LINEAR, change, text)


@pytest.mark.parametrize("change", [
    dict(idx=A), dict(idx=A + 4 * 3 * 64 - 4), dict(w=A), dict(w=A - 4 * 11), dict(w=3 * A), dict(idx=2 * A), dict(w=2 * A + 4 * 63),
    dict(w=3 * A + 4 * 11), dict(logits_dt=1, idx=A + 2 * 3 * 64 - 4)])
def test_router(change):
    refused("vybdq_moe_route_groups", ROUTE, change, "overlap")


@pytest.mark.parametrize("change", [{b: a} for b in ("idx", "w") for a in (A, 2 * A, 3 * A, 4 * A, 5 * A, 6 * A, 8 * A, 9 * A, 14 * A, 15 * A,
                                                                          16 * A, 19 * A)] +
                         [dict(idx=18 * A), dict(idx=4 * A + 64 * 256 * 128 - 4), dict(w=10 * A + 256 * 128 - 4)] +
                         [{b: 19 * A + 256} for b in ("x", "logits", "bias", "gate", "gate_s", "up", "up_s", "down", "down_s", "sg", "sgs",
                                                      "su", "sus", "sd", "sds", "out")])
def test_layer(change):
    refused("vybdq_moe_forward_fp8", MOE, change, "overlap")
