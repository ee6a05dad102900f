"""8-bit floating-point weights on the GPU at the sizes where offsets outgrow 32 bits, and at the largest that the calls accept."""

import numpy as np
import pytest
import torch

from oracle import fp8
from vybforge_amd import ops

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn


def room(gib):
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < gib << 30:
        pytest.skip(f"needs {gib} GiB of free device memory")


def signs(shape, dev):
    """e4m3 codes of -1, 0 and 1."""
    r = torch.randint(0, 256, shape, dtype=torch.uint8, device=dev)
    return ((r & 1) * 0x38 | (r & 0x80)).view(E4M3)


def any_codes(shape, dev):
    """e4m3 codes of any magnitude below 256, no NaN."""
    return torch.randint(0, 256, shape, dtype=torch.uint8, device=dev).bitwise_and_(0xf7).view(E4M3)


def ones(dev, *shape):
    return torch.ones(shape, device=dev)


def check_product(dev, M, N, K, y, rows=1 << 16):
    """All of X W^T for codes -1, 0, 1 (every partial sum is one float32 holds), `rows` rows of W and of X at a time."""
    X, W = signs((M, K), dev), signs((N, K), dev)
    got = ops.gemm_fp8(W, ones(dev, fp8.blocks(N), fp8.blocks(K)), X, ones(dev, M, fp8.blocks(K)), y_dtype=y)
    for n in range(0, N, rows):
        w = W[n:n + rows].float()
        for m in range(0, M, rows):
            assert torch.equal(got[m:m + rows, n:n + rows], (X[m:m + rows].float() @ w.t()).to(y)), (m, n)


@pytest.mark.parametrize("y", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M", [1, 40, 300])
def test_matrix_of_more_than_4_gib(dev, M, y):
    room(24)
    check_product(dev, M, 540000, 8192, y)


@pytest.mark.parametrize("K", [128, 512, 528])
def test_output_of_more_than_2_to_the_32_elements(dev, K):
    room(40)
    check_product(dev, 70000, 62000, K, torch.bfloat16, rows=20000)


@pytest.mark.parametrize("M,N", [(2 ** 24 - 1, 1), (1, 2 ** 24 - 1), (17, 2 ** 24 - 1)])
def test_most_rows_and_columns(dev, M, N):
    room(24)
    for y in (torch.float32, torch.float16):
        check_product(dev, M, N, 16, y, rows=1 << 24)


@pytest.mark.parametrize("M,N", [(1, 3), (3, 40), (130, 300)])
def test_longest_rows(dev, M, N):
    room(40)
    for y in (torch.float32, torch.bfloat16):
        check_product(dev, M, N, 2 ** 23 - 16, y)


def test_most_rows_of_the_quantizer(dev):
    room(40)
    M, K = 2 ** 28 - 16, 16
    X = torch.empty(M, K, dtype=torch.float16, device=dev)
    for i in range(0, M, 1 << 24):
        X[i:i + (1 << 24)] = torch.randn(X[i:i + (1 << 24)].shape, device=dev)
    q, s = ops.quant_fp8(X)
    for i in (0, M // 2, M - 3000):
        want = fp8.quant(X[i:i + 3000].float().cpu().numpy())
        np.testing.assert_array_equal(q[i:i + 3000].view(torch.uint8).cpu().numpy(), want[0])
        np.testing.assert_array_equal(s[i:i + 3000].cpu().numpy(), want[1])
    for i in range(0, M, 1 << 24):
        a, b = ops.quant_fp8(X[i:i + (1 << 24)])
        assert torch.equal(a.view(torch.uint8), q[i:i + (1 << 24)].view(torch.uint8)) and torch.equal(b, s[i:i + (1 << 24)])


def test_router_of_more_than_2_to_the_31_logits(dev):
    room(24)
    T, E = 2200000, 1024
    logits = torch.empty(T, E, dtype=torch.bfloat16, device=dev).normal_()
    kw = dict(groups=8, top_groups=4, score="softmax", renorm=False)
    idx, w = ops.moe_route(logits, 8, **kw)
    for i in (0, 2 ** 31 // E - 500, T - 1000):
        a, b = ops.moe_route(logits[i:i + 1000].clone(), 8, **kw)
        assert torch.equal(idx[i:i + 1000], a) and torch.equal(w[i:i + 1000], b)
    want = fp8.route(logits[-50:].double().cpu().numpy(), 8, softmax=True, renorm=False, scale=2.5, groups=8, top_groups=4)
    np.testing.assert_array_equal(idx[-50:].cpu().numpy(), want[0])


def layer_of(dev, E, H, I, k, lead=None):
    """A layer whose outputs are near 1; lead: experts before the last that are NaN throughout."""
    pairs = []
    for n, m in ((I, H), (I, H), (H, I)):
        c, s = any_codes((E, n, m), dev), torch.full((E, n // 128, m // 128), 1.0 / (60 * m ** 0.5), device=dev)
        if lead:
            c[:lead].view(torch.uint8).fill_(0x7f)
        pairs.append((c, s))
    return pairs, ops.MoeFp8Layer(*pairs, topk=k)


@pytest.mark.parametrize("T,E,k,H,I", [(2 ** 19 - 1, 16, 8, 128, 128), (65500, 2, 1, 65536, 128), (65500, 2, 1, 65536, 512)])
def test_layer_of_the_most_tokens(dev, T, E, k, H, I):
    """Four million rows, and inputs of nearly 2^32 bytes: any 300 tokens are what they are by themselves."""
    room(100)
    _, layer = layer_of(dev, E, H, I, k)
    x = torch.empty(T, H, dtype=torch.bfloat16, device=dev).normal_()
    logits = torch.randn(T, E, device=dev)
    got = layer(x, logits, out_dtype=torch.bfloat16)
    assert torch.isfinite(got[-300:]).all() and got[-300:].abs().max() > 0
    for i in (0, T // 2, T - 300):
        assert torch.equal(got[i:i + 300], layer(x[i:i + 300], logits[i:i + 300], out_dtype=torch.bfloat16))


@pytest.mark.parametrize("T", [3, 300])
def test_experts_of_4_gib_each(dev, T):
    """The second of two experts, behind one that is NaN throughout, is what it is as the only one."""
    room(60)
    H = I = 65536
    pairs, layer = layer_of(dev, 2, H, I, 1, lead=1)
    x, logits = torch.randn(T, H, device=dev), torch.zeros(T, 2, device=dev)
    logits[:, 1] = 1.0
    alone = ops.MoeFp8Layer(*[(c[1:], s[1:]) for c, s in pairs], topk=1)
    got = layer(x, logits)
    assert torch.isfinite(got).all() and got.abs().max() > 0 and torch.equal(got, alone(x, logits[:, 1:].contiguous()))
