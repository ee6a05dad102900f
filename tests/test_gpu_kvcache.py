"""The paged 8-bit key/value cache on the GPU: kv_append bit for bit against the oracle, KvAttention against float64,
at the sizes, tables and masks where they can go wrong, and both together as a decoding host runs them."""

import numpy as np
import pytest
import torch

from oracle import kvcache, matmul
from vybforge_amd import _lib, ops, synth

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def angles(n_pos, R, seed=0):
    a = np.arange(n_pos)[:, None] * 10000.0 ** (-np.arange(0, R, 2) / R)
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


def tables(rng, lens, page, spare=3):
    """Pages in random order; entries behind a sequence's end are out of the cache's range."""
    used = [-(-c // page) for _, c in lens]
    W, n_pages = max(used + [1]), sum(used) + spare
    order = list(rng.permutation(n_pages))
    table = np.full((len(lens), W), n_pages + 77, np.int32)
    for b, u in enumerate(used):
        table[b, :u] = [order.pop() for _ in range(u)]
    start = np.concatenate([[0], np.cumsum([n for n, _ in lens])]).astype(np.int32)
    return table, start, np.array([c for _, c in lens], np.int32), n_pages


def on(dev, *arrays):
    return [None if a is None else torch.from_numpy(np.ascontiguousarray(a)).to(dev) for a in arrays]


def device_cache(dev, c):
    k, v = (torch.from_numpy(a).to(dev).view(torch.float8_e4m3fn) for a in (c.k, c.v))
    return ops.KvCache(k, v, *on(dev, c.k_scale, c.v_scale))


def random_cache(rng, n_pages, H, page, D, nan=False):
    """Codes of N(0, 1) values, or NaN everywhere; scales of their own for every page and head."""
    fill = lambda shape: (np.full(shape, 0x7f, np.uint8) if nan else kvcache.e4m3_encode(rng.standard_normal(shape) * 80))
    scale = lambda: (2.0 ** rng.integers(-9, -4, (n_pages, H))).astype(np.float32)
    return kvcache.Cache(fill((n_pages, H, page, D)), fill((n_pages, H, page // 4, D, 4)), scale(), scale())


def same_cache(got, want):
    np.testing.assert_array_equal(got.k.view(torch.uint8).cpu().numpy(), want.k)
    np.testing.assert_array_equal(got.v.view(torch.uint8).cpu().numpy(), want.v)
    np.testing.assert_array_equal(got.k_scale.cpu().numpy(), want.k_scale)
    np.testing.assert_array_equal(got.v_scale.cpu().numpy(), want.v_scale)


def oracle_append(want, k, v, q, table, start, ctx, cos, sin, inter):
    """Appends to `want`; the rotated q in float32."""
    q_out = None if q is None else q.copy()
    for b in range(len(ctx)):
        r = slice(start[b], start[b + 1])
        want.append(k[r], v[r], table[b], ctx[b], cos, sin, inter)
        if q is not None:
            for i in range(start[b], start[b + 1]):
                q_out[i] = kvcache.rotate(q[i], ctx[b] - start[b + 1] + i, cos, sin, inter)
    return q_out


def run_append(dev, rng, lens, Hq, Hkv, D, R, page, inter, x, scale=1.0, max_new=None, fused=True):
    table, start, ctx, n_pages = tables(rng, lens, page)
    want = random_cache(rng, n_pages, Hkv, page, D)
    cache = device_cache(dev, want)
    T = int(start[-1])
    qkv = torch.from_numpy((rng.standard_normal((T, (Hq + 2 * Hkv) * D)) * scale).astype(np.float32)).to(DT[x]).to(dev)
    parts = [t.unflatten(1, (-1, D)) for t in qkv.split([Hq * D, Hkv * D, Hkv * D], 1)]
    if not fused:
        parts = [t.contiguous() for t in parts]
    q, k, v = parts
    cos, sin = angles(max(int(ctx.max()), 1), R) if R else (None, None)
    got = ops.kv_append(cache, k, v, *on(dev, table, start, ctx), q=q, interleaved=inter, max_new=max_new,
                        **dict(zip(("cos", "sin"), on(dev, cos, sin))))
    f = lambda t: t.float().cpu().numpy()
    q_want = oracle_append(want, f(k), f(v), f(q), table, start, ctx, cos, sin, inter)
    same_cache(cache, want)
    assert torch.equal(got.cpu(), torch.from_numpy(q_want).to(DT[x]))
    ops.kv_status()


# ---- append -----------------------------------------------------------------------------------

@pytest.mark.parametrize("x", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D,R,page,inter", [(64, 64, 16, False), (128, 128, 64, False), (128, 32, 256, True),
                                            (192, 96, 32, False), (256, 64, 16, True), (128, 0, 128, False)])
def test_append_matches_oracle(dev, rng, x, D, R, page, inter):
    # from an empty cache, inside a page, from a page's first slot to its last, over several pages, and no rows at all
    lens = [(1, 1), (5, 23), (page, 2 * page), (0, 40), (2 * page + 3, 3 * page + 1), (1, page), (1, page + 1), (0, 0)]
    run_append(dev, rng, lens, 6, 2, D, R, page, inter, x)


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (5, 5), (8, 1), (21, 3)])
def test_append_head_layouts(dev, rng, Hq, Hkv):
    run_append(dev, rng, [(1, 70), (3, 3), (17, 90)], Hq, Hkv, 64, 32, 32, False, "bf16", fused=False)


@pytest.mark.parametrize("max_new", [None, 1, 7, 1000])
def test_append_any_bound_is_right(dev, rng, max_new):
    run_append(dev, rng, [(9, 50), (1, 33), (40, 40), (0, 5)], 4, 2, 64, 64, 16, False, "f16", max_new=max_new)


@pytest.mark.parametrize("scale", [1e-30, 2.0 ** -60, 1e-4, 3e4, 1e20, 1e30])
def test_append_magnitudes(dev, rng, scale):
    run_append(dev, rng, [(1, 5), (30, 61)], 2, 1, 64, 0, 32, False, "f32", scale=scale)


def test_append_many_sequences(dev, rng):
    lens = [(int(n), int(n + c)) for n, c in zip(rng.integers(0, 4, 200), rng.integers(0, 40, 200))]
    run_append(dev, rng, lens, 2, 1, 64, 32, 16, False, "bf16")
    run_append(dev, rng, [(1, 1 + int(c)) for c in rng.integers(0, 40, 300)], 2, 1, 64, 32, 16, False, "bf16", max_new=1)


def test_append_token_by_token_grows_goes_back_and_starts_again(dev, rng):
    """A page filled one token at a time with growing values, stepped back into, and used anew from its first slot."""
    P, D = 16, 64
    table, _, _, n_pages = tables(rng, [(0, 2 * P)], P)
    want = random_cache(rng, n_pages, 1, P, D)
    cache = device_cache(dev, want)
    steps = [(1, t + 1, 1.5 ** t) for t in range(20)] + [(2, 9, 1e-3), (3, 14, 1e3), (1, 1, 1e-2), (31, 32, 1.0)]
    for n, c, size in steps:
        k, v = ((rng.standard_normal((n, 1, D)) * size).astype(np.float32) for _ in range(2))
        start, ctx = np.array([0, n], np.int32), np.array([c], np.int32)
        ops.kv_append(cache, *on(dev, k, v, table, start, ctx))
        want.append(k, v, table[0], c)
        same_cache(cache, want)
    ops.kv_status()


def test_append_tokens_with_infinities_and_nan(dev, rng):
    """Such a token is stored as K NaN, V zero, and its finite values still count for the page's scale; heads apart."""
    table, start, ctx, n_pages = tables(rng, [(20, 21)], 16)
    want = random_cache(rng, n_pages, 2, 16, 64)
    cache = device_cache(dev, want)
    k, v = (rng.standard_normal((20, 2, 64)).astype(np.float32) for _ in range(2))
    k[3, 0, 5], k[17, 1, 0], v[9, 1, 63], v[0, 0, 0] = np.nan, np.inf, -np.inf, np.nan
    ops.kv_append(cache, *on(dev, k, v, table, start, ctx))
    oracle_append(want, k, v, None, table, start, ctx, None, None, False)
    same_cache(cache, want)
    assert (want.k == 0x7f).reshape(n_pages, 2, 16, 64).all(-1).sum() == 4


def test_append_bad_tables_are_reported_and_nothing_else_is_written(dev, rng):
    D, page = 64, 16
    good = [(2, 20), (3, 30), (1, 9)]
    table, start, ctx, n_pages = tables(rng, good, page)
    before = random_cache(rng, n_pages, 1, page, D)
    k, v, q = ((rng.standard_normal((6, h, D))).astype(np.float32) for h in (1, 1, 2))
    cos, sin = angles(31, 64)

    def case(text, table, start, ctx, skipped, cos=cos, sin=sin, max_new=None):
        want = kvcache.Cache(*(a.copy() for a in (before.k, before.v, before.k_scale, before.v_scale)))
        cache = device_cache(dev, want)
        ops.kv_append(cache, *on(dev, k, v, table, start, ctx), q=on(dev, q)[0], max_new=max_new,
                      **dict(zip(("cos", "sin"), on(dev, cos, sin))))
        for b in range(3):
            if b not in skipped:
                want.append(k[start[b]:start[b + 1]], v[start[b]:start[b + 1]], table[b], ctx[b], cos, sin)
        with pytest.raises(_lib.VybdqError, match=text):
            ops.kv_status()
        ops.kv_status()  # cleared
        same_cache(cache, want)

    for max_new in (None, 1):
        t = table.copy()
        t[1, 1] = -1
        case("page of the table", t, start, ctx, {1}, max_new=max_new)
        t[1, 1] = n_pages
        case("page of the table", t, start, ctx, {1}, max_new=max_new)
        for c in (1, -5, -2 ** 31, 33, 2 ** 31 - 1):
            x = ctx.copy()
            x[0] = c
            case("ctx", table, start, x, {0}, max_new=max_new)
        for s in (7, -1, 2 ** 31 - 1):
            x = start.copy()
            x[3] = s
            case("q_start", table, x, ctx, {2}, max_new=max_new)
        case("cos and sin", table, start, ctx, {1}, *angles(29, 64), max_new=max_new)


# ---- attention ----------------------------------------------------------------------------------

def tolerance(out, lse, weight, reach, D, L, x):
    """Bounds on |out - exact| and |lse - exact|, term by term: a score's float32 sum of D products and its exponent
    (2^-24 each, relative to the products' magnitudes and to |t| < 64 + 1.5 reach), for float32 queries their rounding to
    two fp16 terms (2^-22); a weight's rounding to fp16 (2^-11, two terms 2^-21) and exp2 (2^-22); L float32 additions
    of weighted values and of weights (2^-23 each, not rounded to nearest); the output's own rounding."""
    two = x == "f32"
    ds = reach * ((D + 8) * 2.0 ** -24 + (2.0 ** -22 if two else 0)) + (64 + 1.5 * reach) * 2.0 ** -24 + 2.0 ** -22
    rel = (2.0 ** -21 if two else 2.0 ** -11) + 2 * ds + (2 * L + 128) * 2.0 ** -23
    half = torch.finfo(DT[x]).eps / 2
    return half * np.abs(out) + rel[..., None] * weight * (1 + half), ds + (L + 64) * 2.0 ** -23 + 2.0 ** -22 * (1 + np.abs(lse))


def check_attention(got, stats, q, want, table, start, ctx, scale, causal, window, x):
    T, Hq, D = q.shape
    G = Hq // want.k.shape[1]
    got, stats = got.double().cpu().numpy(), None if stats is None else stats.double().cpu().numpy()
    for b in range(len(ctx)):
        r = slice(start[b], start[b + 1])
        for hq in range(Hq):
            k, v = want.values(table[b], max(ctx[b], 0), hq // G)
            o, z, weight, reach = kvcache.attention(q[r, hq], k, v, ctx[b] - (start[b + 1] - start[b]), max(ctx[b], 0), scale,
                                                    causal, window)
            to, tz = tolerance(o, np.where(np.isfinite(z), z, 0), weight, reach, D, ctx[b], x)
            err = np.abs(got[r, hq] - o)
            assert (err <= to)[~np.isnan(o)].all(), (b, hq, np.nanmax(err - to))
            np.testing.assert_array_equal(np.isnan(got[r, hq]), np.isnan(o))
            if stats is not None:
                np.testing.assert_array_equal(np.isneginf(stats[r, hq]), np.isneginf(z))
                ok = np.isfinite(z)
                assert (np.abs(stats[r, hq][ok] - z[ok]) <= tz[ok]).all(), (b, hq)


def run_attention(dev, rng, lens, Hq, Hkv, D, page, x, causal=True, window=0, scale=None, lse=True, max_new=None,
                  max_ctx=None, q_scale=1.0, attend=None):
    table, start, ctx, n_pages = tables(rng, lens, page)
    want = random_cache(rng, n_pages, Hkv, page, D)
    # what no token of a sequence wrote may hold anything: here NaN codes, and NaN scales where a page is unused
    written = {int(p) for b, (_, c) in enumerate(lens) for p in table[b, :-(-c // page)]}
    for p in set(range(n_pages)) - written:
        want.k[p], want.v[p], want.k_scale[p], want.v_scale[p] = 0x7f, 0x7f, np.nan, np.nan
    for b, (_, c) in enumerate(lens):
        if c % page:
            p, s = int(table[b, c // page]), c % page
            want.k[p, :, s:] = 0x7f
            flat = want.v[p].transpose(0, 1, 3, 2).reshape(Hkv, page, D)
            flat[:, s:] = 0x7f
            want.v[p] = flat.reshape(Hkv, page // 4, 4, D).transpose(0, 1, 3, 2)
    q = torch.from_numpy((rng.standard_normal((int(start[-1]), Hq, D)) * q_scale).astype(np.float32)).to(DT[x])
    attend = attend or ops.KvAttention(Hq, Hkv, D, dev)
    got = attend(q.to(dev), device_cache(dev, want), *on(dev, table, start, ctx), causal=causal, window=window, scale=scale,
                 lse=lse, max_new=max_new, max_ctx=max_ctx)
    got, stats = got if lse else (got, None)
    check_attention(got, stats, q.double().numpy(), want, table, start, ctx, D ** -0.5 if scale is None else scale, causal,
                    window, x)
    ops.kv_status()


DECODE = [(1, 1), (1, 15), (1, 16), (1, 17), (1, 32), (1, 33), (0, 9), (1, 129), (1, 700)]
MIXED = [(3, 3), (1, 200), (0, 0), (40, 41), (70, 333), (2, 17)]


@pytest.mark.parametrize("x", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D", [64, 128, 192, 256])
@pytest.mark.parametrize("lens", [DECODE, MIXED], ids=["decode", "mixed"])
def test_attention_types_and_dims(dev, rng, x, D, lens):
    run_attention(dev, rng, lens, 4, 2, D, 32, x)


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (3, 3), (12, 2), (16, 1), (17, 1), (40, 1), (21, 3)])
@pytest.mark.parametrize("n", [1, 3, 37])
def test_attention_head_layouts(dev, rng, Hq, Hkv, n):
    run_attention(dev, rng, [(n, 100), (n, n), (n, 61)], Hq, Hkv, 64, 16, "bf16", max_new=n)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("n", [1, 50])
def test_attention_pages(dev, rng, page, n):
    run_attention(dev, rng, [(n, n + c) for c in (0, page - 1, page, page + 1, 3 * page + 7)], 4, 1, 64, page, "f16")


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("window", [0, 1, 5, 31, 32, 33, 100, 2 ** 30 - 1])
@pytest.mark.parametrize("n", [1, 4, 45])
def test_attention_masks(dev, rng, causal, window, n):
    run_attention(dev, rng, [(n, 150), (n, n), (n, n + 31)], 4, 2, 64, 16, "f16", causal=causal, window=window)


@pytest.mark.parametrize("x", ["bf16", "f32"])
@pytest.mark.parametrize("window,causal", [(0, True), (3, True), (3, False)])
def test_attention_rows_that_see_nothing(dev, rng, x, window, causal):
    """More rows than tokens: the first rows' positions are negative. They are zero, with lse -inf."""
    run_attention(dev, rng, [(9, 4), (1, 0), (3, 0), (50, 7)], 2, 1, 64, 16, x, window=window, causal=causal)


@pytest.mark.parametrize("max_new,max_ctx", [(None, None), (1, 1), (1, 40), (3, 5000), (300, 100), (0, 0)])
def test_attention_any_bounds_are_right(dev, rng, max_new, max_ctx):
    run_attention(dev, rng, MIXED + [(1, 600)], 6, 2, 64, 16, "bf16", max_new=max_new, max_ctx=max_ctx)


@pytest.mark.parametrize("x", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("n", [1, 6, 90])
def test_attention_split_keys(dev, rng, x, n):
    """One sequence of a few thousand tokens: the keys are split over workgroups and joined."""
    run_attention(dev, rng, [(n, 3001)], 4, 1, 64, 64, x, max_new=n)


@pytest.mark.parametrize("variant", [0, 1, 2, 3])
@pytest.mark.parametrize("splits", [1, 2, 7, -2, -7])
@pytest.mark.parametrize("x,D", [("bf16", 128), ("f32", 256), ("f16", 64), ("f32", 128), ("bf16", 192)])
def test_attention_every_variant(dev, rng, monkeypatch, variant, splits, x, D):
    """Kernel variants and key splits other than the chosen ones, on odd lengths, with and without a window; more keys than
    a batch of 64 steps."""
    monkeypatch.setenv("VYBDQ_KV_VARIANT", str(variant))
    monkeypatch.setenv("VYBDQ_KV_SPLITS", str(splits))
    lens = [(1, 2300), (70, 333), (0, 50), (33, 33), (5, 90)]
    run_attention(dev, rng, lens, 3, 1, D, 16, x)
    run_attention(dev, rng, lens, 4, 2, D, 64, x, window=77, causal=False)


@pytest.mark.parametrize("q_scale", [1e-30, 1e-4, 30.0])
@pytest.mark.parametrize("x", ["bf16", "f32"])
def test_attention_query_magnitudes(dev, rng, x, q_scale):
    run_attention(dev, rng, [(1, 90), (20, 64)], 2, 1, 64, 16, x, q_scale=q_scale)


@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0])
def test_attention_scales(dev, rng, scale):
    run_attention(dev, rng, [(1, 90), (40, 64)], 2, 1, 64, 16, "f32", scale=scale)


def test_attention_page_scales_far_apart(dev, rng):
    """Pages whose value scales differ by 2^70, the ones with small values with nearly all the weight."""
    D, page = 64, 16
    table, start, ctx, n_pages = tables(rng, [(1, 48)], page)
    want = random_cache(rng, n_pages, 1, page, D)
    want.v_scale[table[0, :3], 0] = [2.0 ** -30, 2.0 ** 10, 2.0 ** -60]
    want.k_scale[table[0, :3], 0] = [2.0 ** -6, 2.0 ** -20, 2.0 ** -6]
    q = np.zeros((1, 1, D), np.float32)
    q[0, 0] = kvcache.e4m3_decode(want.k[table[0, 0], 0, 3]) / 40  # the first page's fourth key has nearly all the weight
    for x in ("f16", "f32"):
        qt = torch.from_numpy(q).to(DT[x])
        got, stats = ops.KvAttention(1, 1, D, dev)(qt.to(dev), device_cache(dev, want), *on(dev, table, start, ctx), lse=True)
        check_attention(got, stats, qt.double().numpy(), want, table, start, ctx, D ** -0.5, True, 0, x)


def test_attention_nan_reaches_only_rows_that_see_it(dev, rng):
    """A token stored from a NaN, a NaN query row and an infinite one."""
    D, page, Hkv = 64, 16, 1
    table, start, ctx, n_pages = tables(rng, [(40, 50), (2, 30)], page)
    want = random_cache(rng, n_pages, Hkv, page, D)
    cache = device_cache(dev, want)
    k, v = (rng.standard_normal((42, Hkv, D)).astype(np.float32) for _ in range(2))
    v[20, 0, 7] = np.nan  # position 30 of the first sequence
    t = on(dev, table, start, ctx)
    ops.kv_append(cache, *on(dev, k, v), *t)
    oracle_append(want, k, v, None, table, start, ctx, None, None, False)
    q = torch.from_numpy(rng.standard_normal((42, 2, D)).astype(np.float32)).to(torch.bfloat16)
    q[5, 0, 3], q[41, 1, 60] = float("nan"), float("inf")
    for window in (0, 12):
        got = ops.KvAttention(2, Hkv, D, dev)(q.to(dev), cache, *t, window=window)
        nan = torch.isnan(got.float()).all(-1).cpu().numpy()
        some = torch.isnan(got.float()).any(-1).cpu().numpy()
        seen = np.zeros((42, 2), bool)
        seen[20:(40 if not window else 32)] = True
        seen[5, 0] = seen[41, 1] = True
        np.testing.assert_array_equal(nan, seen)
        np.testing.assert_array_equal(some, seen)


def test_attention_bad_tables(dev, rng):
    """Rows that see a page outside the cache, or tokens past the table, are NaN, the others right; and it is reported."""
    D, page = 64, 16
    lens = [(30, 60), (1, 20), (2, 40)]
    table, start, ctx, n_pages = tables(rng, lens, page)
    want = random_cache(rng, n_pages, 1, page, D)
    cache = device_cache(dev, want)
    q = torch.from_numpy(rng.standard_normal((33, 2, D)).astype(np.float32)).to(torch.float16)
    attend = ops.KvAttention(2, 1, D, dev)
    good = attend(q.to(dev), cache, *on(dev, table, start, ctx)).clone()

    def case(text, table, start, ctx, nan_rows, skipped=()):
        for max_new in (None, 1):
            out = torch.full((33, 2, D), 7.0, dtype=torch.float16, device=dev)
            attend(q.to(dev), cache, *on(dev, table, start, ctx), out=out, max_new=max_new, max_ctx=64)
            with pytest.raises(_lib.VybdqError, match=text):
                ops.kv_status()
            for r in range(33):
                if r in skipped:
                    assert (out[r] == 7.0).all(), r
                elif r in nan_rows:
                    assert torch.isnan(out[r]).all(), r
                else:
                    assert (out[r] - good[r]).abs().max() < 2e-3 and not torch.isnan(out[r]).any(), r

    for bad in (-1, n_pages, 2 ** 31 - 1, -2 ** 31):
        t = table.copy()
        t[0, 2] = bad  # tokens 32 .. 47: the rows at positions 32 and up see them
        case("page of the table", t, start, ctx, set(range(2, 30)))
    c = ctx.copy()
    c[1] = 2 ** 31 - 1
    case("ctx", table, start, c, {30})
    s = start.copy()
    s[3] = 40
    case("q_start", table, s, ctx, (), skipped={31, 32})


def test_attention_of_nothing(dev):
    cache = ops.KvCache.empty(1, 1, 64, device=dev)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)
    q = torch.empty(0, 2, 64, device=dev)
    table, kv = i32(0).view(1, 1), torch.empty(0, 1, 64, device=dev)
    assert ops.KvAttention(2, 1, 64, dev)(q, cache, table, i32(0, 0), i32(0)).shape == (0, 2, 64)
    assert ops.kv_append(cache, kv, kv, table, i32(0, 0), i32(0), q=q).shape == (0, 2, 64)
    none = torch.empty(0, 1, dtype=torch.int32, device=dev)
    assert ops.kv_append(cache, kv, kv, none, i32(0), i32()) is None
    ops.kv_status()


def test_attention_strided_queries_and_given_output(dev, rng):
    """q as a slice of a projection's output, out given: rows behind the last one stay as they were."""
    D, page = 128, 64
    table, start, ctx, n_pages = tables(rng, [(1, 100), (1, 7)], page)
    want = random_cache(rng, n_pages, 2, page, D)
    cache = device_cache(dev, want)
    qkv = torch.randn(2, 8 * D, device=dev).to(torch.bfloat16)
    q = qkv[:, :4 * D].unflatten(1, (4, D))
    attend = ops.KvAttention(4, 2, D, dev)
    room = torch.full((3, 4, D), 5.0, dtype=torch.bfloat16, device=dev)
    t = on(dev, table, start, ctx)
    got = attend(q, cache, *t, out=room[:2])
    assert torch.equal(got, attend(q.contiguous(), cache, *t)) and (room[2] == 5.0).all()
    check_attention(got, None, q.double().cpu().numpy(), want, table, start, ctx, D ** -0.5, True, 0, "bf16")


def test_attention_is_reproducible(dev, rng):
    table, start, ctx, n_pages = tables(rng, [(1, 5000), (1, 3000)], 64)
    cache = device_cache(dev, random_cache(rng, n_pages, 2, 64, 64))
    q = torch.randn(2, 8, 64, device=dev)
    attend, t = ops.KvAttention(8, 2, 64, dev), on(dev, table, start, ctx)
    first = attend(q, cache, *t, max_new=1, max_ctx=5000).clone()
    for _ in range(20):
        assert torch.equal(attend(q, cache, *t, max_new=1, max_ctx=5000), first)


def test_offsets_past_32_bits(dev, rng):
    """A cache of more than 4 GiB of codes: its last pages are written and read at their own places."""
    Hkv, page, D = 8, 256, 256
    n_pages = (1 << 32) // (Hkv * page * D) + 5
    cache = ops.KvCache.empty(n_pages, Hkv, D, page, dev)
    lens = [(300, 300)]
    table = np.array([[n_pages - 1, n_pages - 3]], np.int32)
    start, ctx = np.array([0, 300], np.int32), np.array([300], np.int32)
    k, v = (rng.standard_normal((300, Hkv, D)).astype(np.float32) for _ in range(2))
    t = on(dev, table, start, ctx)
    ops.kv_append(cache, *on(dev, k, v), *t)
    small = kvcache.Cache(np.zeros((2, Hkv, page, D), np.uint8), np.zeros((2, Hkv, page // 4, D, 4), np.uint8),
                          np.ones((2, Hkv), np.float32), np.ones((2, Hkv), np.float32))
    oracle_append(small, k, v, None, np.array([[0, 1]]), start, ctx, None, None, False)
    last = [n_pages - 1, n_pages - 3]
    np.testing.assert_array_equal(cache.k[last[0]].view(torch.uint8).cpu().numpy(), small.k[0])
    np.testing.assert_array_equal(cache.v[last[0]].view(torch.uint8).cpu().numpy(), small.v[0])
    q = torch.from_numpy(rng.standard_normal((1, Hkv, D)).astype(np.float32))
    one = on(dev, np.array([0, 1], np.int32))[0]
    got = ops.KvAttention(Hkv, Hkv, D, dev)(q.to(dev), cache, t[0], one, t[2])
    check_attention(got, None, q.double().numpy(), small, np.array([[0, 1]]), np.array([0, 1]), ctx, D ** -0.5, True, 0, "f32")
    ops.kv_status()


@pytest.mark.parametrize("splits", [-2, -3, -40])
@pytest.mark.parametrize("B", [2, 64, 65, 200])
def test_attention_splits_by_length(dev, rng, monkeypatch, B, splits):
    """Splits that go with the sequences' lengths: one long and many short, all empty but one, all alike, no rows at all."""
    monkeypatch.setenv("VYBDQ_KV_VARIANT", "0")
    monkeypatch.setenv("VYBDQ_KV_SPLITS", str(splits))
    attend = ops.KvAttention(2, 1, 64, dev)
    for lens in ([(1, int(c)) for c in rng.integers(1, 400, B - 1)] + [(2, 3000)],
                 [(0, 0)] * (B - 2) + [(1, 2000), (0, 50)],
                 [(1, 130)] * B,
                 [(0, 0)] * B):
        for _ in range(2):
            run_attention(dev, rng, lens, 2, 1, 64, 16, "f16", window=0 if B < 65 else 1000, attend=attend)
    run_attention(dev, rng, [(1, 0), (1, 1)] * (B // 2), 2, 1, 64, 16, "f16", attend=attend)


def test_attention_splits_by_length_with_bad_tables(dev, rng, monkeypatch):
    """A sequence whose rows, length or pages are wrong among good ones; a good call of the same workspace afterwards."""
    monkeypatch.setenv("VYBDQ_KV_SPLITS", "-5")
    D, page = 64, 16
    lens = [(1, 600), (1, 20), (1, 300)]
    table, start, ctx, n_pages = tables(rng, lens, page)
    cache = device_cache(dev, random_cache(rng, n_pages, 1, page, D))
    attend, q = ops.KvAttention(2, 1, D, dev), torch.randn(3, 2, D, device=dev)
    good = attend(q, cache, *on(dev, table, start, ctx))
    for change in ((0, 2 ** 31 - 1), (0, -2 ** 31), (2, 2 ** 30), (1, -1)):
        c = ctx.copy()
        c[change[0]] = change[1]
        out = attend(q, cache, *on(dev, table, start, c))
        torch.cuda.synchronize()
        for b in range(3):
            assert b == change[0] or (out[b] - good[b]).abs().max() < 1e-5, (change, b)
        if change[1] > 0:
            with pytest.raises(_lib.VybdqError, match="ctx"):
                ops.kv_status()
        assert torch.equal(attend(q, cache, *on(dev, table, start, ctx)), good)
    s = start.copy()
    s[2] = 40
    attend(q, cache, *on(dev, table, s, ctx))
    with pytest.raises(_lib.VybdqError, match="q_start"):
        ops.kv_status()
    assert torch.equal(attend(q, cache, *on(dev, table, start, ctx)), good)
    ops.kv_status()


@pytest.mark.parametrize("n,splits", [(1, None), (1, 256), (33, 256)])
def test_attention_over_half_a_billion_keys(dev, rng, monkeypatch, n, splits):
    """2^29 + 100 keys in 256 splits (steps times splits pass 32 bits), held in five pages that the table repeats, a quarter
    of the context each and one at its end; their values have different means. A lane adds 2^29 / 32 / 256 steps of 8 weights,
    each to half a unit in the last place of their sum: 2^19 2^-24 = 2^-5 of it; an output sums as many steps, at most four
    roundings of 2^-23 to a step: 2^18 2^-23 = 2^-5 again. 2^-4 covers both."""
    if splits:
        monkeypatch.setenv("VYBDQ_KV_SPLITS", str(splits))
    D, page = 64, 256
    ctx = 2 ** 29 + 100
    W = -(-ctx // page)
    want = random_cache(rng, 5, 1, page, D)
    want.k_scale[:] = 2.0 ** -9
    want.v[:] = kvcache.e4m3_encode(rng.standard_normal(want.v.shape) * 40 + np.array([-200, -100, 100, 200, 0])[:, None, None, None, None])
    want.v_scale[:] = 2.0 ** -7
    table = (np.arange(W, dtype=np.int64) * 4 // W).astype(np.int32)
    table[-1] = 4
    cache = device_cache(dev, want)
    q = torch.from_numpy(rng.standard_normal((n, 1, D)).astype(np.float32))
    got, stats = ops.KvAttention(1, 1, D, dev)(q.to(dev), cache, *on(dev, table[None], np.array([0, n], np.int32), np.array([ctx], np.int32)),
                                               causal=False, lse=True, max_new=n, max_ctx=ctx)
    times = np.bincount(table[:-1], minlength=5).astype(np.float64)[:, None] * np.ones(page)
    times[4, :100] += 1
    k, v = (kvcache.e4m3_decode(x).astype(np.float64) for x in (want.k[:, 0], want.v[:, 0]))
    v = v.transpose(0, 1, 3, 2).reshape(5, page, D) * want.v_scale[:, 0, None, None]
    s = np.einsum("nd,pkd->npk", q[:, 0].double().numpy(), k) * want.k_scale[:, 0, None] * D ** -0.5
    w = np.exp(s - s.max()) * times
    l = w.sum((1, 2))
    o = np.einsum("npk,pkd->nd", w, v) / l[:, None]
    assert np.abs(stats[:, 0].double().cpu().numpy() - np.log(l) - s.max()).max() < 2.0 ** -4
    assert np.abs(got[:, 0].double().cpu().numpy() - o).max() < 2.0 ** -4 * np.abs(v).max()
    ops.kv_status()


# ---- streams, graphs, and the operators together --------------------------------------------------

def test_other_stream(dev, rng):
    table, start, ctx, n_pages = tables(rng, [(1, 2000)], 64)
    want = random_cache(rng, n_pages, 1, 64, 64)
    cache, t = device_cache(dev, want), on(dev, table, start, ctx)
    q = torch.randn(1, 4, 64, device=dev)
    attend = ops.KvAttention(4, 1, 64, dev)
    here = attend(q, cache, *t).clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = attend(q, cache, *t)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(here, there)


def test_workspace_made_behind_other_work_is_ready_on_another_stream(dev, rng):
    table, start, ctx, n_pages = tables(rng, [(1, 4000)], 64)
    cache, t = device_cache(dev, random_cache(rng, n_pages, 1, 64, 64)), on(dev, table, start, ctx)
    q = torch.randn(1, 4, 64, device=dev)
    want = ops.KvAttention(4, 1, 64, dev)(q, cache, *t).clone()
    side, a = torch.cuda.Stream(), torch.randn(4096, 4096, device=dev)
    torch.cuda.synchronize()
    for _ in range(20):
        a = a @ a * 1e-3
    attend = ops.KvAttention(4, 1, 64, dev)
    with torch.cuda.stream(side):
        got = attend(q, cache, *t)
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_graphs_of_a_decode_loop(dev, rng):
    """Append and attention captured for two batch sizes over one cache and one workspace; the tables move on between
    replays, eager calls run between them, and every replay equals the eager result."""
    D, page, Hq, Hkv, W = 64, 16, 4, 2, 40
    attend = ops.KvAttention(Hq, Hkv, D, dev)
    cos, sin = on(dev, *angles(W * page, D))

    class Loop:
        def __init__(self, B, first_page):
            self.B, self.ctx = B, torch.full((B,), 500, dtype=torch.int32, device=dev)
            self.table = (first_page + torch.arange(B * W, device=dev, dtype=torch.int32)).view(B, W).contiguous()
            self.start = torch.arange(B + 1, dtype=torch.int32, device=dev)
            self.q, self.k, self.v = (torch.zeros(B, h, D, device=dev, dtype=torch.bfloat16) for h in (Hq, Hkv, Hkv))

        def step(self, cache):
            q = ops.kv_append(cache, self.k, self.v, self.table, self.start, self.ctx, q=self.q, cos=cos, sin=sin, max_new=1)
            return attend(q, cache, self.table, self.start, self.ctx, max_new=1, max_ctx=W * page)

    both = [Loop(1, 0), Loop(5, W)]
    want = random_cache(rng, 6 * W, Hkv, page, D)
    live, shadow = device_cache(dev, want), device_cache(dev, want)
    graphs = []
    for loop in both:
        loop.step(live)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = loop.step(live)
        graphs.append((g, out))
    live = [t.copy_(s) for t, s in ((live.k.view(torch.uint8), shadow.k.view(torch.uint8)), (live.v.view(torch.uint8), shadow.v.view(torch.uint8)),
                                    (live.k_scale, shadow.k_scale), (live.v_scale, shadow.v_scale))]
    for i in range(12):
        for loop, (g, out) in zip(both, graphs):
            for x in (loop.q, loop.k, loop.v):
                x.copy_(torch.randn(x.shape, device=dev) * 1.3 ** i)
            loop.ctx += 1
            g.replay()
            eager = loop.step(shadow)
            torch.cuda.synchronize()
            assert torch.equal(out, eager), i
            assert torch.equal(live[0], shadow.k.view(torch.uint8)) and torch.equal(live[2], shadow.k_scale), i
            assert torch.equal(live[1], shadow.v.view(torch.uint8)) and torch.equal(live[3], shadow.v_scale), i
    ops.kv_status()


@pytest.mark.parametrize("Hq,n", [(2, 90), (4, 12)])
def test_graph_of_a_chunk(dev, rng, Hq, n):
    """A chunk's attention with its keys split (a launch for the join at 90 rows a head), captured and replayed at other
    lengths, with eager calls of the same workspace between the replays."""
    table, start, ctx, n_pages = tables(rng, [(n, 3000), (1, 900)], 64)
    cache = device_cache(dev, random_cache(rng, n_pages, 1, 64, 64))
    attend, t = ops.KvAttention(Hq, 1, 64, dev), on(dev, table, start, ctx)
    q = torch.zeros(n + 1, Hq, 64, device=dev, dtype=torch.float16)
    args = dict(max_new=n, max_ctx=3000, lse=True)
    attend(q, cache, *t, **args)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, lse = attend(q, cache, *t, **args)
    for i in range(6):
        q.copy_(torch.randn(q.shape, device=dev))
        t[2].copy_(torch.tensor([3000 - 411 * i, 900 - 170 * i], dtype=torch.int32))
        g.replay()
        eager, eager_lse = attend(q, cache, *t, **args)
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and torch.equal(lse, eager_lse), i
    ops.kv_status()


def test_two_streams_at_once(dev, rng):
    """Two batches in one cache on two streams, each with a workspace of its own; their contexts share pages."""
    D, page = 128, 64
    table, _, _, n_pages = tables(rng, [(0, 4000), (0, 4000)], page)
    table[1, :40] = table[0, :40]
    cache = device_cache(dev, random_cache(rng, n_pages, 2, page, D))
    start, ctx = on(dev, np.array([0, 3], np.int32), np.array([3999], np.int32))
    batches = [on(dev, table[b:b + 1])[0] for b in range(2)]
    attends = [ops.KvAttention(4, 2, D, dev) for _ in range(2)]
    q = [torch.randn(3, 4, D, device=dev) for _ in range(2)]
    k, v = (torch.randn(3, 2, D, device=dev) for _ in range(2))
    step = lambda b: (ops.kv_append(cache, k, v, batches[b], start, ctx), attends[b](q[b], cache, batches[b], start, ctx))[1]
    alone = [step(b).clone() for b in range(2)]
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for b in range(2):
            with torch.cuda.stream(sides[b]):
                got.append(step(b))
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(alone, got))
    ops.kv_status()


@pytest.mark.parametrize("x", ["bf16", "f32"])
def test_rows_behind_the_last_sequence_stay(dev, rng, x):
    """A padded batch: rows past q_start[B], and sequences without rows, leave outputs and cache as they were."""
    D, page = 64, 16
    lens = [(3, 20), (0, 0), (40, 40), (0, 7)]
    table, start, ctx, n_pages = tables(rng, lens, page)
    want = random_cache(rng, n_pages, 1, page, D)
    cache, t = device_cache(dev, want), on(dev, table, start, ctx)
    T = 50
    q, k, v = (torch.randn(T, h, D, device=dev).to(DT[x]) for h in (2, 1, 1))
    q_out, out = (torch.full((T, 2, D), 7.0, device=dev, dtype=DT[x]) for _ in range(2))
    attend = ops.KvAttention(2, 1, D, dev)
    for max_new in (None, 1, 40):
        ops.kv_append(cache, k, v, *t, q=q, q_out=q_out, max_new=max_new)
        attend(q, cache, *t, out=out, max_new=max_new)
        assert (q_out[43:] == 7.0).all() and (out[43:] == 7.0).all()
        assert torch.equal(q_out[:43], q[:43])
    f = lambda a: a.float().cpu().numpy()
    for _ in range(3):
        oracle_append(want, f(k), f(v), None, table, start, ctx, None, None, False)
    same_cache(cache, want)
    check_attention(out[:43], None, q[:43].double().cpu().numpy(), want, table, start, ctx, D ** -0.5, True, 0, x)
    ops.kv_status()


@pytest.mark.parametrize("n,Hq", [(1, 4), (5, 6), (100, 2)])
def test_outputs_in_place(dev, rng, n, Hq):
    """q_out and out may be q."""
    D, page = 64, 64
    table, start, ctx, n_pages = tables(rng, [(n, 2000), (n, 300)], page)
    cache, t = device_cache(dev, random_cache(rng, n_pages, 2, page, D)), on(dev, table, start, ctx)
    cos, sin = on(dev, *angles(2000, D))
    q, k, v = (torch.randn(2 * n, h, D, device=dev).bfloat16() for h in (Hq, 2, 2))
    attend, args = ops.KvAttention(Hq, 2, D, dev), dict(max_new=n, max_ctx=2000)
    turned = ops.kv_append(cache, k, v, *t, q=q, cos=cos, sin=sin)
    want = attend(turned, cache, *t, **args)
    assert ops.kv_append(cache, k, v, *t, q=q, cos=cos, sin=sin, q_out=q) is q and torch.equal(q, turned)
    assert attend(q, cache, *t, out=q, **args) is q and torch.equal(q, want)
    ops.kv_status()


def test_attention_block_of_a_decoding_host(dev, rng):
    """A prompt, then decoded tokens, of one attention block as a host runs it: RMSNorm, fused q|k|v GEMV on packed q4_0
    weights, append, attention, output projection with the residual. Every stage against float64 on that stage's own inputs."""
    H, Hq, Hkv, D, page, eps = 256, 4, 2, 64, 16, 1e-6
    wq, wk, wv, wo = (synth.q4_0_weights(rng, n, kk) for n, kk in ((Hq * D, H), (Hkv * D, H), (Hkv * D, H), (H, Hq * D)))
    dw = on(dev, wq, wk, wv, wo)
    norm = torch.from_numpy(np.abs(rng.standard_normal(H)).astype(np.float32)).to(dev)
    lens = [11, 30]
    table, _, _, n_pages = tables(rng, [(0, 64), (0, 64)], page)
    want = random_cache(rng, n_pages, Hkv, page, D)
    cache = device_cache(dev, want)
    cos, sin = angles(64, D)
    dcos, dsin = on(dev, cos, sin)
    attend = ops.KvAttention(Hq, Hkv, D, dev)
    ctx = np.zeros(2, np.int32)
    for step in range(6):
        n = np.array(lens if step == 0 else [1, 1])
        ctx = (ctx + n).astype(np.int32)
        start = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
        T = int(start[-1])
        x = torch.randn(T, H, device=dev)
        h = ops.rmsnorm_q8(x, norm, eps, y_dtype=torch.float32, q8=False)[0]
        qkv = torch.empty(T, (Hq + 2 * Hkv) * D, device=dev)
        for r in range(T):  # one row at a time, as a GEMV host does
            row = qkv[r]
            ops.gemv_q4_0_seg3(h[r], H, [(dw[0], row[:Hq * D], Hq * D), (dw[1], row[Hq * D:(Hq + Hkv) * D], Hkv * D),
                                         (dw[2], row[(Hq + Hkv) * D:], Hkv * D)])
        q, k, v = (t.unflatten(1, (-1, D)) for t in qkv.split([Hq * D, Hkv * D, Hkv * D], 1))
        t = on(dev, table, start, ctx)
        qr = ops.kv_append(cache, k, v, *t, q=q, cos=dcos, sin=dsin)
        f = lambda a: a.cpu().numpy()
        q_want = oracle_append(want, f(k), f(v), f(q), table, start, ctx, cos, sin, False)
        same_cache(cache, want)
        np.testing.assert_array_equal(f(qr), q_want)
        o = attend(qr, cache, *t)
        check_attention(o, None, q_want.astype(np.float64), want, table, start, ctx, D ** -0.5, True, 0, "f32")
        for r in range(T):
            y = ops.gemv(ops.GGML_Q4_0, dw[3], o[r].reshape(-1), H, Hq * D, residual=x[r])
            ref = matmul.gemv_q4_0_f64(wo, f(o[r].reshape(-1)), H, Hq * D)[0] + f(x[r]).astype(np.float64)
            assert matmul.rel_maxnorm(f(y), ref) < matmul.TOL
    ops.kv_status()
