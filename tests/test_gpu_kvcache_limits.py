"""Attention over the 8-bit cache at the ends of its ranges: scores past the whole numbers that float32 tells apart, and
below every reference; sliding windows behind which pages are gone; batches larger than one lane or one counter each."""

import concurrent.futures
import threading

import numpy as np
import pytest
import torch

from oracle import kvcache
from vybforge_amd import _lib, ops

from test_gpu_kvcache import DT, check_attention, device_cache, on, random_cache, same_cache, tables, tolerance

pytestmark = pytest.mark.gpu

VARIANTS = [(0, "bf16", 64), (0, "f32", 256), (1, "f16", 128), (1, "f32", 64), (2, "f16", 64), (2, "f32", 128), (2, "bf16", 192),
            (2, "f32", 256), (3, "bf16", 128), (3, "f16", 128)]
LENS = [(1, 700), (70, 203), (0, 50), (33, 33), (5, 90), (3, 2)]


def force(monkeypatch, variant, splits):
    monkeypatch.setenv("VYBDQ_KV_VARIANT", str(variant))
    monkeypatch.setenv("VYBDQ_KV_SPLITS", str(splits))


def score_error(reach, D, x):
    """tolerance()'s bound on a score's error, in nats."""
    return reach * ((D + 8) * 2.0 ** -24 + (2.0 ** -22 if x == "f32" else 0)) + (64 + 1.5 * reach) * 2.0 ** -24 + 2.0 ** -22


def check_large(got, stats, q, want, table, start, ctx, scale, window, x):
    """Rows whose scores stay below 2^18 by tolerance(). Of the others, whose scores are only known to more than one nat: the
    output lies among the values that the row sees, lse at the largest score; and where the largest score leads the next by
    more than both may be off and 40 nats (the weights of 3000 keys together below 2^-46), the output is that key's value,
    up to the rounding of its weight (2^-11, of two terms 2^-21), of their quotient and of the output. How many were led."""
    T, Hq, D = q.shape
    G, led, large = Hq // want.k.shape[1], 0, 0
    got, stats = got.double().cpu().numpy(), stats.double().cpu().numpy()
    half, wr = torch.finfo(DT[x]).eps / 2, 2.0 ** -21 if x == "f32" else 2.0 ** -11
    for b in range(len(ctx)):
        n = int(start[b + 1] - start[b])
        heads = [want.values(table[b], ctx[b], h) for h in range(Hq // G)]
        for hq in range(Hq):
            k, v = heads[hq // G]
            r = slice(start[b], start[b + 1])
            o, z, weight, reach = kvcache.attention(q[r, hq], k, v, ctx[b] - n, ctx[b], scale, True, window)
            to, tz = tolerance(o, np.where(np.isfinite(z), z, 0), weight, reach, D, ctx[b], x)
            for i in range(n):
                y, s, pos = got[start[b] + i, hq], stats[start[b] + i, hq], ctx[b] - n + i
                seen = np.arange(max(0, pos - window + 1) if window else 0, pos + 1)
                if not len(seen):
                    assert (y == 0).all() and np.isneginf(s), (b, hq, i)
                    continue
                if reach[i] < 2.0 ** 18:
                    assert (np.abs(y - o[i]) <= to[i]).all() and abs(s - z[i]) <= tz[i], (b, hq, i)
                    continue
                large += 1
                ds = score_error(reach[i], D, x)
                t, vs = (k[seen] @ q[start[b] + i, hq]) * scale, v[seen]
                assert abs(s - z[i]) <= ds + 2.0 ** -22 * abs(z[i]), (b, hq, i, s, z[i])
                room = (half + wr + (2 * len(seen) + 128) * 2.0 ** -23) * (1 + half) * np.abs(vs).max(0)
                assert (y <= vs.max(0) + room).all() and (y >= vs.min(0) - room).all(), (b, hq, i, y)
                order = np.argsort(t)
                if len(t) > 1 and t[order[-1]] - t[order[-2]] <= 2 * ds + 40:
                    continue
                led += 1
                top = vs[order[-1]]
                assert (np.abs(y - top) <= (half + wr + 2.0 ** -21) * (1 + half) * np.abs(top)).all(), (b, hq, i)
    return led, large


def run_large(dev, rng, lens, Hq, Hkv, D, page, x, size, sign=1, window=0, mixed=False):
    """Scores of about `size` nats, all negative with sign < 0; mixed: rows of sizes of their own, and pages whose keys are
    small, so that a row's scores jump from small to large and back."""
    table, start, ctx, n_pages = tables(rng, lens, page)
    want = random_cache(rng, n_pages, Hkv, page, D)
    want.k_scale[:] = 2.0 ** rng.integers(-1, 2, want.k_scale.shape)
    if mixed:
        want.k_scale *= 2.0 ** rng.choice([0, -30], want.k_scale.shape)
    if sign < 0:
        want.k &= 0x7f
    q = rng.standard_normal((int(start[-1]), Hq, D)) * (2.0 ** rng.integers(-30, 1, (int(start[-1]), Hq, 1)) if mixed else 1)
    q = torch.from_numpy((-np.abs(q) if sign < 0 else q).astype(np.float32)).to(DT[x])
    scale = size / (80 * D ** 0.5)
    got, stats = ops.KvAttention(Hq, Hkv, D, dev)(q.to(dev), device_cache(dev, want), *on(dev, table, start, ctx), scale=scale,
                                                  window=window, lse=True)
    ops.kv_status()
    return check_large(got, stats, q.double().numpy(), want, table, start, ctx, scale, window, x)


@pytest.mark.parametrize("size", [1e8, 1e9, 1e12, 1e33])
@pytest.mark.parametrize("variant,x,D", VARIANTS)
def test_large_scores(dev, rng, monkeypatch, variant, x, D, size):
    for splits in (1, 3):
        force(monkeypatch, variant, splits)
        led, large = run_large(dev, rng, LENS, 2, 1, D, 16, x, size)
        assert large > 100 and led > 0.9 * large


@pytest.mark.parametrize("size", [1e9, 1e35])
@pytest.mark.parametrize("variant,x,D", VARIANTS)
def test_rows_whose_scores_are_all_far_below_zero(dev, rng, monkeypatch, variant, x, D, size):
    """They have weights that sum to one like any others, and a finite lse."""
    for splits in (1, 3):
        force(monkeypatch, variant, splits)
        led, large = run_large(dev, rng, LENS, 2, 2, D, 32, x, size, sign=-1)
        assert large > 100 and led > 0.9 * large


@pytest.mark.parametrize("variant,x,D", VARIANTS)
def test_large_and_small_scores_side_by_side(dev, rng, monkeypatch, variant, x, D):
    """Rows of all sizes in one wave, over pages of small and of large keys."""
    for splits, window in ((1, 0), (3, 0), (2, 40)):
        force(monkeypatch, variant, splits)
        led, large = run_large(dev, rng, LENS, 3, 1, D, 16, x, 1e9, window=window, mixed=True)
        assert large > 50 and led > 0.5 * large


@pytest.mark.parametrize("x", ["f16", "f32"])
@pytest.mark.parametrize("n", [1, 6, 80])
def test_large_queries_and_keys(dev, rng, x, n):
    """Entries of some thousands in q and K at the usual scale, by the plan's own choice of kernel and splits."""
    D, page, Hq = 128, 64, 4
    table, start, ctx, n_pages = tables(rng, [(n, 2000), (n, 100)], page)
    want = random_cache(rng, n_pages, 1, page, D)
    want.k_scale[:] = 2.0 ** 6
    q = torch.from_numpy((rng.standard_normal((2 * n, Hq, D)) * 3000).astype(np.float32)).to(DT[x])
    got, stats = ops.KvAttention(Hq, 1, D, dev)(q.to(dev), device_cache(dev, want), *on(dev, table, start, ctx), lse=True, max_new=n)
    led, large = check_large(got, stats, q.double().numpy(), want, table, start, ctx, D ** -0.5, 0, x)
    assert large == 2 * n * Hq and led > 0.9 * large


@pytest.mark.parametrize("size", [1.0, 1e9, -1e9, -1e32])
@pytest.mark.parametrize("variant,x,D", VARIANTS)
def test_equal_scores_have_equal_weights(dev, rng, monkeypatch, variant, x, D, size):
    """All keys alike, over pages with scales of their own (the same values by other codes): every row is the mean of the
    values that it sees, whatever the scores' size, with lse the score and the logarithm of their number."""
    page, lens = 16, LENS[:-1]
    table, start, ctx, n_pages = tables(rng, lens, page)
    want = random_cache(rng, n_pages, 1, page, D)
    key, shift = rng.choice([8.0, 9.0, 12.0, 15.0, 30.0], D), rng.integers(-3, 4, n_pages)
    want.k[:] = kvcache.e4m3_encode(key * 2.0 ** -shift[:, None, None, None])
    want.k_scale[:] = 2.0 ** (shift[:, None] - 3.0)
    scale = size / (1.5 * D)
    q = torch.from_numpy(np.abs(rng.standard_normal((int(start[-1]), 2, D))).astype(np.float32)).to(DT[x])
    for splits in (1, 5):
        force(monkeypatch, variant, splits)
        got, stats = ops.KvAttention(2, 1, D, dev)(q.to(dev), device_cache(dev, want), *on(dev, table, start, ctx), scale=scale, lse=True)
        got, stats = got.double().cpu().numpy(), stats.double().cpu().numpy()
        for b, (n, c) in enumerate(lens):
            k, v = want.values(table[b], c, 0)
            for i in range(n):
                seen = c - n + i + 1
                for h in range(2):
                    qr = q[start[b] + i, h].double().numpy()
                    z, reach = qr @ k[0] * scale + np.log(seen), abs(qr @ k[0] * scale)
                    mean, weight = v[:seen].mean(0), np.abs(v[:seen]).mean(0)
                    rel = (2.0 ** -21 if x == "f32" else 2.0 ** -11) + (2 * c + 128) * 2.0 ** -23 + 2.0 ** -20
                    half = torch.finfo(DT[x]).eps / 2
                    at = start[b] + i, h
                    assert (np.abs(got[at] - mean) <= half * np.abs(mean) + rel * (1 + half) * weight).all(), (b, i, h)
                    assert abs(stats[at] - z) <= score_error(reach, D, x) + (c + 64) * 2.0 ** -23 + 2.0 ** -22 * (1 + abs(z)), (b, i, h)
    ops.kv_status()


def test_large_scores_and_value_scales_far_apart(dev, rng, monkeypatch):
    """The page of the leading key has values 2^12 below the largest page's."""
    for variant, x, D in VARIANTS:
        force(monkeypatch, variant, 2)
        table, start, ctx, n_pages = tables(rng, [(2, 200)], 16)
        want = random_cache(rng, n_pages, 1, 16, D)
        want.k_scale[:] = 1.0
        want.v_scale[:, 0] = 2.0 ** rng.choice([-12, -6, 0], n_pages)
        q = torch.from_numpy(rng.standard_normal((2, 4, D)).astype(np.float32)).to(DT[x])
        scale = 1e9 / (80 * D ** 0.5)
        got, stats = ops.KvAttention(4, 1, D, dev)(q.to(dev), device_cache(dev, want), *on(dev, table, start, ctx), scale=scale, lse=True)
        led, large = check_large(got, stats, q.double().numpy(), want, table, start, ctx, scale, 0, x)
        assert led >= 7 and large == 8


@pytest.mark.parametrize("gone", ["outside", "reused"])
@pytest.mark.parametrize("variant,x,D", VARIANTS)
def test_pages_behind_the_window_are_not_looked_at(dev, rng, monkeypatch, variant, x, D, gone):
    """A host that frees them leaves entries that name no page, or a page with NaN codes and scales."""
    for page, window, splits in ((16, 5, 1), (16, 40, 2), (16, 65, 1), (32, 40, 2), (64, 33, 1)):
        force(monkeypatch, variant, splits)
        lens = [(n, c) for n in (1, 3, 40) for c in (120, 129, 150, 160, 185)]
        table, start, ctx, n_pages = tables(rng, lens, page)
        want = random_cache(rng, n_pages + 1, 1, page, D)
        want.k[n_pages], want.v[n_pages], want.k_scale[n_pages], want.v_scale[n_pages] = 0x7f, 0x7f, np.nan, np.nan
        left = table.copy()
        for b, (n, c) in enumerate(lens):
            first = max(0, c - n - window + 1) // page  # the page of the first key that the first row sees
            left[b, :first] = -1 - b if gone == "outside" else n_pages
        q = torch.from_numpy(rng.standard_normal((int(start[-1]), 2, D)).astype(np.float32)).to(DT[x])
        for causal in (True, False):
            got, stats = ops.KvAttention(2, 1, D, dev)(q.to(dev), device_cache(dev, want), *on(dev, left, start, ctx), causal=causal,
                                                       window=window, lse=True)
            check_attention(got, stats, q.double().numpy(), want, table, start, ctx, D ** -0.5, causal, window, x)
            ops.kv_status()


@pytest.mark.parametrize("variant,x,D", VARIANTS)
def test_a_tile_is_not_touched_by_rows_of_another(dev, rng, monkeypatch, variant, x, D):
    """The places of a sequence's last tile that hold no row do not take part: its rows have the same bits whatever the first
    row holds (which another workgroup may be writing, with the output in place of q), however large its scores are."""
    force(monkeypatch, variant, 1)
    table, start, ctx, n_pages = tables(rng, [(133, 300)], 16)
    want = random_cache(rng, n_pages, 1, 16, D)
    cache, t = device_cache(dev, want), on(dev, table, start, ctx)
    attend = ops.KvAttention(1, 1, D, dev)
    q = torch.from_numpy(rng.standard_normal((133, 1, D)).astype(np.float32)).to(DT[x]).to(dev)
    got, stats = attend(q, cache, *t, lse=True)
    for first in (30.0, 1000.0, 0.0):
        q[0] = q[0].sign() * first
        again, again_stats = attend(q, cache, *t, lse=True)
        assert torch.equal(again[128:], got[128:]) and torch.equal(again_stats[128:], stats[128:]), first
        here = q.clone()
        assert torch.equal(attend(here, cache, *t, out=here), again)


def test_attention_object_is_refused_in_a_capture(dev):
    a = torch.ones(4, device=dev)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        b = a + 1
        with pytest.raises(RuntimeError, match="before a capture"):
            ops.KvAttention(2, 1, 64, dev)
    for _ in range(2):
        g.replay()
    torch.cuda.synchronize()
    assert (b == 2).all()


def test_append_at_a_position_past_two_to_the_thirty(dev, rng):
    """The last angles of tables of 2^30 + 16 rows (32 GiB each, of which one row is written and read)."""
    D, page, R, pos = 64, 256, 16, 2 ** 30 + 7
    if torch.cuda.mem_get_info()[0] < 70 << 30:
        pytest.skip("needs 70 GiB of free device memory")
    cos, sin = (torch.empty(2 ** 30 + 16, R // 2, device=dev) for _ in range(2))
    angle = torch.from_numpy(rng.uniform(0, 6, R // 2).astype(np.float32))
    cos[pos], sin[pos] = angle.cos().to(dev), angle.sin().to(dev)
    want = random_cache(rng, 2, 1, page, D)
    cache = device_cache(dev, want)
    table = torch.ones(1, pos // page + 1, dtype=torch.int32, device=dev)
    k, v = (rng.standard_normal((1, 1, D)).astype(np.float32) for _ in range(2))
    got = ops.kv_append(cache, *on(dev, k, v), table, *on(dev, np.array([0, 1], np.int32), np.array([pos + 1], np.int32)),
                        q=on(dev, k)[0], cos=cos, sin=sin)
    ops.kv_status()
    turned = kvcache.rotate(k[0], 0, angle.cos().numpy()[None], angle.sin().numpy()[None], False)
    np.testing.assert_array_equal(got[0].cpu().numpy(), turned)
    want.append(turned[None], v, np.array([1]), pos % page + 1)
    same_cache(cache, want)
    del cos, sin
    torch.cuda.empty_cache()


# ---- batches and splits that other tests do not reach ------------------------------------------------

@pytest.mark.parametrize("splits", [1, 2, 7])
@pytest.mark.parametrize("variant,x,D", VARIANTS)
def test_every_kernel_by_name(dev, rng, monkeypatch, variant, x, D, splits):
    """Each kernel where it exists (128 rows a workgroup: fp16 and bf16 queries, D = 128), past a batch of 64 steps."""
    force(monkeypatch, variant, splits)
    lens = [(1, 2300), (140, 333), (0, 50), (33, 33), (5, 90)]
    for Hq, Hkv, page, window, causal in ((3, 1, 16, 0, True), (4, 2, 64, 77, False)):
        table, start, ctx, n_pages = tables(rng, lens, page)
        want = random_cache(rng, n_pages, Hkv, page, D)
        q = torch.from_numpy(rng.standard_normal((int(start[-1]), Hq, D)).astype(np.float32)).to(DT[x])
        got, stats = ops.KvAttention(Hq, Hkv, D, dev)(q.to(dev), device_cache(dev, want), *on(dev, table, start, ctx), window=window,
                                                      causal=causal, lse=True)
        check_attention(got, stats, q.double().numpy(), want, table, start, ctx, D ** -0.5, causal, window, x)
    ops.kv_status()


def test_chosen_splits_by_length(dev, rng):
    """A call long enough that the plan itself gives longer sequences more splits: eager, and captured and replayed at other
    lengths; every replay equals the eager result, which is checked once."""
    D, page, n, Hq, Hkv = 256, 16, 5, 24, 4
    lens = [(n, int(c)) for c in np.linspace(6000, 300, 12)]
    table, start, ctx, n_pages = tables(rng, lens, page)
    want = random_cache(rng, n_pages, Hkv, page, D)
    cache, t = device_cache(dev, want), on(dev, table, start, ctx)
    attend, args = ops.KvAttention(Hq, Hkv, D, dev), dict(max_new=n, max_ctx=6000, lse=True)
    q = torch.from_numpy(rng.standard_normal((12 * n, Hq, D)).astype(np.float32))
    qd = q.to(dev)
    first, first_stats = (a.clone() for a in attend(qd, cache, *t, **args))
    for h in (0, 11, 23):  # (all heads would take the oracle a while)
        k_of, part = h // (Hq // Hkv), kvcache.Cache(want.k[:, [h // 6]], want.v[:, [h // 6]], want.k_scale[:, [h // 6]], want.v_scale[:, [h // 6]])
        check_attention(first[:, h:h + 1], first_stats[:, h:h + 1], q[:, h:h + 1].double().numpy(), part, table, start, ctx, D ** -0.5,
                        True, 0, "f32")
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        out, stats = attend(qd, cache, *t, **args)
    for i in range(5):
        t[2].copy_(torch.from_numpy(np.roll(ctx, i) - 13 * i))
        t[0].copy_(torch.from_numpy(np.roll(table, i, 0)))
        g.replay()
        eager, eager_stats = attend(qd, cache, *t, **args)
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and torch.equal(stats, eager_stats), i
        if i == 0:
            assert torch.equal(out, first) and torch.equal(stats, first_stats)
    ops.kv_status()


@pytest.mark.parametrize("variant,n", [(0, 1), (1, 1), (2, 33)])
@pytest.mark.parametrize("splits", [None, 40, 256])
def test_every_key_of_half_a_billion_counts_once(dev, monkeypatch, variant, n, splits):
    """2^29 + 100 keys of equal scores and values of one: all weights are the same power of two, so that a lane's sums (at most
    2^24 keys, four to an addition) are exact whole numbers of it, and the joined ones are rounded 300 times at most: a split
    of 256 that is lost, doubled or short of one key in 2^10 of its own would show."""
    D, page, ctx = 64, 256, 2 ** 29 + 100
    monkeypatch.setenv("VYBDQ_KV_VARIANT", str(variant))
    if splits:
        monkeypatch.setenv("VYBDQ_KV_SPLITS", str(splits))
    attend, cache, batch = half_a_billion(dev, n, D, page, ctx)
    got, stats = attend(torch.zeros(n, 1, D, device=dev), cache, *batch, causal=False, lse=True, max_new=n, max_ctx=ctx)
    assert np.abs(stats.double().cpu().numpy() - np.log(ctx)).max() < 300 * 2.0 ** -23 / 16
    assert np.abs(got.double().cpu().numpy() - 1).max() < 300 * 2.0 ** -23
    ops.kv_status()


def half_a_billion(dev, n, D, page, ctx):
    codes = lambda *s: torch.full(s, 0x38, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)  # (ones)
    cache = ops.KvCache(codes(1, 1, page, D), codes(1, 1, page // 4, D, 4), *(torch.ones(1, 1, device=dev) for _ in range(2)))
    table = torch.zeros(1, -(-ctx // page), dtype=torch.int32, device=dev)
    return ops.KvAttention(1, 1, D, dev), cache, (table, *on(dev, np.array([0, n], np.int32), np.array([ctx], np.int32)))


@pytest.mark.parametrize("variant", [0, 1, 2])
@pytest.mark.parametrize("splits", [1, 5, 32])
def test_more_keys_to_a_split_than_float32_sums_are_refused(dev, monkeypatch, variant, splits):
    force(monkeypatch, variant, splits)
    attend, cache, batch = half_a_billion(dev, 1, 64, 256, 2 ** 29 + 100)
    with pytest.raises(_lib.VybdqError, match="2\\^24"):
        attend(torch.zeros(1, 1, 64, device=dev), cache, *batch, causal=False, max_new=1)
    got, stats = attend(torch.zeros(1, 1, 64, device=dev), cache, *batch, max_new=1, window=1000, lse=True)
    assert (got == 1).all() and abs(stats.item() - np.log(1000)) < 2.0 ** -20


@pytest.mark.parametrize("B,Hkv,max_new", [(5000, 1, 1), (700, 8, 1), (700, 8, None), (70000, 1, None)])
def test_thousands_of_sequences(dev, rng, B, Hkv, max_new):
    """First tokens of more sequences than a wave has lanes twice over, and of more (sequence, head) pairs than the workspace
    counts arrivals for: attention returns what append stored, with the score as lse."""
    D, G = 64, 2
    q, k, v = (torch.randn(B, h, D, device=dev) for h in (G * Hkv, Hkv, Hkv))
    cache = ops.KvCache.empty(B, Hkv, D, 16, dev)
    cache.k.view(torch.uint8).fill_(0x7f)
    cache.v.view(torch.uint8).fill_(0x7f)
    table = torch.randperm(B, device=dev).to(torch.int32)[:, None].contiguous()
    start, ctx = torch.arange(B + 1, dtype=torch.int32, device=dev), torch.ones(B, dtype=torch.int32, device=dev)
    ops.kv_append(cache, k, v, table, start, ctx, max_new=max_new)
    out, lse = ops.KvAttention(G * Hkv, Hkv, D, dev)(q, cache, table, start, ctx, lse=True, max_new=max_new, max_ctx=4000)
    at = table[:, 0].long()
    kept = cache.k.view(torch.uint8)[at, :, 0].view(torch.float8_e4m3fn).double() * cache.k_scale[at, :, None].double()
    vals = cache.v.view(torch.uint8)[at, :, 0, :, 0].contiguous().view(torch.float8_e4m3fn).double() * cache.v_scale[at, :, None].double()
    assert ((kept - k.double()).abs() <= 2.0 ** -4 * k.double().abs() + cache.k_scale[at, :, None] * 2.0 ** -10).all()
    assert ((vals - v.double()).abs() <= 2.0 ** -4 * v.double().abs() + cache.v_scale[at, :, None] * 2.0 ** -10).all()
    each = lambda t: t.repeat_interleave(G, 1)
    score, reach = ((f(q.double()) * f(each(kept))).sum(-1) * D ** -0.5 for f in (lambda t: t, torch.abs))
    assert ((out.double() - each(vals)).abs() <= (2.0 ** -21 + 2.0 ** -22) * each(vals).abs()).all()
    assert ((lse.double() - score).abs() <= reach * (D + 8) * 2.0 ** -24 + reach * 2.0 ** -21 + 64 * 2.0 ** -24 + 2.0 ** -21).all()
    ops.kv_status()


@pytest.mark.parametrize("variant,x,D", [v for v in VARIANTS if v[0] >= 2])
def test_chunks_of_many_sequences(dev, rng, monkeypatch, variant, x, D):
    """More sequences than a wave has lanes, of many rows each, some of none."""
    force(monkeypatch, variant, 2)
    lens = [(int(n), int(n + c)) for n, c in zip(rng.integers(0, 40, 150), rng.integers(0, 60, 150))]
    table, start, ctx, n_pages = tables(rng, lens, 16)
    want = random_cache(rng, n_pages, 1, 16, D)
    q = torch.from_numpy(rng.standard_normal((int(start[-1]), 1, D)).astype(np.float32)).to(DT[x])
    got, stats = ops.KvAttention(1, 1, D, dev)(q.to(dev), device_cache(dev, want), *on(dev, table, start, ctx), lse=True)
    check_attention(got, stats, q.double().numpy(), want, table, start, ctx, D ** -0.5, True, 0, x)
    ops.kv_status()


@pytest.mark.parametrize("Hq,Hkv", [(1024, 1024), (2048, 1), (999, 3)])
def test_many_heads(dev, rng, Hq, Hkv):
    D, page, lens = 64, 16, [(1, 40), (2, 3)]
    table, start, ctx, n_pages = tables(rng, lens, page)
    want = random_cache(rng, n_pages, Hkv, page, D)
    q = torch.from_numpy(rng.standard_normal((3, Hq, D)).astype(np.float32)).to(torch.bfloat16)
    got, stats = ops.KvAttention(Hq, Hkv, D, dev)(q.to(dev), device_cache(dev, want), *on(dev, table, start, ctx), lse=True)
    check_attention(got, stats, q.double().numpy(), want, table, start, ctx, D ** -0.5, True, 0, "bf16")
    ops.kv_status()


def test_an_error_is_reported_once_whoever_asks(dev):
    """Four threads ask at once after a bad batch: one of them is told."""
    cache = ops.KvCache.empty(2, 1, 64, 16, dev)
    k = torch.zeros(1, 1, 64, device=dev)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)
    table, start, ctx, together = i32(7)[None], i32(0, 1), i32(1), threading.Barrier(4)

    def ask(_):
        together.wait()
        try:
            ops.kv_status()
        except _lib.VybdqError as e:
            return str(e)

    with concurrent.futures.ThreadPoolExecutor(4) as pool:
        for i in range(40):
            ops.kv_append(cache, k, k, table, start, ctx)
            torch.cuda.synchronize()
            told = [e for e in pool.map(ask, range(4)) if e]
            assert len(told) == 1 and "page of the table" in told[0], (i, told)
    ops.kv_status()


@pytest.mark.parametrize("n", [1, 20, 70])
def test_small_workspaces(dev, rng, n):
    """None, no room behind the counters, room for a few rows of splits: fewer splits, the same results to their rounding; what
    lies behind the given bytes stays."""
    D, page, Hq, Hkv = 64, 64, 4, 2
    table, start, ctx, n_pages = tables(rng, [(n, 5000), (n, 900)], page)
    want = random_cache(rng, n_pages, Hkv, page, D)
    cache, t = device_cache(dev, want), on(dev, table, start, ctx)
    q = torch.from_numpy(rng.standard_normal((2 * n, Hq, D)).astype(np.float32))
    attend, counters = ops.KvAttention(Hq, Hkv, D, dev), 16384
    whole = attend.ws_bytes
    for room in (-counters, 0, 1000, 200000, 3000000, whole - counters):
        attend.ws_bytes = counters + room
        attend.ws.zero_()
        end = attend.ws_ptr - attend.ws.data_ptr() + attend.ws_bytes
        attend.ws[end:] = 0x5a
        got, stats = attend(q.to(dev), cache, *t, max_new=n, max_ctx=5000, lse=True)
        check_attention(got, stats, q.double().numpy(), want, table, start, ctx, D ** -0.5, True, 0, "f32")
        assert (attend.ws[end:] == 0x5a).all() and (attend.ws[attend.ws_ptr - attend.ws.data_ptr():][:max(0, min(counters, counters + room))] == 0).all()
    ops.kv_status()
