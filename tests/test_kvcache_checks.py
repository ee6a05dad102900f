"""Refusals of the key/value cache's entry points: return codes of the C-ABI before any launch, and the wrappers' checks.
CPU only: no call here reaches the GPU."""

import re

import pytest
import torch

from vybforge_amd import _lib, ops

APPEND = dict(K=256, V=256, Ks=4, Vs=4, n_pages=4, Hkv=2, D=64, page=16, k=16, v=16, q=16, q_out=16, x_dt=0, ldk=128, ldv=128,
              ldq=256, Hq=4, cos=16, sin=16, R=64, n_pos=10, interleaved=0, table=4, W=2, q_start=4, ctx=4, T=3, B=1, max_new=0,
              stream=0)
ATTN = dict(K=256, V=256, Ks=4, Vs=4, n_pages=4, Hkv=2, D=64, page=16, q=16, x_dt=0, ldq=256, Hq=4, out=16, lse=0, table=4, W=2,
            q_start=4, ctx=4, T=3, B=1, max_new=0, max_ctx=0, scale=0.125, causal=1, window=0, ws=256, ws_bytes=0, stream=0)
BOTH = [
    (dict(x_dt=3), _lib.ERR_ARG, "x_dt"), (dict(D=96), _lib.ERR_SHAPE, "D must"), (dict(page=24), _lib.ERR_SHAPE, "page must"),
    (dict(page=8), _lib.ERR_SHAPE, "page must"), (dict(page=512), _lib.ERR_SHAPE, "page must"),
    (dict(n_pages=0), _lib.ERR_SHAPE, "n_pages"), (dict(n_pages=2 ** 31), _lib.ERR_SHAPE, "n_pages"),
    (dict(Hkv=0), _lib.ERR_SHAPE, "Hkv"), (dict(Hq=3), _lib.ERR_SHAPE, "multiple of Hkv"), (dict(Hq=0), _lib.ERR_SHAPE, "multiple of Hkv"),
    (dict(T=-1), _lib.ERR_SHAPE, "T must"), (dict(T=2 ** 30), _lib.ERR_SHAPE, "T must"), (dict(B=2 ** 20), _lib.ERR_SHAPE, "B below"),
    (dict(W=0), _lib.ERR_SHAPE, "W must"), (dict(W=2 ** 28), _lib.ERR_SHAPE, "W \\* page"),
    (dict(K=0), _lib.ERR_ARG, "null"), (dict(table=0), _lib.ERR_ARG, "null"), (dict(ctx=0), _lib.ERR_ARG, "null"),
    (dict(K=264), _lib.ERR_ALIGN, "16-byte"), (dict(q=24), _lib.ERR_ALIGN, "16-byte"), (dict(ldq=258), _lib.ERR_ALIGN, "16-byte"),
    (dict(ldq=252), _lib.ERR_SHAPE, "stride"), (dict(Ks=6), _lib.ERR_ALIGN, "4-byte"), (dict(q_start=6), _lib.ERR_ALIGN, "4-byte"),
]


@pytest.mark.parametrize("change,code,text", BOTH + [
    (dict(R=24), _lib.ERR_SHAPE, "R must"), (dict(R=80), _lib.ERR_SHAPE, "R must"), (dict(cos=0), _lib.ERR_ARG, "cos and sin"),
    (dict(n_pos=0), _lib.ERR_ARG, "cos and sin"), (dict(q_out=0), _lib.ERR_ARG, "q_out"), (dict(ldv=120), _lib.ERR_SHAPE, "stride"),
    (dict(v=20), _lib.ERR_ALIGN, "16-byte"), (dict(sin=20), _lib.ERR_ALIGN, "16-byte"),
    (dict(B=2 ** 20 - 1, Hkv=8, Hq=8), _lib.ERR_SHAPE, "2\\^23"), (dict(T=2 ** 26, page=16, Hkv=2), _lib.ERR_SHAPE, "2\\^23"),
])
def test_append_refuses(change, code, text):
    assert _lib.lib.vybdq_kv_append(*(APPEND | change).values()) == code
    assert re.search(text, _lib.last_error())


@pytest.mark.parametrize("change,code,text", BOTH + [
    (dict(window=-1), _lib.ERR_SHAPE, "window"), (dict(window=2 ** 30), _lib.ERR_SHAPE, "window"), (dict(out=0), _lib.ERR_ARG, "null"),
    (dict(B=2 ** 20 - 1, Hkv=32, Hq=32), _lib.ERR_SHAPE, "2\\^24"), (dict(T=2 ** 28, Hkv=4, Hq=4), _lib.ERR_SHAPE, "2\\^24"),
    (dict(out=20), _lib.ERR_ALIGN, "16-byte"), (dict(lse=6), _lib.ERR_ALIGN, "4-byte"), (dict(ws=128), _lib.ERR_ALIGN, "256-byte"),
])
def test_attention_refuses(change, code, text):
    assert _lib.lib.vybdq_kv_attn(*(ATTN | change).values()) == code
    assert re.search(text, _lib.last_error())


@pytest.mark.parametrize("change", [dict(), dict(ws=0, ws_bytes=0, max_ctx=2 ** 24 + 1), dict(window=2 ** 25), dict(x_dt=1, T=100),
                                    dict(Hq=64, Hkv=2, ldq=4096)])
def test_attention_refuses_more_keys_than_a_split_can_sum(change):
    """No workspace to split 2^29 keys, or a bound on them, in."""
    assert _lib.lib.vybdq_kv_attn(*(ATTN | dict(W=2 ** 25) | change).values()) == _lib.ERR_SHAPE
    assert "2^24" in _lib.last_error()


def test_nothing_to_do_is_no_launch():
    assert _lib.lib.vybdq_kv_append(*(APPEND | dict(T=0)).values()) == _lib.OK
    assert _lib.lib.vybdq_kv_append(*(APPEND | dict(B=0)).values()) == _lib.OK
    assert _lib.lib.vybdq_kv_attn(*(ATTN | dict(T=0)).values()) == _lib.OK
    assert _lib.lib.vybdq_kv_attn(*(ATTN | dict(B=0)).values()) == _lib.OK


def test_workspace_size():
    for D in ops.KV_HEAD_DIMS:
        assert _lib.lib.vybdq_kv_attn_workspace_size(D) > 0
    assert _lib.lib.vybdq_kv_attn_workspace_size(96) == -1


def test_cache_shapes():
    code = lambda *s: torch.empty(s, dtype=torch.float8_e4m3fn)
    scale = torch.ones(3, 2)
    good = code(3, 2, 16, 64), code(3, 2, 4, 64, 4)
    for k, v, ks, vs, text in (
            (code(3, 2, 16, 80), good[1], scale, scale, "D must"), (code(3, 2, 24, 64), good[1], scale, scale, "page must"),
            (good[0], code(3, 2, 16, 64), scale, scale, "v must"), (good[0].view(torch.int8), good[1], scale, scale, "float8"),
            (*good, scale.double(), scale, "scales"), (*good, scale, scale[:2], "scales"), (*good, scale, scale, "on the GPU")):
        with pytest.raises(ValueError, match=text):
            ops.KvCache(k, v, ks, vs)


class FakeCache:
    """What the wrappers ask of a cache, without a GPU."""
    n_heads, head_dim, page, index, _args = 2, 64, 16, -1, (256, 256, 4, 4, 4, 2, 64, 16)


def test_wrapper_checks():
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)
    k, q = torch.zeros(3, 2, 64), torch.zeros(3, 4, 64)
    batch = (i32(1, 2), i32(2), i32(1))
    for b, text in (((i32(1, 2), i32(3), i32(1)), "sequences"), ((i32(1, 2), i32(2), i32(2)), "sequences"), ((i32(2), i32(2), i32(1)), "page_table"),
                    ((i32(1, 2).long(), i32(2), i32(1)), "int32"), ((i32(1, 4)[:, ::2], i32(2), i32(1)), "contiguous")):
        with pytest.raises(ValueError, match=text):
            ops.kv_append(FakeCache, k, k, *b)
    more = (dict(cos=torch.zeros(4, 32)), "together"), (dict(q=q.half()), "q must"), (dict(q=q[:, :3]), "multiple"), (dict(q=q[:2]), "q must"), (
        dict(q_out=q), "needs q"), (dict(q=q, q_out=q[:2]), "q_out must"), (dict(cos=torch.zeros(4, 32).double(), sin=torch.zeros(4, 32)), "float32")
    for extra, text in more:
        with pytest.raises(ValueError, match=text):
            ops.kv_append(FakeCache, k, k, *batch, **extra)
    for kk, vv, text in ((k[:, :1], k, "k must"), (k, k[:2], "v must"), (k, k.half(), "dtype"), (k.transpose(0, 1), k, "k must"),
                         (torch.zeros(3, 64, 2).transpose(1, 2), k, "consecutive"), (torch.zeros(3, 2, 128)[:, :, :64], k, "consecutive")):
        with pytest.raises(ValueError, match=text):
            ops.kv_append(FakeCache, kk, vv, *batch)


def test_attention_object_checks():
    for args in ((4, 3, 64), (0, 1, 64), (4, 2, 100)):
        with pytest.raises(ValueError):
            ops.KvAttention(*args, device="cpu")


def test_attention_object_is_not_made_in_a_capture(monkeypatch):
    """Its workspace would be cleared by replays only, and an eager call before the first one would count on what was there."""
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="before a capture"):
        ops.KvAttention(4, 2, 64, device="cuda")
    with pytest.raises(RuntimeError, match="before a capture"):
        ops.KvAttention(4, 2, 64, device=torch.device("cuda", 0))
