"""The key/value cache operators as they are measured: appending to a paged 8-bit cache, and attention over it.

The cache of one layer is four tensors. Page p holds `page` consecutive tokens of one sequence:
  k        float8_e4m3fn [n_pages, Hkv, page, D]          code of key dim d of the token in slot s
  v        float8_e4m3fn [n_pages, Hkv, page / 4, D, 4]   value dim d of slot s at [s / 4, d, s % 4]
  k_scale  float32 [n_pages, Hkv], v_scale the same       a power of two; value = code * scale
The batch: q_start int32 [B + 1] (rows of sequence b are q_start[b] .. q_start[b + 1] - 1 of q, k, v), ctx int32 [B]
(tokens of the sequence after this step: its rows are the last ones), table int32 [B, W] (page of each run of
`page` tokens). Head sizes are those of the benchmark's decode stack (32 query heads, 8 key/value heads of 128)
and generic ones.
"""

import math

import torch

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
E4M3 = torch.float8_e4m3fn
E_MIN, E_MAX = -60, 60  # exponents that a page's scale may have


def listed():
    return [
        # one decoding sequence: latency only
        dict(name="append_b1", op="append", B=1, n=1, ctx=2000, ragged=False, Hq=32, Hkv=8, D=128, R=128, page=64,
             inter=False, x="bf16"),
        # a serving batch of decoding sequences at their own lengths
        dict(name="append_b128", op="append", B=128, n=1, ctx=1500, ragged=True, Hq=32, Hkv=8, D=128, R=128, page=64,
             inter=False, x="bf16"),
        # prompts of odd lengths, partly rotated interleaved heads of 256, small pages, float32 activations
        dict(name="append_f32_d256", op="append", B=7, n=301, ctx=700, ragged=True, Hq=24, Hkv=4, D=256, R=64, page=16,
             inter=True, x="f32"),
        # a prefill step of 8 k tokens
        dict(name="append_8k", op="append", B=5, n=1638, ctx=1800, ragged=True, Hq=32, Hkv=8, D=128, R=128, page=64,
             inter=False, x="bf16"),
        # one decoding sequence of a few thousand tokens
        dict(name="attn_b1", op="attn", B=1, n=1, ctx=4001, ragged=False, Hq=32, Hkv=8, D=128, page=64, window=0,
             causal=True, lse=False, x="bf16"),
        # a serving batch at its own lengths
        dict(name="attn_b48", op="attn", B=48, n=1, ctx=8192, ragged=True, Hq=32, Hkv=8, D=128, page=64, window=0,
             causal=True, lse=False, x="bf16"),
        # drafted tokens checked together, float32 activations, heads of 256, six query heads a key head
        dict(name="attn_draft_f32", op="attn", B=12, n=5, ctx=6000, ragged=True, Hq=24, Hkv=4, D=256, page=16, window=0,
             causal=True, lse=True, x="f32"),
        # a few very long sequences
        dict(name="attn_long", op="attn", B=4, n=1, ctx=131072, ragged=True, Hq=32, Hkv=8, D=128, page=128, window=0,
             causal=True, lse=False, x="f16"),
        # a prompt from its beginning
        dict(name="attn_prompt", op="attn", B=1, n=4096, ctx=4096, ragged=False, Hq=32, Hkv=8, D=128, page=64, window=0,
             causal=True, lse=False, x="bf16"),
        # odd prompt chunks behind longer contexts, sliding window, small heads and pages, statistics kept
        dict(name="attn_chunk_window", op="attn", B=3, n=1000, ctx=9000, ragged=True, Hq=16, Hkv=16, D=64, page=16,
             window=4096, causal=True, lse=True, x="f16"),
        # a chunk behind a long context
        dict(name="attn_chunk_long", op="attn", B=1, n=513, ctx=32768, ragged=False, Hq=32, Hkv=8, D=128, page=64,
             window=0, causal=True, lse=False, x="bf16"),
    ]


def draw(rng):
    def log(a, b):
        return min(b, max(a, int(round(math.exp(rng.uniform(math.log(a), math.log(b + 1)))))))

    x, page = rng.choice(("bf16", "bf16", "f16", "f32")), rng.choice((16, 32, 64, 128, 256))
    D = rng.choice((64, 128, 128, 192, 256))
    Hkv = rng.choice((1, 2, 4, 5, 8))
    Hq = Hkv * rng.choice((1, 2, 3, 4, 6, 7, 8))
    kind = rng.choice(("append", "decode", "decode", "draft", "prompt"))
    if kind == "append":
        R = rng.choice([r for r in (0, 32, 64, 96, 128, 192, 256) if r <= D])
        if rng.random() < 0.5:
            B, n = log(1, 256), 1
        else:
            B = log(1, 16)
            n = log(2, 8192 // B)
        return dict(op="append", B=B, n=n, ctx=n + log(1, 2000), ragged=B > 1, Hq=Hq, Hkv=Hkv, D=D, R=R, page=page,
                    inter=rng.random() < 0.4, x=x)
    window = log(64, 8192) if rng.random() < 0.25 else 0
    if kind == "prompt":
        B, n = log(1, 4), log(17, 2048)
        ctx = min(n + (log(1, 12000) if rng.random() < 0.6 else 0), max(n, (1 << 23) // (n * B)))
    else:
        B, n = log(1, 64), rng.randint(2, 8) if kind == "draft" else 1
        ctx = max(n, min(log(n, 131072), 400000 // (B * n)))
    return dict(op="attn", B=B, n=n, ctx=ctx, ragged=B > 1 and rng.random() < 0.8, Hq=Hq, Hkv=Hkv, D=D, page=page,
                window=window, causal=rng.random() < 0.9, lse=rng.random() < 0.3, x=x)


# ---- inputs -----------------------------------------------------------------------------------

def _lengths(case):
    """Rows and tokens of every sequence: (n_b, ctx_b), the first of the full size, ragged ones below it."""
    B, n, ctx = case["B"], case["n"], case["ctx"]
    if not case["ragged"]:
        return [(n, ctx)] * B
    got = []
    for b in range(B):
        f = 1.0 - 0.75 * ((b * 0.6180339887) % 1.0)  # spread over [0.25, 1]
        nb = n if n < 2 else max(1, int(n * f))
        got.append((nb, max(nb, int(ctx * f))))
    return got


def _batch(case, g):
    page, lens = case["page"], _lengths(case)
    W = -(-max(c for _, c in lens) // page)
    used = [-(-c // page) for _, c in lens]
    n_pages = sum(used) + 3
    order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    at = torch.arange(W, device="cuda")[None, :]
    use = torch.tensor(used, device="cuda")[:, None]
    base = use.cumsum(0) - use
    table = order[(base + torch.minimum(at, use - 1)).long()].contiguous()
    start = torch.tensor([0] + [n for n, _ in lens], dtype=torch.int32).cumsum(0).to(torch.int32).cuda()
    ctx = torch.tensor([c for _, c in lens], dtype=torch.int32).cuda()
    return {"T": sum(n for n, _ in lens), "B": case["B"], "W": W, "n_pages": n_pages, "max_new": max(n for n, _ in lens),
            "max_ctx": max(c for _, c in lens), "table": table, "q_start": start, "ctx": ctx}


def _codes(g, n_pages, Hkv, page, D):
    """Codes and scales as appending N(0, 1) values leaves them: the largest of a page between 224 and 448."""
    k = torch.empty(n_pages, Hkv, page, D, device="cuda", dtype=E4M3)
    v = torch.empty(n_pages, Hkv, page // 4, D, 4, device="cuda", dtype=E4M3)
    for t in (k, v):
        t.copy_((torch.randn(t.shape, generator=g, device="cuda") * 80.0).clamp(-448, 448))
    scale = lambda: torch.exp2(torch.randint(-8, -5, (n_pages, Hkv), generator=g, device="cuda").float())  # noqa: E731
    return k, v, scale(), scale()


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    s = dict(case)
    s |= _batch(case, g)
    T, Hq, Hkv, D, dt = s["T"], s["Hq"], s["Hkv"], s["D"], DT[s["x"]]
    s["k_code"], s["v_code"], s["k_scale"], s["v_scale"] = _codes(g, s["n_pages"], Hkv, s["page"], D)
    if s["op"] == "append":
        # one projection's output: q, k and v of a token side by side
        qkv = torch.randn(T, (Hq + 2 * Hkv) * D, generator=g, device="cuda").to(dt)
        s["q"] = qkv[:, :Hq * D].unflatten(1, (Hq, D))
        s["k"] = qkv[:, Hq * D:(Hq + Hkv) * D].unflatten(1, (Hkv, D))
        s["v"] = qkv[:, (Hq + Hkv) * D:].unflatten(1, (Hkv, D))
        s["cos"] = s["sin"] = None
        if s["R"]:
            # angles in 64 bits: position / 10000^(2 i / R)
            freq = 10000.0 ** (-torch.arange(0, s["R"], 2, device="cuda", dtype=torch.float64) / s["R"])
            angle = torch.arange(s["max_ctx"], device="cuda", dtype=torch.float64)[:, None] * freq
            s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    else:
        s["q"] = torch.randn(T, Hq, D, generator=g, device="cuda").to(dt)
    if own:
        from vybforge_amd import ops
        s["cache"] = ops.KvCache(s["k_code"], s["v_code"], s["k_scale"], s["v_scale"])
        s["attention"] = ops.KvAttention(Hq, Hkv, D, "cuda")
    return s


# ---- the operators ----------------------------------------------------------------------------

def run(s):
    if s["op"] == "append":
        if own:
            from vybforge_amd import ops
            q = ops.kv_append(s["cache"], s["k"], s["v"], s["table"], s["q_start"], s["ctx"], q=s["q"], cos=s["cos"],
                              sin=s["sin"], interleaved=s["inter"], max_new=s["max_new"])
        else:
            q = _append(s)
        return {"q": q, "k": s["k_code"], "v": s["v_code"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    if own:
        return s["attention"](s["q"], s["cache"], s["table"], s["q_start"], s["ctx"], causal=s["causal"],
                              window=s["window"], max_new=s["max_new"], max_ctx=s["max_ctx"], lse=s["lse"])
    return _attention(s)


def _rows(s):
    """Sequence and position of every row."""
    row = torch.arange(s["T"], device=s["q_start"].device)
    b = torch.searchsorted(s["q_start"].long(), row, right=True) - 1
    return b, row - s["q_start"].long()[b + 1] + s["ctx"].long()[b]


def _rotate(x, pos, s):
    """x float32 [T, H, D] with its first R dims turned by the angles of the rows' positions."""
    R = s["R"]
    if not R:
        return x
    c, n = s["cos"][pos][:, None], s["sin"][pos][:, None]
    out = x.clone()
    a, b = (slice(0, R, 2), slice(1, R, 2)) if s["inter"] else (slice(0, R // 2), slice(R // 2, R))
    out[..., a] = x[..., a] * c - x[..., b] * n
    out[..., b] = x[..., b] * c + x[..., a] * n
    return out


def _exponent(amax):
    """The least e with amax <= 448 * 2^e, within E_MIN .. E_MAX: 448 = 0.875 * 2^9."""
    f, x = torch.frexp(amax)
    e = torch.where(f <= 0.875, x - 9, x - 8)
    return torch.where(amax == 0, E_MIN, e).clamp(E_MIN, E_MAX)


def _append(s):
    page, Hkv, D = s["page"], s["Hkv"], s["D"]
    b, pos = _rows(s)
    pg, slot = s["table"][b, pos // page].long(), pos % page
    q = _rotate(s["q"].float(), pos, s).to(s["q"].dtype)
    # pages that the rows reach: of every sequence the first and the following, the last one again where there are fewer
    n = s["q_start"].diff().long()
    first, last = (s["ctx"].long() - n) // page, (s["ctx"].long() - 1) // page
    most = (s["max_new"] + page - 2) // page + 1
    index = torch.minimum(first[:, None] + torch.arange(most, device=pos.device), last[:, None])
    pages = torch.gather(s["table"], 1, index).long()
    # tokens that stay in them: those before the sequence's first row
    kept = ((s["ctx"].long() - n)[:, None] - index * page).clamp(0, page)
    for x, codes, scale in ((_rotate(s["k"].float(), pos, s), s["k_code"], s["k_scale"]), (s["v"].float(), s["v_code"], s["v_scale"])):
        need = torch.zeros_like(scale)
        need.scatter_reduce_(0, pg[:, None].expand(-1, Hkv), x.abs().amax(-1), "amax")
        e_new, e_old = _exponent(need[pages]), torch.frexp(scale[pages])[1] - 1
        e_new = torch.where(kept[..., None] > 0, torch.maximum(e_new, e_old), e_new)
        raw = codes.view(torch.uint8)
        held = raw[pages]
        rest = (1,) * (codes.dim() - 2)  # a page's dims of one head
        again = held.view(E4M3).float() * torch.exp2((e_old - e_new).float()).reshape(e_new.shape + rest)
        again = again.to(E4M3).view(torch.uint8)
        at = torch.arange(page, device=pos.device)
        at = at[:, None] if codes.dim() == 4 else at.view(page // 4, 1, 4)
        stays = at < kept.reshape(kept.shape + (1,) + rest)
        raw[pages] = torch.where(stays, again, held)
        scale[pages] = torch.exp2(e_new.float())
        new = (x * torch.reciprocal(scale[pg])[..., None]).clamp(-448, 448).to(E4M3).view(torch.uint8)
        if codes.dim() == 4:
            raw[pg, :, slot] = new
        else:
            raw[pg, :, slot // 4, :, slot % 4] = new
    return q


def _attention(s):
    B, Hq, Hkv, D, page, n = s["B"], s["Hq"], s["Hkv"], s["D"], s["page"], s["max_new"]
    G, L = Hq // Hkv, s["W"] * page
    table = s["table"].long()
    # keys and values of every sequence in order, float32 [B, Hkv, L, D]
    k = (s["k_code"].view(torch.uint8)[table].view(E4M3).float() * s["k_scale"][table][..., None, None])
    k = k.transpose(1, 2).reshape(B, Hkv, L, D)
    v = (s["v_code"].view(torch.uint8)[table].view(E4M3).float() * s["v_scale"][table][..., None, None, None])
    v = v.permute(0, 2, 1, 3, 5, 4).reshape(B, Hkv, L, D)
    # rows padded to the longest sequence's
    start, end, ctx = s["q_start"][:-1].long(), s["q_start"][1:].long(), s["ctx"].long()
    i = torch.arange(n, device=k.device)
    row = torch.minimum(start[:, None] + i, end[:, None] - 1)
    q = s["q"].float()[row].unflatten(2, (Hkv, G)).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * n, D)
    t = (q @ k.transpose(2, 3)) * (D ** -0.5)
    pos = ctx[:, None] - end[:, None] + start[:, None] + i
    j = torch.arange(L, device=k.device)
    seen = (j < ctx[:, None])[:, None, :].expand(B, n, L)
    if s["causal"]:
        seen = seen & (j <= pos[..., None])
    if s["window"]:
        seen = seen & (j > pos[..., None] - s["window"])
    t = t.view(B, Hkv, G, n, L).masked_fill_(~seen[:, None, None], -math.inf)
    m = t.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    p = t.sub_(m).exp_()
    l = p.sum(-1, keepdim=True)
    o = (p.view(B, Hkv, G * n, L) @ v).view(B, Hkv, G, n, D) / torch.where(l == 0, 1.0, l)
    b, at = _rows(s)[0], torch.arange(s["T"], device=k.device)
    at = at - start[b]
    out = o[b, :, :, at].reshape(s["T"], Hq, D).to(s["q"].dtype)
    if not s["lse"]:
        return out
    return out, (m + l.log())[b, :, :, at].reshape(s["T"], Hq)


# ---- what a pass cannot do without --------------------------------------------------------------

def work(case):
    es, lens = DT[case["x"]].itemsize, _lengths(case)
    Hq, Hkv, D, page = case["Hq"], case["Hkv"], case["D"], case["page"]
    T = sum(n for n, _ in lens)
    if case["op"] == "append":
        pages = sum((c - 1) // page - (c - n) // page + 1 for n, c in lens)
        return {"bytes": T * D * ((2 * Hq + 2 * Hkv) * es + 2 * Hkv) + T * case["R"] * 4 + pages * (4 + 16 * Hkv),
                "flops": T * (Hq + Hkv) * case["R"] * 3}
    seen, read = 0, 0
    for n, c in lens:
        w = case["window"] or c + n
        first = max(0, c - n - w + 1)
        read += c - first
        if case["causal"]:
            seen += sum(min(w, c - n + i + 1) for i in range(n))
        else:
            seen += sum(c - max(0, c - n + i + 1 - w) for i in range(n))
    pages = -(-read // page)
    return {"bytes": 2 * read * Hkv * D + pages * (4 + 8 * Hkv) + 2 * T * Hq * D * es + (4 * T * Hq if case["lse"] else 0),
            "flops": 4 * seen * Hq * D}


# ---- the definition in 64 bits --------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    dev, page, Hkv, D, G = s["q"].device, s["page"], s["Hkv"], s["D"], s["Hq"] // s["Hkv"]
    lens, F = _lengths(case), torch.float64
    table, at = s["table"].cpu().tolist(), 0
    if s["op"] == "append":
        q_out = s["q"].to(F)
        k_val, v_val = s["k_code"].to(F), s["v_code"].to(F)
        k_scale, v_scale = s["k_scale"].to(F), s["v_scale"].to(F)
        half = s["R"] // 2

        def turned(x, p0):
            if not half:
                return x
            z = torch.complex(x[..., 0:2 * half:2], x[..., 1:2 * half:2]) if s["inter"] else torch.complex(x[..., :half], x[..., half:2 * half])
            span = slice(p0, p0 + x.shape[0])
            z = z * torch.complex(s["cos"][span].to(F), s["sin"][span].to(F))[:, None]
            y = torch.view_as_real(z).flatten(-2) if s["inter"] else torch.cat((z.real, z.imag), -1)
            return torch.cat((y, x[..., 2 * half:]), -1)

        def code(x):
            """x rounded to a value of e4m3, ties to even: three bits behind the leading one, steps of 2^-9 at least."""
            step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
            return (torch.round(x / step) * step).clamp(-448, 448)

        for b, (n, c) in enumerate(lens):
            rows, p0 = slice(at, at + n), c - n
            q_out[rows] = turned(s["q"][rows].to(F), p0)
            news = ((turned(s["k"][rows].to(F), p0), k_val, k_scale), (s["v"][rows].to(F), v_val, v_scale))
            for x, val, scale in news:
                for i in range(p0 // page, (c - 1) // page + 1):
                    lo, hi, pg = max(p0, i * page), min(c, (i + 1) * page), table[b][i]
                    new = x[lo - p0:hi - p0].transpose(0, 1)                      # [Hkv, tokens, D]
                    have = val[pg] if val.dim() == 4 else val[pg].transpose(-1, -2).reshape(Hkv, page, D)
                    e = torch.ceil(torch.log2(new.abs().amax((1, 2)) / 448).clamp(E_MIN, E_MAX))
                    keep = lo - i * page
                    if keep:
                        e = torch.maximum(e, torch.log2(scale[pg]))
                        have[:, :keep] = code(have[:, :keep] * (scale[pg] / torch.exp2(e))[:, None, None])
                    scale[pg] = torch.exp2(e)
                    have[:, keep:keep + hi - lo] = code(new / scale[pg][:, None, None])
                    val[pg] = have if val.dim() == 4 else have.view(Hkv, page // 4, 4, D).transpose(-1, -2)
            at += n
        return {"q": q_out, "k": k_val, "v": v_val, "k_scale": k_scale, "v_scale": v_scale}
    if work(case)["flops"] > 5e12:
        return None
    out = torch.empty(s["T"], s["Hq"], D, dtype=F, device=dev)
    lse = torch.empty(s["T"], s["Hq"], dtype=F, device=dev)
    for b, (n, c) in enumerate(lens):
        pg = torch.tensor(table[b][:-(-c // page)], device=dev)
        for h in range(Hkv):
            k = (s["k_code"].view(torch.uint8)[pg, h].view(E4M3).to(F) * s["k_scale"][pg, h].to(F)[:, None, None]).reshape(-1, D)[:c]
            v = s["v_code"].view(torch.uint8)[pg, h].view(E4M3).to(F) * s["v_scale"][pg, h].to(F)[:, None, None, None]
            v = v.transpose(-1, -2).reshape(-1, D)[:c]
            j = torch.arange(c, device=dev)
            for i0 in range(0, n, 512):
                i1 = min(n, i0 + 512)
                pos = torch.arange(c - n + i0, c - n + i1, device=dev)[:, None]
                hidden = torch.zeros(i1 - i0, c, dtype=torch.bool, device=dev)
                if s["causal"]:
                    hidden |= j > pos
                if s["window"]:
                    hidden |= j <= pos - s["window"]
                q = s["q"][at + i0:at + i1, h * G:(h + 1) * G].to(F)
                t = (q.reshape(-1, D) @ k.T).view(i1 - i0, G, c) / math.sqrt(D)
                t = t.masked_fill(hidden[:, None], -math.inf)
                z = torch.logsumexp(t, -1, keepdim=True)
                w = torch.where(z == -math.inf, 0.0, torch.exp(t - z))
                out[at + i0:at + i1, h * G:(h + 1) * G] = (w.view(-1, c) @ v).view(i1 - i0, G, D)
                lse[at + i0:at + i1, h * G:(h + 1) * G] = z[..., 0]
        at += n
    return (out, lse) if s["lse"] else out
