"""Operators on 8-bit floating-point weights as they are measured: the quantizer of activations, the linear layer, the
router with groups of experts, and the mixture-of-experts layer.

A matrix W [N, K] is float8_e4m3fn codes [N, K] with float32 scales [ceil(N / 128), ceil(K / 128)], one for each block of
128 x 128: weight = code * scale. Activations X [M, K] get codes [M, K] and float32 scales [M, ceil(K / 128)], one for each
row and 128 columns: scale = 2^e with the least e in -100 .. 120 for which all |x| <= 448 * 2^e, code = e4m3(x / scale).
Sizes are those of the benchmark's layers (9728 x 2560, 17408 x 5120, 256 experts of 6144 x 2048 with 8 to a token) and
generic ones.
"""

import math

import torch

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
E4M3 = torch.float8_e4m3fn
BLOCK = 128
E_MIN, E_MAX = -100, 120  # exponents that a scale of activations may have


def listed():
    big = dict(H=6144, I=2048, E=256, k=8, shared=True, bias=True, score="sigmoid", renorm=True, scale=2.5)
    return [
        # one token's hidden state before a projection: latency only
        dict(name="quant_1", op="quant", M=1, K=6144, x="bf16"),
        # a prefill step's hidden states
        dict(name="quant_8k", op="quant", M=8192, K=6144, x="bf16"),
        # a decode step's projection, one sequence
        dict(name="linear_1", op="linear", M=1, N=9728, K=2560, x="bf16", y="bf16"),
        # a few rows through a small ragged projection that keeps float32 (a low-rank bottleneck)
        dict(name="linear_13_f32", op="linear", M=13, N=1003, K=2576, x="f32", y="f32"),
        # a serving batch through a down projection
        dict(name="linear_48", op="linear", M=48, N=5120, K=17408, x="bf16", y="bf16"),
        # a prompt through an up projection
        dict(name="linear_512", op="linear", M=512, N=17408, K=5120, x="bf16", y="bf16"),
        # a prefill step of several prompts through it
        dict(name="linear_4096", op="linear", M=4096, N=17408, K=5120, x="bf16", y="bf16"),
        # one token over experts in groups
        dict(name="route_1", op="route", T=1, E=256, k=8, groups=8, top_groups=4, group_top=2, bias=True, score="sigmoid",
             renorm=True, scale=2.5, x="f32"),
        # a prefill step over softmax scores whose weights stay as they are
        dict(name="route_16k", op="route", T=16384, E=160, k=6, groups=8, top_groups=3, group_top=1, bias=False,
             score="softmax", renorm=False, scale=1.0, x="bf16"),
        # a layer's decode step: one token
        dict(name="moe_1", op="moe", T=1, groups=1, top_groups=1, group_top=2, x="bf16", **big),
        # a decode step of a serving batch
        dict(name="moe_48", op="moe", T=48, groups=8, top_groups=4, group_top=2, x="bf16", **big),
        # a prefill step
        dict(name="moe_4096", op="moe", T=4096, groups=8, top_groups=4, group_top=2, x="bf16", **big),
    ]


def draw(rng):
    def log(a, b):
        return min(b, max(a, int(round(math.exp(rng.uniform(math.log(a), math.log(b + 1)))))))

    x, op = rng.choice(("bf16", "bf16", "f16", "f32")), rng.choice(("quant", "linear", "linear", "linear", "route", "moe", "moe"))
    if op == "quant":
        K = 16 * log(1, 1200)
        return dict(op=op, M=log(1, min(20000, 60000000 // K)), K=K, x=x)
    if op == "linear":
        M, K = log(1, 4096), 16 * log(8, 1100)
        N = min(log(16, 20000), max(16, 365000000000 // (M * K)))
        return dict(op=op, M=M, N=N, K=K, x=x, y=rng.choice(("bf16", "bf16", "f16", "f32")))
    groups = rng.choice((1, 1, 2, 4, 8))
    top_groups = rng.randint(1, groups)
    size = log(4, 64 if groups < 8 else 40)  # experts to a group
    E = groups * size
    rest = dict(E=E, k=rng.randint(1, min(8, top_groups * size)), groups=groups, top_groups=top_groups,
                group_top=rng.choice((1, 2)), bias=rng.random() < 0.6, score=rng.choice(("sigmoid", "sigmoid", "softmax")),
                renorm=rng.random() < 0.7, scale=rng.choice((1.0, 2.5)))
    if op == "route":
        return dict(op=op, T=log(1, 16384), x=rng.choice(("f32", "bf16", "f16")), **rest)
    H, I = 128 * log(2, 48), 128 * log(1, 16)
    return dict(op=op, T=log(1, min(4096, 32768 // rest["k"])), H=H, I=I, shared=rng.random() < 0.5, x=x, **rest)


# ---- inputs -----------------------------------------------------------------------------------

def _blocks(n):
    return -(-n // BLOCK)


def _weights(g, N, K, lead=()):
    """Codes and scales as quantizing N(0, 1 / K) weights block by block leaves them: the largest code near 448."""
    codes = torch.empty(lead + (N, K), dtype=E4M3, device="cuda")
    flat = codes.view(-1)
    step = 1 << 28
    for i in range(0, flat.numel(), step):
        part = flat[i:i + step]
        part.copy_((torch.randn(part.shape, generator=g, device="cuda") * 110.0).clamp_(-448, 448))
    scales = torch.rand(lead + (_blocks(N), _blocks(K)), generator=g, device="cuda") + 0.5
    return codes, scales * (K ** -0.5 / 110.0)


def _activations(g, rows, K, dt):
    """N(0, 1) with a few columns that are much larger, as hidden states have."""
    x = torch.randn(rows, K, generator=g, device="cuda")
    x *= 1.0 + 30.0 * (torch.rand(K, generator=g, device="cuda") < 0.002)
    return x.to(dt)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    s = dict(case)
    op, dt = s["op"], DT[s["x"]]
    if op in ("quant", "linear"):
        s["X"] = _activations(g, s["M"], s["K"], dt)
    if op == "linear":
        s["W"] = _weights(g, s["N"], s["K"])
    if op in ("route", "moe"):
        s["logits"] = torch.randn(s["T"], s["E"], generator=g, device="cuda") * 1.5
        if op == "route":
            s["logits"] = s["logits"].to(dt)
        s["b"] = torch.randn(s["E"], generator=g, device="cuda") * 0.05 if s["bias"] else None
    if op == "moe":
        H, I, E = s["H"], s["I"], s["E"]
        s["X"] = _activations(g, s["T"], H, dt)
        s["experts"] = [_weights(g, I, H, (E,)), _weights(g, I, H, (E,)), _weights(g, H, I, (E,))]
        s["one"] = [_weights(g, I, H), _weights(g, I, H), _weights(g, H, I)] if s["shared"] else None
    if own:
        from vybforge_amd import ops
        if op == "linear":
            s["layer"] = ops.Fp8Linear(*s["W"], max_rows=s["M"])
        if op == "moe":
            s["layer"] = ops.MoeFp8Layer(*s["experts"], topk=s["k"], shared=s["one"], bias=s["b"], **_routing(s))
    return s


def _routing(s):
    return {n: s[n] for n in ("scale", "score", "renorm", "groups", "top_groups", "group_top")}


# ---- the operators ----------------------------------------------------------------------------

def run(s):
    op = s["op"]
    if own:
        from vybforge_amd import ops
        if op == "quant":
            return ops.quant_fp8(s["X"])
        if op == "linear":
            return s["layer"](s["X"], y_dtype=DT[s["y"]])
        if op == "route":
            return ops.moe_route(s["logits"], s["k"], bias=s["b"], **_routing(s))
        return s["layer"](s["X"], s["logits"], out_dtype=torch.bfloat16)
    if op == "quant":
        return _quant(s["X"])
    if op == "linear":
        return (_values(*_quant(s["X"])) @ _matrix(*s["W"]).T).to(DT[s["y"]])
    if op == "route":
        return _route(s)
    return _moe(s)


def _quant(x):
    M, K = x.shape
    pad = torch.zeros(M, _blocks(K) * BLOCK, device=x.device)
    pad[:, :K] = x
    pad = pad.view(M, -1, BLOCK)
    f, e = torch.frexp(pad.abs().amax(-1))
    e = torch.where(f <= 0.875, e - 9, e - 8)  # 448 = 0.875 * 2^9
    e = torch.where(f == 0, E_MIN, e).clamp(E_MIN, E_MAX).float()
    codes = (pad * torch.exp2(-e)[..., None]).clamp(-448, 448).to(E4M3)
    return codes.view(M, -1)[:, :K].contiguous(), torch.exp2(e)


def _values(codes, scales):
    return codes.float() * scales.repeat_interleave(BLOCK, 1)[:, :codes.shape[1]]


def _matrix(codes, scales):
    return codes.float() * scales.repeat_interleave(BLOCK, 0)[:codes.shape[0]].repeat_interleave(BLOCK, 1)[:, :codes.shape[1]]


def _route(s):
    """Experts and weights of every token; the comparisons are made in 64 bits."""
    l, E, k, n = s["logits"].double(), s["E"], s["k"], s["groups"]
    score = 1.0 / (1.0 + torch.exp(-l)) if s["score"] == "sigmoid" else _softmax(l)
    choice = score if s["b"] is None else score + s["b"].double()
    if n > 1:
        per = choice.view(-1, n, E // n)
        value = torch.sort(per, dim=-1, descending=True)[0][..., :s["group_top"]].sum(-1)
        best = torch.sort(value, dim=-1, descending=True, stable=True)[1][:, :s["top_groups"]]
        keep = torch.zeros_like(value, dtype=torch.bool).scatter_(1, best, True)
        choice = per.masked_fill(~keep[..., None], -math.inf).reshape(-1, E)
    idx = torch.sort(choice, dim=-1, descending=True, stable=True)[1][:, :k]
    w = torch.gather(score, 1, idx)
    if s["renorm"]:
        w = w / (w.sum(-1, keepdim=True) + 1e-20)
    return idx.int(), (w * s["scale"]).float()


def _softmax(l):
    p = torch.exp(l - l.amax(-1, keepdim=True))
    return p / p.sum(-1, keepdim=True)


def _ffn(x, gate, up, down):
    g, u = x @ _matrix(*gate).T, x @ _matrix(*up).T
    g, u = g.clamp(max=10.0), u.clamp(-10.0, 10.0)
    a = g / (1.0 + torch.exp(-g)) * u
    return _values(*_quant(a)) @ _matrix(*down).T


def _moe(s):
    idx, w = _route(s)
    x = _values(*_quant(s["X"]))
    rows = torch.zeros(s["T"], s["k"], s["H"], device=x.device)
    for e in idx.unique().tolist():
        t, slot = torch.nonzero(idx == e, as_tuple=True)
        rows[t, slot] = _ffn(x[t], *[(c[e], d[e]) for c, d in s["experts"]])
    out = (rows * w[..., None]).sum(1)
    if s["one"]:
        out += _ffn(x, *s["one"])
    return out.bfloat16()


# ---- what a pass cannot do without --------------------------------------------------------------

def work(case):
    op, es = case["op"], DT[case["x"]].itemsize
    if op == "quant":
        M, K = case["M"], case["K"]
        return {"bytes": M * K * (es + 1) + M * _blocks(K) * 4, "flops": 4 * M * K}
    if op == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": N * K + _blocks(N) * _blocks(K) * 4 + M * K * es + M * N * DT[case["y"]].itemsize, "flops": 2 * M * N * K}
    T, E, k = case["T"], case["E"], case["k"]
    if op == "route":
        return {"bytes": T * E * es + 8 * T * k + (4 * E if case["bias"] else 0), "flops": 8 * T * E}
    H, I = case["H"], case["I"]
    hit = E * (1.0 - (1.0 - k / E) ** T)  # experts that some token chooses, on the average
    one = 1 if case["shared"] else 0
    return {"bytes": int((hit + one) * 3 * (H * I + (H // BLOCK) * (I // BLOCK) * 4)) + T * H * (es + 2) + T * E * 4,
            "flops": 6 * T * (k + one) * H * I}


# ---- the definition in 64 bits --------------------------------------------------------------------

def _code64(x):
    """x rounded to a value of e4m3, ties to even: three bits behind the leading one, steps of 2^-9 at least."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)


def _quant64(x):
    """Codes and scales of every 128 columns in turn."""
    codes, scales = torch.empty_like(x), []
    for i in range(0, x.shape[1], BLOCK):
        part = x[:, i:i + BLOCK]
        d = torch.exp2(torch.ceil(torch.log2(part.abs().max(1, keepdim=True)[0] / 448)).clamp(E_MIN, E_MAX))
        codes[:, i:i + BLOCK] = _code64(part / d)
        scales.append(d)
    return codes, torch.cat(scales, 1)


def _product64(x, w):
    """x [M, K] (codes and scales) times the matrix w, block column by block column."""
    (xc, xs), (wc, ws) = x, w
    out = torch.zeros(xc.shape[0], wc.shape[0], dtype=torch.float64, device=xc.device)
    rows = torch.arange(wc.shape[0], device=xc.device) // BLOCK
    for b in range(xs.shape[1]):
        at = slice(b * BLOCK, (b + 1) * BLOCK)
        out += (xc[:, at] @ wc[:, at].double().T) * xs[:, b, None] * ws[:, b].double()[rows]
    return out


def _route64(s):
    l, E, n = s["logits"].double().cpu(), s["E"], s["groups"]
    score = torch.sigmoid(l) if s["score"] == "sigmoid" else torch.exp(l - torch.logsumexp(l, 1, keepdim=True))
    choice = score.clone() if s["b"] is None else score + s["b"].double().cpu()
    T, ar = l.shape[0], torch.arange(l.shape[0])
    if n > 1:
        left, value = choice.view(T, n, -1).clone(), torch.zeros(T, n, dtype=torch.float64)
        for _ in range(min(s["group_top"], E // n)):
            top, at = left.max(-1)
            value += top
            left.scatter_(2, at[..., None], -math.inf)
        allowed = torch.zeros(T, n, dtype=torch.bool)
        for _ in range(s["top_groups"]):
            best = (value == value.max(1, keepdim=True)[0]).int().argmax(1)
            allowed[ar, best] = True
            value[ar, best] = -math.inf
        choice[~allowed.repeat_interleave(E // n, 1)] = -math.inf
    idx = torch.empty(T, s["k"], dtype=torch.int32)
    for j in range(s["k"]):
        best = (choice == choice.max(1, keepdim=True)[0]).int().argmax(1)
        idx[:, j] = best
        choice[ar, best] = -math.inf
    w = score.gather(1, idx.long())
    if s["renorm"]:
        w = w / w.sum(1, keepdim=True)
    return idx.to(s["logits"].device), (w * s["scale"]).to(s["logits"].device)


def exact(case, seed):
    op = case["op"]
    if op == "moe" and work(case)["flops"] > 2e14:
        return None
    s = prepare(case, seed)
    if op == "quant":
        return _quant64(s["X"].double())
    if op == "linear":
        return _product64(_quant64(s["X"].double()), s["W"])
    idx, w = _route64(s)
    if op == "route":
        return idx, w

    def layer(rows, gate, up, down):
        g, u = _product64(rows, gate).clamp(max=10.0), _product64(rows, up).clamp(-10.0, 10.0)
        return _product64(_quant64(g * torch.sigmoid(g) * u), down)

    codes, scales = _quant64(s["X"].double())
    out = layer((codes, scales), *s["one"]) if s["one"] else torch.zeros_like(codes)
    for t in range(s["E"]):
        hit = idx == t
        of = hit.any(1).nonzero()[:, 0]
        if of.numel():
            y = layer((codes[of], scales[of]), *[(c[t], d[t]) for c, d in s["experts"]])
            out[of] += y * (w * hit).sum(1)[of, None]
    return out
