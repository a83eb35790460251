"""Cases for the routing and 8-bit operators: their inputs, their plain form in elementary torch operations, the calls
a user makes of this package for the same work, and what their definitions give in 64 bits.

Operators: routing to experts from logits (exl3_router.LogitsRouter), rows quantised to e4m3 with one scale per 128
columns (exl3_fp8.quantize_rows), the linear layer over e4m3 weights with one scale per 128 x 128 block
(exl3_fp8.fp8_linear), and the routed experts stored that way (exl3_fp8.fp8_prefill).
"""
import math
import os
import sys
import types

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "glm53-exl3-prefill_b200")
_DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
BLOCK = 128
E4M3_MAX = 448.0
AMAX_MIN = 2.0 ** -64        # the block maximum a scale is made from is at least this
LIMIT = 7.0                  # SwiGLU clamp


def _use_package():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)


# ------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one token of a decode step through the GLM-5.3-Flash router: latency only
        {"name": "route_decode", "op": "route", "T": 1, "E": 288, "k": 8, "scoring": "sigmoid", "bias": True,
         "groups": 1, "keep": 1, "norm": True, "dtype": "fp32"},
        # a batch of 997 tokens with softmax gates over an expert count that is no multiple of 32
        {"name": "route_softmax_odd", "op": "route", "T": 997, "E": 90, "k": 6, "scoring": "softmax", "bias": False,
         "groups": 1, "keep": 1, "norm": False, "dtype": "bf16"},
        # a prefill chunk of 8192 tokens through the GLM-5.3-Flash router
        {"name": "route_prefill", "op": "route", "T": 8192, "E": 288, "k": 8, "scoring": "sigmoid", "bias": True,
         "groups": 1, "keep": 1, "norm": True, "dtype": "fp32"},
        # the largest chunk (32768 tokens), experts in 8 groups of which 4 are kept
        {"name": "route_groups", "op": "route", "T": 32768, "E": 256, "k": 8, "scoring": "sigmoid", "bias": True,
         "groups": 8, "keep": 4, "norm": True, "dtype": "fp32"},
        # the rows of a small batch before an 8-bit product: latency
        {"name": "quantize_small", "op": "quantize", "T": 33, "K": 4096, "dtype": "bf16", "pow2": False},
        # a prefill chunk at the dense MLP's intermediate width
        {"name": "quantize_prefill", "op": "quantize", "T": 8192, "K": 12288, "dtype": "fp16", "pow2": True},
        # one token through a square projection: the weights' bytes and latency
        {"name": "linear_decode", "op": "linear", "T": 1, "N": 4096, "K": 4096, "dtype": "bf16"},
        # a ragged chunk through a projection whose width is no multiple of 128
        {"name": "linear_ragged", "op": "linear", "T": 777, "N": 576, "K": 4096, "dtype": "fp16"},
        # a prefill chunk through one matrix of the dense MLP
        {"name": "linear_prefill", "op": "linear", "T": 8192, "N": 12288, "K": 4096, "dtype": "bf16"},
        # one token through the routed experts: the bytes of eight experts
        {"name": "experts_decode", "op": "experts", "T": 1, "E": 288, "d": 4096, "f": 1536, "k": 8, "dtype": "bf16"},
        # the small configuration: 16 experts, 64 rows each
        {"name": "experts_small", "op": "experts", "T": 256, "E": 16, "d": 1024, "f": 512, "k": 4, "dtype": "fp16"},
        # the full layer on a prefill chunk
        {"name": "experts_prefill", "op": "experts", "T": 8192, "E": 288, "d": 4096, "f": 1536, "k": 8, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["route", "route", "quantize", "linear", "linear", "experts", "experts"])
    dt = rng.choice(["bf16", "fp16"])
    if op == "route":
        groups = rng.choice([1, 1, 4, 8])
        E = groups * _log(rng, 8, 512 // groups)
        keep = rng.randint(max(1, groups // 2), groups)
        k = rng.randint(1, min(16, keep * (E // groups)))
        return {"op": op, "T": _log(rng, 1, min(32768, 32768 * 256 // E)), "E": E, "k": k, "scoring": rng.choice(["sigmoid", "softmax"]),
                "bias": rng.random() < 0.5, "groups": groups, "keep": keep, "norm": rng.random() < 0.7,
                "dtype": rng.choice(["fp32", "bf16", "fp16"])}
    if op == "quantize":
        K = 16 * _log(rng, 8, 768)
        return {"op": op, "T": _log(rng, 1, 8192), "K": K, "dtype": rng.choice(["fp32", "bf16", "fp16"]) if K < 6144 else dt,
                "pow2": rng.random() < 0.5}
    if op == "linear":
        T, K, N = _log(rng, 1, 8192), 16 * _log(rng, 8, 768), _log(rng, 64, 12288)
        while T * N * K > 8192 * 12288 * 4096 or T * (N + K) > 8192 * 16384:
            T = (T + 1) // 2
        return {"op": op, "T": T, "N": N, "K": K, "dtype": dt}
    E, d, f = _log(rng, 4, 288), 128 * _log(rng, 4, 32), 128 * _log(rng, 2, 12)
    return {"op": op, "T": _log(rng, 1, 8192), "E": E, "d": d, "f": f, "k": rng.randint(1, min(8, E)), "dtype": dt}


def work(case):
    c = case
    b = 4 if c["dtype"] == "fp32" else 2
    if c["op"] == "route":
        return {"bytes": c["T"] * c["E"] * b + (4 * c["E"] if c["bias"] else 0) + c["T"] * c["k"] * 12,
                "flops": c["T"] * c["E"] * 8}
    if c["op"] == "quantize":
        nb = -(-c["K"] // BLOCK)
        return {"bytes": c["T"] * (c["K"] * (b + 1) + 4 * nb), "flops": c["T"] * c["K"] * 3}
    if c["op"] == "linear":
        T, N, K = c["T"], c["N"], c["K"]
        return {"bytes": T * K * b + N * K + 4 * -(-N // BLOCK) * -(-K // BLOCK) + T * N * b, "flops": 2 * T * N * K}
    T, E, d, f, k = c["T"], c["E"], c["d"], c["f"], c["k"]
    touched = E * (1 - (1 - k / E) ** T)                       # experts that some token chose, on average
    return {"bytes": touched * 3 * d * f * (1 + 4 / BLOCK ** 2) + 2 * T * d * b + T * k * 12, "flops": 6 * T * k * d * f}


# ------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _weights(g, E, n, k):
    """e4m3 [E, n, k] as a block quantiser leaves normal weights (block maximum at 448, about four standard
    deviations), and its scales [E, n / 128, k / 128], for rows of unit variance to stay so."""
    q = torch.empty(E, n, k, dtype=torch.float8_e4m3fn, device="cuda")
    step = max(1, (1 << 27) // (n * k))
    for e in range(0, E, step):
        w = torch.randn(min(step, E - e), n, k, generator=g, device="cuda")
        q[e:e + step] = w.mul_(E4M3_MAX / 4.2).clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    s = (0.75 + 0.5 * torch.rand(E, nb, kb, generator=g, device="cuda")) * (4.2 / E4M3_MAX / math.sqrt(k))
    return q, s


def _rows(g, T, K, dtype):
    """Hidden states: normal, with a few channels that are much larger than the rest."""
    loud = 1 + 15 * (torch.rand(K, generator=g, device="cuda") < 0.01).float()
    return (torch.randn(T, K, generator=g, device="cuda") * loud).to(_DT[dtype])


def _routes(g, T, E, k):
    """Each token's k experts and its weights, from scores that favour some experts over others."""
    scores = torch.randn(T, E, generator=g, device="cuda") + 0.3 * torch.randn(E, generator=g, device="cuda")
    v, ids = torch.topk(scores, k, dim=-1)
    return ids, torch.softmax(v, dim=-1)


def prepare(case, seed):
    c, g = case, _gen(seed)
    s = types.SimpleNamespace(**{k: v for k, v in c.items() if k != "name"})
    if s.op == "route":
        s.logits = (1.5 * torch.randn(s.T, s.E, generator=g, device="cuda")).to(_DT[s.dtype])
        s.b = 0.1 * torch.randn(s.E, generator=g, device="cuda") if s.bias else None
        s.group_top = 2 if s.scoring == "sigmoid" else 1
        s.scale = 2.5
        if own:
            _use_package()
            import exl3_router
            s.router = exl3_router.LogitsRouter(s.k, scoring=s.scoring, bias=s.b, n_group=s.groups, topk_group=s.keep,
                                                group_top=s.group_top, norm=s.norm, scale=s.scale)
    elif s.op == "quantize":
        s.x = _rows(g, s.T, s.K, s.dtype)
    elif s.op == "linear":
        s.x = _rows(g, s.T, s.K, s.dtype)
        w, ws = _weights(g, 1, s.N, s.K)
        s.w, s.ws = w[0], ws[0]
    else:
        s.x = _rows(g, s.T, s.d, s.dtype)
        s.ids, s.rw = _routes(g, s.T, s.E, s.k)
        s.layer = types.SimpleNamespace(_exl3_intermediate_local=s.f)
        s.layer.w13_fp8, s.layer.w13_scale = _weights(g, s.E, 2 * s.f, s.d)
        s.layer.w2_fp8, s.layer.w2_scale = _weights(g, s.E, s.d, s.f)
    return s


# ------------------------------------------------------------------------------------------ plain forms
def _route_plain(s):
    x = s.logits.double()                   # ranks go by values next to one another: 64 bits
    masked = ~(x > -math.inf)               # -inf and NaN
    score = torch.sigmoid(x) if s.scoring == "sigmoid" else torch.softmax(x.masked_fill(masked, -math.inf), dim=-1)
    pick = (score if s.b is None else score + s.b.double()).masked_fill(masked, -math.inf)
    if s.keep < s.groups:
        by = pick.view(s.T, s.groups, -1)
        top = by.sort(dim=-1, descending=True, stable=True).values[..., :s.group_top]
        kept = top.sum(-1).sort(dim=-1, descending=True, stable=True).indices[:, :s.keep]
        keep = torch.zeros(s.T, s.groups, dtype=torch.bool, device=x.device).scatter_(1, kept, True)
        pick = by.masked_fill(~keep[..., None], -math.inf).view(s.T, s.E)
    v, ids = pick.sort(dim=-1, descending=True, stable=True)
    v, ids = v[:, :s.k], ids[:, :s.k]
    w = score.gather(1, ids).masked_fill(v == -math.inf, 0.0)
    if s.norm:
        w = w / (w.sum(-1, keepdim=True) + 1e-20)
    return ids.masked_fill(v == -math.inf, -1), (w * s.scale).float()


def _to_e4m3(v):
    """Nearest e4m3 of double values within +-448, as doubles (ties to even): the step is 2^(e-3), e >= -6."""
    e = torch.frexp(v.abs()).exponent.clamp_(min=-5) - 4
    step = torch.ldexp(torch.ones_like(v), e)
    return torch.round(v / step) * step


def _quantize_plain(x, pow2=False):
    """(values in e4m3 as fp32 [T, K], scales fp32 [T, K / 128]); the borders between values in 64 bits."""
    T, K = x.shape
    nb = -(-K // BLOCK)
    xb = torch.nn.functional.pad(x.float(), (0, nb * BLOCK - K)).view(T, nb, BLOCK)
    amax = xb.abs().amax(-1).clamp(min=AMAX_MIN)
    if pow2:
        m, e = torch.frexp(amax)                            # amax = m 2^e, 0.5 <= m < 1; 448 = 0.875 * 2^9
        s = torch.ldexp(torch.ones_like(amax), torch.where(m <= 0.875, e - 9, e - 8))
    else:
        s = (amax.double() / torch.full_like(amax, E4M3_MAX, dtype=torch.float64)).float()   # one rounding: a
        # scalar divisor would be taken as a product with its rounded reciprocal
    q = _to_e4m3(xb.double() / s.double()[..., None])
    return q.float().view(T, nb * BLOCK)[:, :K], s


def _spread(s, n, k):
    """Scales [..., n / 128, k / 128] spread over [..., n, k]."""
    return s.repeat_interleave(BLOCK, -2)[..., :n, :].repeat_interleave(BLOCK, -1)[..., :k]


def _rows_plain(x):
    q, s = _quantize_plain(x)
    return q * s.repeat_interleave(BLOCK, -1)[:, :x.shape[1]]


def _act(gu, f):
    g, u = gu[..., :f].clamp(max=LIMIT), gu[..., f:].clamp(-LIMIT, LIMIT)
    return g / (1 + torch.exp(-g)) * u


def _experts_plain(s):
    T, k, d, f = s.T, s.k, s.d, s.f
    flat = s.ids.reshape(-1)
    active, pos, counts = torch.unique(flat, return_inverse=True, return_counts=True)
    order = torch.argsort(pos, stable=True)                              # routed slots by expert
    row = torch.arange(T * k, device=flat.device) - (counts.cumsum(0) - counts)[pos[order]]
    at = pos[order] * int(counts.max()) + row                            # each slot's row in [experts, most, d]
    L = s.layer
    w13 = L.w13_fp8[active].float().mul_(_spread(L.w13_scale[active], 2 * f, d))
    w2 = L.w2_fp8[active].float().mul_(_spread(L.w2_scale[active], d, f))
    x = _rows_plain(s.x)
    xe = torch.zeros(active.numel() * int(counts.max()), d, device=x.device)
    xe[at] = x[order // k]
    a = _act(torch.bmm(xe.view(active.numel(), -1, d), w13.transpose(1, 2)), f)
    a = _rows_plain(a.view(-1, f)).view(a.shape)
    y = torch.bmm(a, w2.transpose(1, 2)).view(-1, d)
    slots = torch.empty(T * k, d, device=x.device)
    slots[order] = y[at]
    return (slots.view(T, k, d) * s.rw[..., None]).sum(1).to(s.x.dtype)


def run(state):
    s = state
    if own:
        if s.op == "route":
            return s.router.route(s.logits)
        _use_package()
        import exl3_fp8
        if s.op == "quantize":
            return exl3_fp8.quantize_rows(s.x, pow2=s.pow2)
        if s.op == "linear":
            return exl3_fp8.fp8_linear(s.x, s.w, s.ws, out_dtype=s.x.dtype)
        return exl3_fp8.fp8_prefill(s.x, s.ids, s.rw, s.layer, LIMIT, out_dtype=s.x.dtype)
    if s.op == "route":
        return _route_plain(s)
    if s.op == "quantize":
        q, scale = _quantize_plain(s.x, s.pow2)
        return q.to(torch.float8_e4m3fn), scale
    if s.op == "linear":
        w = s.w.float() * _spread(s.ws, s.N, s.K)
        return (_rows_plain(s.x) @ w.t()).to(s.x.dtype)
    return _experts_plain(s)


# ------------------------------------------------------------------------------------------ 64 bits
def _exact_quantize(x, pow2=False):
    """Values and scales in 64 bits (a scale is a 32-bit number by definition, so it is rounded to one)."""
    T, K = x.shape
    q, scales = torch.empty(T, K, dtype=torch.float64, device=x.device), []
    for k0 in range(0, K, BLOCK):
        xb = x[:, k0:k0 + BLOCK].double()
        s = xb.abs().max(dim=1, keepdim=True).values.clamp(min=AMAX_MIN)
        if pow2:                                            # the least power of two with 448 s >= the maximum
            amax, s = s, torch.ldexp(torch.ones_like(s), torch.floor(torch.log2(s)).int() - 10)
            for _ in range(3):
                s = torch.where(s * E4M3_MAX < amax, 2 * s, s)
        else:
            s = (s / torch.full_like(s, E4M3_MAX)).float().double()
        v = xb / s
        unit = torch.ldexp(torch.ones_like(v), torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))).int() - 3)
        q[:, k0:k0 + BLOCK] = torch.round(v / unit) * unit
        scales.append(s)
    return q, torch.cat(scales, 1)


def _exact_rows(x):
    q, s = _exact_quantize(x)
    for b in range(s.shape[1]):
        q[:, b * BLOCK:(b + 1) * BLOCK] *= s[:, b:b + 1]
    return q


def _exact_weight(q, s):
    w = q.float().double()
    for b in range(s.shape[0]):
        w[b * BLOCK:(b + 1) * BLOCK] *= s[b].double().repeat_interleave(BLOCK)[:w.shape[1]]
    return w


def _exact_route(s):
    l = s.logits.double()
    p = 1 / (1 + torch.exp(-l)) if s.scoring == "sigmoid" else torch.exp(l - torch.logsumexp(l, -1, keepdim=True))
    c = p + (s.b.double() if s.b is not None else 0)
    if s.groups > 1:
        per = s.E // s.groups
        gs = torch.stack([c[:, i * per:(i + 1) * per].topk(min(s.group_top, per), dim=1).values.sum(1) for i in range(s.groups)], 1)
        bar = gs.topk(s.keep, dim=1).values[:, -1:]
        c = torch.where((gs >= bar).repeat_interleave(per, 1), c, torch.full_like(c, -math.inf))
    ids, left = [], c.clone()
    for _ in range(s.k):
        best = (left == left.max(1, keepdim=True).values).int().argmax(1, keepdim=True)     # the first of equals
        left.scatter_(1, best, -math.inf)
        ids.append(best)
    ids = torch.cat(ids, 1)
    w = p.gather(1, ids)
    return ids, w / (w.sum(1, keepdim=True) + 1e-20) * s.scale if s.norm else w * s.scale


def exact(case, seed):
    global own
    was, own = own, False
    s = prepare(case, seed)
    own = was
    if s.op == "route":
        return _exact_route(s)
    if s.op == "quantize":
        return _exact_quantize(s.x, s.pow2)
    if s.op == "linear":
        return _exact_rows(s.x) @ _exact_weight(s.w, s.ws).t()
    L, f = s.layer, s.f
    x, out = _exact_rows(s.x), torch.zeros(s.T, s.d, dtype=torch.float64, device=s.x.device)
    for e in torch.unique(s.ids).tolist():
        t, j = (s.ids == e).nonzero(as_tuple=True)
        gu = x[t] @ _exact_weight(L.w13_fp8[e], L.w13_scale[e]).t()
        g, u = gu[:, :f].clamp(max=LIMIT), gu[:, f:].clamp(-LIMIT, LIMIT)
        a = _exact_rows(g * torch.sigmoid(g) * u)
        out.index_add_(0, t, (a @ _exact_weight(L.w2_fp8[e], L.w2_scale[e]).t()) * s.rw[t, j].double()[:, None])
    return out
