"""The block-scaled 8-bit floating point operators, as cases to be timed.

A serving engine that holds its weights in e4m3 with one f32 scale per
128 x 128 block calls four operators in a layer:

  quantize  activations to e4m3 with one scale per row and 128 columns
            (ffi.quantize_fp8): once for the projections that share an input
  matmul    dense projections (ffi.matmul_fp8): decode, batched decode, prompt
            chunks and whole prompts, on bf16 / f32 activations quantized within
            the call or on e4m3 activations quantized before
  route     grouped routing (ffi.moe_route_group): scores, a selection-only
            bias, groups, top-k, renormalised weights
  moe       the routed experts (ffi.moe_ffn_fp8): decode, batched decode, prompts

`run` in its plain form computes them with elementary torch operations in f32;
the roundings to 8 bits and the router's comparisons, where a last bit decides,
in f64.  `exact` is the definition in f64.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
BLOCK = 128          # columns of one activation scale, rows and columns of one weight scale
E4M3_MAX = 448.0
MIN_SCALE = 2.0 ** -126
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ------------------------------------------------------------------ the cases

def _quantize(name, m, k, x):
    return {"name": name, "kind": "quantize", "m": m, "k": k, "x": x}


def _matmul(name, m, k, n, x="bf16", out="bf16", epilogue="none"):
    return {"name": name, "kind": "matmul", "m": m, "k": k, "n": n, "x": x, "out": out, "epilogue": epilogue}


def _route(name, t, e, groups, topk_group, k, scoring="sigmoid", group_score="top2", bias=True):
    return {"name": name, "kind": "route", "t": t, "e": e, "groups": groups, "topk_group": topk_group, "k": k,
            "scoring": scoring, "group_score": group_score, "bias": bias}


def _moe(name, t, e, k, dm, dff, shared=0, out="bf16"):
    return {"name": name, "kind": "moe", "t": t, "e": e, "k": k, "dm": dm, "dff": dff, "shared": shared, "out": out}


def listed():
    return [
        # one decode step of 5 rows (a token and its drafts): the input that q, k and v share
        _quantize("quantize_m5", 5, 2048, "bf16"),
        # a whole prompt's hidden states
        _quantize("quantize_m8192", 8192, 4096, "bf16"),
        # a single token through a square projection
        _matmul("matmul_m1_f32", 1, 4096, 4096, x="f32", out="f32"),
        # a step of drafted tokens through a wide projection, quantized once for several projections
        _matmul("matmul_m5_q", 5, 2048, 5120, x="e4m3"),
        # concurrent sequences through a gated pair
        _matmul("matmul_m48_gated", 48, 2048, 1408, epilogue="swiglu"),
        # a prompt chunk, odd rows, into a width that is no multiple of a block, back onto the residual stream
        _matmul("matmul_m517_residual", 517, 4096, 2112, out="f32", epilogue="residual"),
        # a whole prompt through the largest projection
        _matmul("matmul_m2048", 2048, 4096, 14336),
        # the router of one decode step
        _route("route_t5", 5, 256, 8, 4, 8),
        # the router of a prompt: softmax scores, groups by their best expert
        _route("route_t8192", 8192, 512, 8, 3, 10, scoring="softmax", group_score="max", bias=False),
        # the experts of one decode step, with a shared expert
        _moe("moe_t5", 5, 512, 10, 2048, 512, shared=1),
        # the experts of concurrent sequences
        _moe("moe_t48", 48, 64, 6, 2048, 1408),
        # the experts of a whole prompt
        _moe("moe_t8192", 8192, 512, 10, 2048, 512),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("quantize", "matmul", "matmul", "route", "moe"))
    if kind == "quantize":
        k = 16 * _log(rng, 8, 512)
        return {"kind": kind, "m": _log(rng, 1, min(8192, (1 << 25) // k)), "k": k, "x": rng.choice(("bf16", "f32"))}
    if kind == "matmul":
        k, n = 16 * _log(rng, 16, 512), _log(rng, 64, 14336)
        epilogue = rng.choice(("none", "bias", "residual", "swiglu"))
        most = (2048 * 4096 * 14336) // (k * n * (2 if epilogue == "swiglu" else 1))
        return {"kind": kind, "m": _log(rng, 1, min(4096, most)), "k": k, "n": n, "x": rng.choice(("bf16", "f32", "e4m3")),
                "out": rng.choice(("bf16", "f32")), "epilogue": epilogue}
    if kind == "route":
        groups = rng.choice((1, 2, 4, 8, 16))
        per = rng.randint(2, 1024 // groups if groups > 2 else 256)
        topk_group = rng.randint(1, groups)
        e = groups * per
        return {"kind": kind, "t": _log(rng, 1, min(8192, (1 << 22) // e)), "e": e, "groups": groups, "topk_group": topk_group,
                "k": rng.randint(1, min(16, topk_group * per)), "scoring": rng.choice(("softmax", "sigmoid")),
                "group_score": rng.choice(("max", "top2")), "bias": rng.random() < 0.6}
    dm, dff, e, shared = 128 * rng.randint(2, 32), 128 * _log(rng, 2, 16), _log(rng, 8, 512), rng.choice((0, 0, 1))
    while (e + shared) * dm * dff > 512 * 2048 * 512:
        e = max(8, e // 2)
        dff = max(128, 128 * (dff // 256))
    k = rng.randint(1, min(10, e))
    most = (8192 * 10 * 2048 * 512) // ((k + shared) * dm * dff)
    return {"kind": kind, "t": _log(rng, 1, min(8192, most)), "e": e, "k": k, "dm": dm, "dff": dff, "shared": shared,
            "out": "bf16"}


# ------------------------------------------------------------------ inputs

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _activations(m, k, g):
    """N(0, 1) with a few columns twenty times as large, as hidden states have them."""
    x = torch.randn(m, k, generator=g, device=DEV)
    x *= torch.where(torch.rand(k, generator=g, device=DEV) < 0.004, 20.0, 1.0)
    return x


def _weights(rows, k, g):
    """e4m3 weights [rows, k] of standard deviation 0.03 and their f32 scales, one
    per 128 x 128 block, as a checkpoint holds them."""
    nb, kb = -(-rows // BLOCK), -(-k // BLOCK)
    w = torch.randn(nb * BLOCK, kb * BLOCK, generator=g, device=DEV)
    scale = 0.03 * torch.exp(0.3 * torch.randn(nb, kb, generator=g, device=DEV))  # blocks differ in their spread
    blocks = w.view(nb, BLOCK, kb, BLOCK)
    amax = blocks.abs().amax(dim=(1, 3))
    blocks *= (E4M3_MAX / amax)[:, None, :, None]
    codes = w[:rows, :k].clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return codes.contiguous(), (scale * amax / E4M3_MAX).contiguous()


def prepare(case, seed):
    g = _gen(seed)
    kind = case["kind"]
    state = dict(case)
    if kind == "quantize":
        state["data"] = _activations(case["m"], case["k"], g).to(DTYPES[case["x"]])
        return state
    if kind == "matmul":
        m, k, n = case["m"], case["k"], case["n"]
        x = _activations(m, k, g)
        if case["x"] == "e4m3":
            q, s = _quantize_plain(x.to(torch.bfloat16))
            state["data"], state["x_scales"] = q.to(torch.float8_e4m3fn), s
        else:
            state["data"], state["x_scales"] = x.to(DTYPES[case["x"]]), None
        if case["epilogue"] == "swiglu":
            gate, gate_s = _weights(n, k, g)
            up, up_s = _weights(n, k, g)
            state["w"], state["w_scales"] = torch.cat((gate, up)), torch.cat((gate_s, up_s))
        else:
            state["w"], state["w_scales"] = _weights(n, k, g)
        state["bias_v"] = torch.randn(n, generator=g, device=DEV) if case["epilogue"] == "bias" else None
        state["residual_v"] = torch.randn(m, n, generator=g, device=DEV) if case["epilogue"] == "residual" else None
        return state
    if kind == "route":
        t, e = case["t"], case["e"]
        # experts differ in popularity; the bias leans against it
        lean = 0.7 * torch.randn(e, generator=g, device=DEV)
        state["logits"] = torch.randn(t, e, generator=g, device=DEV) + lean
        state["bias_v"] = -0.1 * lean + 0.02 * torch.randn(e, generator=g, device=DEV) if case["bias"] else None
        return state
    t, e, k, dm, dff, shared = (case[i] for i in ("t", "e", "k", "dm", "dff", "shared"))
    state["data"] = _activations(t, dm, g).to(torch.bfloat16)
    logits = torch.randn(t, e, generator=g, device=DEV) + 0.5 * torch.randn(e, generator=g, device=DEV)
    p, ids = torch.topk(torch.softmax(logits, 1), k, dim=1)
    state["ids"], state["weights"] = ids.to(torch.int32), p / p.sum(1, keepdim=True)
    gu, gu_s = _weights((e + shared) * 2 * dff, dm, g)
    dn, dn_s = _weights((e + shared) * dm, dff, g)
    state["gate_up"], state["gate_up_s"] = gu.view(e + shared, 2 * dff, dm), gu_s.view(e + shared, 2 * dff // BLOCK, dm // BLOCK)
    state["down"], state["down_s"] = dn.view(e + shared, dm, dff), dn_s.view(e + shared, dm // BLOCK, dff // BLOCK)
    # the plain form's rows per expert: room for the busiest one
    state["room"] = int(torch.bincount(ids.flatten(), minlength=e).max())
    return state


# ------------------------------------------------------------------ the plain form

def _blocks(x):
    """[m, k] -> [m, kb, 128], zeros behind the last column."""
    m, k = x.shape
    return torch.nn.functional.pad(x, (0, -k % BLOCK)).view(m, -1, BLOCK)


def _quantize_plain(x):
    """(values of the codes, f32 [m, k]; f32 scales [m, kb])."""
    k = x.shape[1]
    b = _blocks(x.float())
    amax = b.abs().amax(2).double()
    s = torch.clamp((amax / torch.full_like(amax, E4M3_MAX)).float(), min=MIN_SCALE)  # a quotient, not a reciprocal's product
    v = b.double() / s.double()[:, :, None]
    exponent = torch.clamp(torch.frexp(v).exponent - 1, min=-6)
    step = ((exponent.long() + (1023 - 3)) << 52).view(torch.float64)  # 2^(exponent - 3): three fraction bits
    q = torch.round(v / step) * step                      # half to even
    return q.float().flatten(1)[:, :k].contiguous(), s


def _spread_rows(s, rows):
    """A scale for each 128 rows, to each row."""
    return s.repeat_interleave(BLOCK, dim=-2)[..., :rows, :]


def _times(q, s):
    """Codes' values and their scales per 128 columns, multiplied."""
    k = q.shape[-1]
    return q.float() * s.repeat_interleave(BLOCK, dim=-1)[..., :k]


def _matmul_plain(st):
    x, n = st["data"], st["n"]
    q, s = (x, st["x_scales"]) if st["x"] == "e4m3" else _quantize_plain(x)
    a = _times(q, s)
    w, ws = st["w"], st["w_scales"]
    half = ws.shape[0] // 2
    if st["epilogue"] == "swiglu":
        gate = a @ _times(w[:n], _spread_rows(ws[:half], n)).T
        up = a @ _times(w[n:], _spread_rows(ws[half:], n)).T
        y = gate / (1.0 + torch.exp(-gate)) * up
    else:
        y = a @ _times(w, _spread_rows(ws, n)).T
        if st["epilogue"] == "bias":
            y = y + st["bias_v"]
        if st["epilogue"] == "residual":
            y = y + st["residual_v"]
    return y.to(DTYPES[st["out"]])


def _largest(c, n):
    """Indices of each row's n largest, descending, ties to the lower index."""
    return torch.sort(c, dim=1, descending=True, stable=True).indices[:, :n]


def _route_plain(st):
    logits = st["logits"].double()
    t, e = logits.shape
    if st["scoring"] == "softmax":
        p = torch.exp(logits - logits.amax(1, keepdim=True))
        p = p / p.sum(1, keepdim=True)
    else:
        p = 1.0 / (1.0 + torch.exp(-logits))
    c = p + st["bias_v"].double() if st["bias"] else p
    per_group = torch.sort(c.view(t, st["groups"], -1), dim=2, descending=True).values
    score = per_group[:, :, :2 if st["group_score"] == "top2" else 1].sum(2)
    kept = torch.zeros(t, st["groups"], dtype=torch.bool, device=c.device)
    kept.scatter_(1, _largest(score, st["topk_group"]), True)
    c = torch.where(kept.repeat_interleave(e // st["groups"], dim=1), c, -math.inf)
    ids = _largest(c, st["k"])
    w = p.gather(1, ids)
    w = w / w.sum(1, keepdim=True) * 2.5
    return ids.to(torch.int32), w.float()


def _moe_plain(st):
    t, k, e, dff, dm = st["t"], st["k"], st["e"], st["dff"], st["dm"]
    gate_up = _times(st["gate_up"], _spread_rows(st["gate_up_s"], 2 * dff))
    down = _times(st["down"], _spread_rows(st["down_s"], dm))
    x = _times(*_quantize_plain(st["data"]))

    def ffn(rows, gu, dn):  # [experts, rows, dm] -> the same, each expert's rows through it
        g = torch.bmm(rows, gu.transpose(1, 2).contiguous())
        h = g[:, :, :dff] / (1.0 + torch.exp(-g[:, :, :dff])) * g[:, :, dff:]
        q, s = _quantize_plain(h.reshape(-1, dff))
        return torch.bmm(_times(q, s).view(h.shape), dn.transpose(1, 2).contiguous())

    # each expert's pairs in a row of their own, st["room"] places long
    owner = st["ids"].flatten().long()
    order = torch.argsort(owner, stable=True)
    pair_owner = owner[order]
    counts = torch.zeros(e, dtype=torch.long, device=owner.device).scatter_add_(0, owner, torch.ones_like(owner))
    place = torch.arange(t * k, device=owner.device) - (torch.cumsum(counts, 0) - counts)[pair_owner]
    rows = torch.zeros(e, st["room"], dm, device=owner.device)
    rows[pair_owner, place] = x[order // k]
    o = torch.empty(t * k, dm, device=owner.device)
    o[order] = ffn(rows, gate_up[:e], down[:e])[pair_owner, place]
    y = (o.view(t, k, dm) * st["weights"][:, :, None]).sum(1)
    if st["shared"]:
        y = y + ffn(x.expand(st["shared"], t, dm), gate_up[e:], down[e:]).sum(0)
    return y.to(DTYPES[st["out"]])


def run(state):
    kind = state["kind"]
    if own:
        from r9v_amd import ffi

        if kind == "quantize":
            return ffi.quantize_fp8(state["data"])
        if kind == "matmul":
            return ffi.matmul_fp8(state["w"], state["w_scales"], state["data"], x_scales=state["x_scales"],
                                  out_dtype=ffi.BF16 if state["out"] == "bf16" else ffi.F32, bias=state["bias_v"],
                                  residual=state["residual_v"], swiglu=state["epilogue"] == "swiglu")
        if kind == "route":
            return ffi.moe_route_group(state["logits"], state["k"], state["groups"], state["topk_group"], bias=state["bias_v"],
                                       scoring=ffi.SCORING_SOFTMAX if state["scoring"] == "softmax" else ffi.SCORING_SIGMOID,
                                       group_score=ffi.GROUP_MAX if state["group_score"] == "max" else ffi.GROUP_TOP2, scale=2.5)
        return ffi.moe_ffn_fp8(state["data"], state["ids"], state["weights"], state["gate_up"], state["gate_up_s"],
                               state["down"], state["down_s"], shared=state["shared"],
                               out_dtype=ffi.BF16 if state["out"] == "bf16" else ffi.F32)
    if kind == "quantize":
        q, s = _quantize_plain(state["data"])
        return q.to(torch.float8_e4m3fn), s
    if kind == "matmul":
        return _matmul_plain(state)
    if kind == "route":
        return _route_plain(state)
    return _moe_plain(state)


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    kind = case["kind"]
    if kind == "quantize":
        m, k = case["m"], case["k"]
        return {"bytes": m * k * (2 if case["x"] == "bf16" else 4) + m * k + 4 * m * -(-k // BLOCK), "flops": 3 * m * k}
    if kind == "matmul":
        m, k, n = case["m"], case["k"], case["n"]
        kb, pair = -(-k // BLOCK), 2 if case["epilogue"] == "swiglu" else 1
        x = m * k * {"bf16": 2, "f32": 4, "e4m3": 1}[case["x"]] + (4 * m * kb if case["x"] == "e4m3" else 0)
        more = {"bias": 4 * n, "residual": 4 * m * n}.get(case["epilogue"], 0)
        return {"bytes": pair * (n * k + 4 * -(-n // BLOCK) * kb) + x + m * n * (2 if case["out"] == "bf16" else 4) + more,
                "flops": 2 * pair * m * n * k}
    if kind == "route":
        t, e, k = case["t"], case["e"], case["k"]
        return {"bytes": 4 * t * e + (4 * e if case["bias"] else 0) + 8 * t * k, "flops": 8 * t * e}
    t, e, k, dm, dff, shared = (case[i] for i in ("t", "e", "k", "dm", "dff", "shared"))
    hit = e * (1.0 - (1.0 - k / e) ** t)  # distinct experts that t tokens are expected to name
    expert = 3 * dm * dff + 4 * 3 * (dm // BLOCK) * (dff // BLOCK)
    return {"bytes": int((hit + shared) * expert) + t * dm * (2 + (2 if case["out"] == "bf16" else 4)) + 8 * t * k,
            "flops": 6 * t * (k + shared) * dm * dff}


# ------------------------------------------------------------------ the definition in 64 bits

def _e4m3(v):
    """|v| <= 448 in f64 to the nearest e4m3 value, ties to the even code."""
    values = [math.ldexp(c % 8 + (8 if c >= 8 else 0), max(c // 8, 1) - 10) for c in range(127)]  # 0 .. 448
    values = torch.tensor(values, device=v.device, dtype=torch.float64)
    middles = (values[1:] + values[:-1]) / 2
    a = v.abs()
    low, high = torch.bucketize(a, middles), torch.bucketize(a, middles, right=True)  # they differ on a tie only
    return values[torch.where(low % 2 == 0, low, high)] * torch.sign(v)


def _exact_quantized(x):
    """(codes' values, scales) in f64."""
    m, k = x.shape
    q, scales = torch.empty(m, k, dtype=torch.float64, device=x.device), []
    for b in range(0, k, BLOCK):
        part = x[:, b:b + BLOCK].double()
        amax = part.abs().amax(1)
        s = torch.div(amax, torch.full_like(amax, E4M3_MAX)).float().clamp(min=MIN_SCALE).double()
        q[:, b:b + BLOCK] = _e4m3(part / s[:, None])
        scales.append(s)
    return q, torch.stack(scales, 1)


def _exact_product(q, s, w, ws):
    """sum over 128-column blocks of (s * ws) * (q . w), f64."""
    m, n = q.shape[0], w.shape[0]
    y = torch.zeros(m, n, dtype=torch.float64, device=q.device)
    row = torch.arange(n, device=q.device) // BLOCK
    for b in range(s.shape[1]):
        c = slice(b * BLOCK, (b + 1) * BLOCK)
        y += (q[:, c] @ w[:, c].double().T) * s[:, b, None] * ws.double()[row, b]
    return y


def _exact_ffn(q, s, gate_up, gate_up_s, down, down_s):
    dff = gate_up.shape[0] // 2
    half = gate_up_s.shape[0] // 2
    g = _exact_product(q, s, gate_up[:dff], gate_up_s[:half])
    u = _exact_product(q, s, gate_up[dff:], gate_up_s[half:])
    return _exact_product(*_exact_quantized(torch.sigmoid(g) * g * u), down, down_s)


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "quantize":
        return _exact_quantized(st["data"])
    if kind == "matmul":
        n = case["n"]
        q, s = (st["data"].double(), st["x_scales"].double()) if case["x"] == "e4m3" else _exact_quantized(st["data"])
        w, ws = st["w"], st["w_scales"]
        if case["epilogue"] == "swiglu":
            g = _exact_product(q, s, w[:n], ws[:ws.shape[0] // 2])
            return torch.sigmoid(g) * g * _exact_product(q, s, w[n:], ws[ws.shape[0] // 2:])
        y = _exact_product(q, s, w, ws)
        if case["epilogue"] == "bias":
            y += st["bias_v"].double()
        if case["epilogue"] == "residual":
            y += st["residual_v"].double()
        return y
    if kind == "route":
        l = st["logits"].double()
        p = torch.softmax(l, 1) if case["scoring"] == "softmax" else torch.sigmoid(l)
        c = p + st["bias_v"].double() if case["bias"] else p.clone()
        g = c.view(case["t"], case["groups"], -1)
        first = g.amax(2)
        score = first if case["group_score"] == "max" else torch.topk(g, 2, dim=2).values.sum(2)
        open_, ids = torch.zeros_like(score, dtype=torch.bool), []
        for _ in range(case["topk_group"]):
            best = torch.where(open_, -math.inf, score).argmax(1)  # the first of equals
            open_[torch.arange(case["t"], device=best.device), best] = True
        c[~open_.repeat_interleave(case["e"] // case["groups"], 1)] = -math.inf
        for _ in range(case["k"]):
            best = c.argmax(1)
            ids.append(best)
            c[torch.arange(case["t"], device=best.device), best] = -math.inf
        ids = torch.stack(ids, 1)
        w = p.gather(1, ids)
        return ids.to(torch.int32), 2.5 * w / w.sum(1, keepdim=True)
    q, s = _exact_quantized(st["data"])
    y = torch.zeros(case["t"], case["dm"], dtype=torch.float64, device=DEV)
    for x in range(case["e"]):
        tok, slot = torch.nonzero(st["ids"] == x, as_tuple=True)
        if tok.numel():
            o = _exact_ffn(q[tok], s[tok], st["gate_up"][x], st["gate_up_s"][x], st["down"][x], st["down_s"][x])
            y.index_add_(0, tok, o * st["weights"][tok, slot].double()[:, None])
    for x in range(case["e"], case["e"] + case["shared"]):
        y += _exact_ffn(q, s, st["gate_up"][x], st["gate_up_s"][x], st["down"][x], st["down_s"][x])
    return y
