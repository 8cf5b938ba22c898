"""Performance cases of the operators around attention in a decoder layer.

  qk_norm_rope             RMS norm of every query and key head and the
                           rotation by its token's position, in one pass
  cross_attention          attention to an encoder's states of another length
  shared_prefix_attention  new tokens of many sequences against a prefix that
                           all of them share and each one's own cache

Each case is one call (or one forward and backward step). `run` makes it
through the public API where `own` is true, and in plain torch operations in
32 bits where it is false; `exact` computes it from the definition in 64 bits.
"""

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZES = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # One new token of each of 16 sequences against its encoder's states: a step of a
        # translation or speech decoder, where latency counts.
        {"name": "cross_token", "op": "cross", "dtype": "bf16", "batch": 16, "heads": 32, "kv_heads": 8, "queries": 1,
         "keys": 1500, "d": 128, "lengths": "ragged", "train": False},
        # Scoring given targets with 64-wide heads, every encoder state valid.
        {"name": "cross_score_d64", "op": "cross", "dtype": "f16", "batch": 8, "heads": 16, "kv_heads": 16,
         "queries": 448, "keys": 1500, "d": 64, "lengths": "none", "train": False},
        # A training step of a decoder over padded encoder states, four query heads to a key head.
        {"name": "cross_train", "op": "cross", "dtype": "bf16", "batch": 4, "heads": 32, "kv_heads": 8, "queries": 1024,
         "keys": 2048, "d": 128, "lengths": "ragged", "train": True},
        # A small fp32 step off every tile size, with a sample that has no encoder states at all.
        {"name": "cross_train_odd", "op": "cross", "dtype": "f32", "batch": 3, "heads": 8, "kv_heads": 8, "queries": 257,
         "keys": 383, "d": 80, "lengths": "empty", "train": True},
        # The longest call: 32 heads of 8192 queries over 8192 states of another sequence.
        {"name": "cross_long", "op": "cross", "dtype": "bf16", "batch": 1, "heads": 32, "kv_heads": 32, "queries": 8192,
         "keys": 8192, "d": 128, "lengths": "none", "train": False},
        # A small chat server: four conversations behind one short instruction.
        {"name": "prefix_small", "op": "prefix", "dtype": "bf16", "batch": 4, "heads": 16, "kv_heads": 16, "queries": 1,
         "prefix": 512, "keys": 256, "d": 64},
        # 64 sequences that sample from one long document, each with up to 1024 tokens of its own.
        {"name": "prefix_serve", "op": "prefix", "dtype": "bf16", "batch": 64, "heads": 32, "kv_heads": 8, "queries": 1,
         "prefix": 8192, "keys": 1024, "d": 128},
        # The same kind of server checking five drafted tokens a sequence at once.
        {"name": "prefix_draft", "op": "prefix", "dtype": "f16", "batch": 24, "heads": 32, "kv_heads": 4, "queries": 5,
         "prefix": 3001, "keys": 700, "d": 128},
        # The new tokens of 32 sequences, at positions of their own.
        {"name": "rope_token", "op": "rope", "dtype": "bf16", "batch": 32, "heads": 32, "kv_heads": 8, "tokens": 1,
         "d": 128, "rot": 128, "interleaved": False, "far": 131072, "train": False},
        # A prompt of 8191 tokens, half of each head rotated, neighbouring elements paired.
        {"name": "rope_prompt", "op": "rope", "dtype": "f16", "batch": 1, "heads": 16, "kv_heads": 16, "tokens": 8191,
         "d": 64, "rot": 32, "interleaved": True, "far": 8192, "train": False},
        # A training step over a fused projection's output.
        {"name": "rope_train", "op": "rope", "dtype": "bf16", "batch": 2, "heads": 32, "kv_heads": 8, "tokens": 8192,
         "d": 128, "rot": 128, "interleaved": False, "far": 8192, "train": True},
        # A small fp32 step with heads of an odd width, at far positions.
        {"name": "rope_train_odd", "op": "rope", "dtype": "f32", "batch": 3, "heads": 9, "kv_heads": 3, "tokens": 333,
         "d": 80, "rot": 40, "interleaved": False, "far": 4000000, "train": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["cross", "cross", "prefix", "rope"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 16])
    heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 8])
    d = rng.choice([16, 40, 64, 64, 80, 96, 120, 128, 128, 128])
    if kind == "rope":
        rot = rng.choice([d, d, d // 2])
        c = {"op": "rope", "dtype": dtype, "batch": _log(rng, 1, 16), "heads": heads, "kv_heads": kv_heads,
             "tokens": rng.choice([1, _log(rng, 1, 8192), _log(rng, 1, 8192)]), "d": d, "rot": rot,
             "interleaved": rng.random() < 0.3, "far": rng.choice([8192, 131072, 4000000]),
             "train": rng.random() < 0.5}
        while c["batch"] * c["tokens"] * (heads + kv_heads) * d > 2 * 8192 * 40 * 128 // 2:
            c["tokens"] = (c["tokens"] + 1) // 2
        return c
    if kind == "prefix":
        c = {"op": "prefix", "dtype": dtype, "batch": _log(rng, 1, 64), "heads": heads, "kv_heads": kv_heads,
             "queries": rng.choice([1, 1, rng.randint(2, 12)]), "prefix": _log(rng, 1, 8192),
             "keys": _log(rng, 16, 2048), "d": d}
        while c["batch"] * heads * c["queries"] * (c["prefix"] + c["keys"]) * d > 64 * 32 * 9216 * 128:
            c["batch"] = (c["batch"] + 1) // 2
            c["prefix"] = (c["prefix"] + 1) // 2
        return c
    train = rng.random() < 0.5
    c = {"op": "cross", "dtype": dtype, "batch": _log(rng, 1, 16), "heads": heads, "kv_heads": kv_heads,
         "queries": 1 if not train and rng.random() < 0.4 else _log(rng, 1, 4096), "keys": _log(rng, 1, 4096), "d": d,
         "lengths": rng.choice(["none", "ragged", "ragged", "empty"]), "train": train}
    while c["batch"] * heads * c["queries"] * c["keys"] > (1 << 27 if dtype == "f32" else 1 << 28):
        c["batch"] = (c["batch"] + 1) // 2
        c["queries"] = (c["queries"] + 1) // 2
    return c


# ----------------------------------------------------------------- inputs


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[c["dtype"]]
    B, H, Hk, D = c["batch"], c["heads"], c["kv_heads"], c["d"]

    def normal(*shape):
        return torch.randn(*shape, device=DEV, generator=g).to(dt)

    def whole(lo, hi, *shape):
        return torch.randint(lo, hi, shape, device=DEV, generator=g)

    s = {"case": c}
    if c["op"] == "rope":
        T = c["tokens"]
        # one projection's output for queries, keys and values; heads as views of it
        fused = normal(B, T, H + 2 * Hk, D)
        s["Q"], s["K"] = fused[:, :, :H].transpose(1, 2), fused[:, :, H:H + Hk].transpose(1, 2)
        s["wq"], s["wk"] = ((1 + 0.1 * torch.randn(D, device=DEV, generator=g)).to(dt) for _ in range(2))
        s["inv_freq"] = 10000.0 ** (-torch.arange(0, c["rot"], 2, device=DEV, dtype=torch.float64) / c["rot"])
        # consecutive tokens from each sequence's own start
        start = whole(0, max(1, c["far"] - T + 1), B, 1)
        s["pos"] = start + torch.arange(T, device=DEV)
        if c["train"]:
            s["gQ"], s["gK"] = normal(B, H, T, D), normal(B, Hk, T, D)
            for k in ("Q", "K", "wq", "wk"):
                s[k].requires_grad_()
        return s
    N = c["queries"]
    s["Q"] = normal(B, N, H, D).transpose(1, 2)  # a projection's output, heads as views of it
    if c["op"] == "prefix":
        kv = normal(2, Hk, c["prefix"], D)
        s["pK"], s["pV"] = kv[0], kv[1]
        cache = normal(2, B, Hk, c["keys"], D)  # rows behind a sequence's tokens hold what was there before
        s["K"], s["V"] = cache[0], cache[1]
        s["lengths"] = whole(min(N, c["keys"]), c["keys"] + 1, B)
        return s
    kv = normal(B, c["keys"], 2, Hk, D)  # keys and values of one projection
    s["K"], s["V"] = kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)
    s["lengths"] = None
    if c["lengths"] != "none":
        s["lengths"] = whole((c["keys"] + 3) // 4, c["keys"] + 1, B)
        if c["lengths"] == "empty":
            s["lengths"][B // 2] = 0
    if c["train"]:
        s["G"] = normal(B, N, H, D).transpose(1, 2)
        for k in ("Q", "K", "V"):
            s[k].requires_grad_()
    return s


# -------------------------------------------------------------------- run


def run(state):
    s, c = state, state["case"]
    if own:
        return _own(s, c)
    with torch.no_grad():
        return {"cross": _cross, "prefix": _prefix, "rope": _rope}[c["op"]](s, c)


def _own(s, c):
    import trnsparse_amd as ts

    if c["op"] == "rope":
        out = ts.qk_norm_rope(s["Q"], s["K"], s["wq"], s["wk"], s["pos"], s["inv_freq"], interleaved=c["interleaved"])
        if not c["train"]:
            return out
        return (*out, *torch.autograd.grad(out, (s["Q"], s["K"], s["wq"], s["wk"]), (s["gQ"], s["gK"])))
    if c["op"] == "prefix":
        return ts.shared_prefix_attention(s["Q"], s["pK"], s["pV"], s["K"], s["V"], s["lengths"])
    out = ts.cross_attention(s["Q"], s["K"], s["V"], s["lengths"])
    if not c["train"]:
        return out
    return (out, *torch.autograd.grad(out, (s["Q"], s["K"], s["V"]), s["G"]))


def _softmax(S):
    """Rows of S to probabilities; a row of -inf alone to zeros."""
    m = S.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    P = torch.exp(S - m)
    total = P.sum(-1, keepdim=True)
    return P / torch.where(total == 0, 1.0, total)


def _cross(s, c):
    B, H, Hk, N, L, D = c["batch"], c["heads"], c["kv_heads"], c["queries"], c["keys"], c["d"]
    dt, scale = s["Q"].dtype, D**-0.5
    Q = s["Q"].float().reshape(B, Hk, H // Hk * N, D)
    K, V = s["K"].float(), s["V"].float()
    S = (Q @ K.transpose(2, 3).contiguous()) * scale
    if s["lengths"] is not None:
        S = torch.where(torch.arange(L, device=DEV) < s["lengths"].view(B, 1, 1, 1), S, -math.inf)
    P = _softmax(S)
    del S
    O = P @ V
    out = O.reshape(B, H, N, D).to(dt)
    if not c["train"]:
        return out
    G = s["G"].float().reshape(B, Hk, H // Hk * N, D)
    dV = P.transpose(2, 3).contiguous() @ G
    dS = P * (G @ V.transpose(2, 3).contiguous() - (G * O).sum(-1, keepdim=True)) * scale
    dQ = dS @ K.contiguous()
    dK = dS.transpose(2, 3).contiguous() @ Q
    return out, dQ.reshape(B, H, N, D).to(dt), dK.to(dt), dV.to(dt)


def _prefix(s, c):
    B, H, Hk, N, L, D = c["batch"], c["heads"], c["kv_heads"], c["queries"], c["keys"], c["d"]
    G, P0 = H // Hk, c["prefix"]
    Q = s["Q"].float().reshape(B, Hk, G * N, D) * D**-0.5
    pK, pV, K, V = (s[k].float() for k in ("pK", "pV", "K", "V"))
    Qp = Q.transpose(0, 1).reshape(Hk, B * G * N, D)
    Sp = (Qp @ pK.transpose(1, 2).contiguous()).view(Hk, B, G * N, P0).transpose(0, 1)
    So = Q @ K.transpose(2, 3).contiguous()
    last = s["lengths"].view(B, 1) - N + 1 + torch.arange(N, device=DEV)  # own keys that each token sees
    seen = torch.arange(L, device=DEV) < last.view(B, 1, N, 1)
    So = torch.where(seen, So.view(B, Hk * G, N, L), -math.inf).view(B, Hk, G * N, L)
    P = _softmax(torch.cat([Sp, So], -1))
    Pp = P[..., :P0].transpose(0, 1).reshape(Hk, B * G * N, P0)
    O = (Pp @ pV).view(Hk, B, G * N, D).transpose(0, 1) + P[..., P0:].contiguous() @ V
    return O.reshape(B, H, N, D).to(s["Q"].dtype)


def _pairs(x, rot, interleaved):
    """The two elements of every rotated pair of x, and what is not rotated."""
    if interleaved:
        return x[..., 0:rot:2], x[..., 1:rot:2], x[..., rot:]
    return x[..., : rot // 2], x[..., rot // 2 : rot], x[..., rot:]


def _join(a, b, rest, interleaved):
    if interleaved:
        return torch.cat([torch.stack([a, b], -1).flatten(-2), rest], -1)
    return torch.cat([a, b, rest], -1)


def _rope(s, c):
    rot, il, eps = c["rot"], c["interleaved"], 1e-6
    angle = s["pos"].double().unsqueeze(1).unsqueeze(-1) * s["inv_freq"]  # (batch, 1, tokens, rot / 2)
    cos, sin = angle.cos().float(), angle.sin().float()
    outs, grads, wgrads = [], [], []
    for x, w, g in (("Q", "wq", "gQ"), ("K", "wk", "gK")):
        dt = s[x].dtype
        X, W = s[x].float(), s[w].float()
        r = torch.rsqrt((X * X).mean(-1, keepdim=True) + eps)
        a, b, rest = _pairs(X * r * W, rot, il)
        outs.append(_join(a * cos - b * sin, b * cos + a * sin, rest, il).to(dt))
        if not c["train"]:
            continue
        a, b, rest = _pairs(s[g].float(), rot, il)
        dn = _join(a * cos + b * sin, b * cos - a * sin, rest, il)
        wgrads.append((dn * X * r).sum((0, 1, 2), dtype=torch.float64).to(dt))
        dn = dn * W
        grads.append((r * dn - X * (r**3) * (X * dn).mean(-1, keepdim=True)).to(dt))
    return (*outs, *grads, *wgrads)


# ------------------------------------------------------------------- work


def work(case):
    c = case
    e, B, H, Hk, D = SIZES[c["dtype"]], c["batch"], c["heads"], c["kv_heads"], c["d"]
    if c["op"] == "rope":
        n = B * c["tokens"] * (H + Hk) * D
        # forward: x in, y out; backward: x and the gradient in, a gradient out
        return {"bytes": (5 if c["train"] else 2) * n * e + 8 * B * c["tokens"], "flops": (20 if c["train"] else 8) * n}
    N, L = c["queries"], c["keys"]
    if c["op"] == "prefix":
        mean = (min(N, L) + L) / 2  # a sequence's own tokens, on average
        pairs = B * H * N * (c["prefix"] + mean)
        return {"bytes": int(e * D * (2 * B * H * N + 2 * Hk * c["prefix"] + 2 * B * Hk * mean)),
                "flops": int(4 * pairs * D)}
    used = 1.0 if c["lengths"] == "none" else 0.625
    if c["lengths"] == "empty":
        used *= (B - 1) / B
    pairs = B * H * N * L * used
    rows = B * H * N * D * e
    cols = B * Hk * L * D * e
    if not c["train"]:
        return {"bytes": int(2 * rows + 2 * cols * used), "flops": int(4 * pairs * D)}
    # Q, dO in; O, dQ out; K, V in; dK, dV out
    return {"bytes": int(4 * rows + 2 * cols * used + 2 * cols), "flops": int(14 * pairs * D)}


# ------------------------------------------------------------------ exact


def exact(case, seed):
    c, s = case, prepare(case, seed)
    s = {k: v.detach() if isinstance(v, torch.Tensor) else v for k, v in s.items()}
    with torch.no_grad():
        return {"cross": _exact_cross, "prefix": _exact_prefix, "rope": _exact_rope}[c["op"]](s, c)


def _exact_cross(s, c):
    B, H, Hk, N, L, D = c["batch"], c["heads"], c["kv_heads"], c["queries"], c["keys"], c["d"]
    f64 = torch.float64
    O, dQ = (torch.zeros(B, H, N, D, dtype=f64, device=DEV) for _ in range(2))
    dK, dV = (torch.zeros(B, Hk, L, D, dtype=f64, device=DEV) for _ in range(2))
    for b in range(B):
        n = L if s["lengths"] is None else int(s["lengths"][b])
        if n == 0:
            continue
        for h in range(H):
            k = h // (H // Hk)
            q, kk, vv = s["Q"][b, h].double(), s["K"][b, k, :n].double(), s["V"][b, k, :n].double()
            p = (torch.mm(q, kk.t()) / math.sqrt(D)).softmax(1)
            O[b, h] = torch.mm(p, vv)
            if c["train"]:
                g = s["G"][b, h].double()
                dp = torch.mm(g, vv.t())
                ds = p * (dp - (dp * p).sum(1, keepdim=True)) / math.sqrt(D)
                dQ[b, h] = torch.mm(ds, kk)
                dK[b, k, :n] += torch.mm(ds.t(), q)
                dV[b, k, :n] += torch.mm(p.t(), g)
    return (O, dQ, dK, dV) if c["train"] else O


def _exact_prefix(s, c):
    B, H, Hk, N = c["batch"], c["heads"], c["kv_heads"], c["queries"]
    pK, pV = s["pK"].double(), s["pV"].double()
    O = torch.zeros(B, H, N, c["d"], dtype=torch.float64, device=DEV)
    lengths = s["lengths"].tolist()
    for b in range(B):
        Kb, Vb = s["K"][b].double(), s["V"][b].double()
        for i in range(N):
            n = max(lengths[b] - (N - 1 - i), 0)
            K, V = torch.cat([pK, Kb[:, :n]], 1), torch.cat([pV, Vb[:, :n]], 1)
            q = s["Q"][b, :, i].double().view(Hk, H // Hk, -1)
            p = (torch.bmm(K, q.transpose(1, 2).contiguous()) / math.sqrt(c["d"])).softmax(1)
            O[b, :, i] = torch.bmm(p.transpose(1, 2).contiguous(), V).view(H, -1)
    return O


def _exact_rope(s, c):
    rot, il = c["rot"], c["interleaved"]
    j = torch.arange(rot // 2, device=DEV)
    first = 2 * j if il else j
    second = first + 1 if il else first + rot // 2
    turn = torch.polar(torch.ones(1, dtype=torch.float64, device=DEV),
                       s["pos"].double()[:, None, :, None] * s["inv_freq"])
    outs, grads, wgrads = [], [], []
    for x, w, g in (("Q", "wq", "gQ"), ("K", "wk", "gK")):
        x, w = s[x].double(), s[w].double()
        size = ((x * x).sum(-1, keepdim=True) / c["d"] + 1e-6).sqrt()
        unit = x / size

        def rotate(t, by):
            z = torch.complex(t[..., first], t[..., second]) * by
            t = t.clone()
            t[..., first], t[..., second] = z.real, z.imag
            return t

        outs.append(rotate(unit * w, turn))
        if c["train"]:
            back = rotate(s[g].double(), turn.conj())
            wgrads.append((back * unit).sum((0, 1, 2)))
            du = back * w
            grads.append((du - unit * (unit * du).sum(-1, keepdim=True) / c["d"]) / size)
    return (*outs, *grads, *wgrads)
