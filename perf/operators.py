"""Cases that measure the token-mixer operators next to the cleaning read: the gated delta rule
(chunked, with its gradients, and token by token over a cache) and layer norm with its gradients.

The gated delta rule keeps one K x V state S per head:

    S <- exp(g_t) S;   u_t = beta_t (v_t - S^T k_t);   S <- S + k_t u_t^T;   o_t = scale S^T q_t

``run`` computes the operators with elementary torch operations in 32 bits (``own`` false) or through
``ccq_b200`` (``own`` true); ``exact`` computes them token by token in 64 bits.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CHUNK = 64


def listed():
    return [
        # the training step of the repository's main benchmark shape
        dict(name="train dense", op="train", dtype="bf16", B=8, T=4096, H=16, HV=16, K=128, V=128, docs=0),
        # packed documents of many lengths, empty and one-token ones among them
        dict(name="train packed", op="train", dtype="bf16", B=1, T=20011, H=16, HV=16, K=128, V=128, docs=24),
        # fine-tuning on short fp16 sequences, two value heads to a key head, wider values
        dict(name="train grouped", op="train", dtype="fp16", B=2, T=333, H=4, HV=8, K=128, V=256, docs=0),
        # fp32 inputs at the size of the repository's CPU configuration
        dict(name="train fp32", op="train", dtype="fp32", B=2, T=512, H=4, HV=4, K=64, V=64, docs=0),
        # prefill of one long prompt on top of a cached prefix: few heads, a long axis
        dict(name="prefill long", op="prefill", dtype="bf16", B=1, T=16384, H=16, HV=16, K=128, V=128, docs=0),
        # prefill of a few short prompts, where latency counts
        dict(name="prefill short", op="prefill", dtype="bf16", B=4, T=77, H=8, HV=8, K=64, V=128, docs=0),
        # generation: one token for each of many requests
        dict(name="step batch", op="step", dtype="bf16", B=256, T=1, H=16, HV=16, K=128, V=128, docs=0),
        # generation for one request with wide heads
        dict(name="step single", op="step", dtype="bf16", B=1, T=1, H=6, HV=6, K=256, V=256, docs=0),
        # a few drafted tokens for each of some requests
        dict(name="step draft", op="step", dtype="fp16", B=24, T=5, H=8, HV=16, K=128, V=128, docs=0),
        # the norm in front of a mixer, with the residual stream added: a training step
        dict(name="norm residual", op="norm", dtype="bf16", rows=32768, D=2048, form="layer", residual=True, grad=True),
        # the gated norm behind a mixer: very many short rows
        dict(name="norm gated", op="norm", dtype="bf16", rows=524288, D=128, form="gated", residual=False, grad=True),
        # one generated token for each of some requests, forward only, an odd width
        dict(name="norm decode", op="norm", dtype="bf16", rows=61, D=1531, form="layer", residual=True, grad=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["train", "train", "train", "prefill", "prefill", "step", "step", "norm", "norm"])
    if op == "norm":
        form = rng.choice(["layer", "rms", "gated"])
        D = _log(rng, 33, 8192) if form != "gated" else rng.choice([64, 96, 128, 256])
        rows = _log(rng, 1, min(524288, 67108864 // D))
        return dict(op=op, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]) if rows * D < 16777216 else "bf16",
                    rows=rows, D=D, form=form, residual=form != "gated" and rng.random() < 0.5, grad=rng.random() < 0.7)
    H = rng.choice([1, 2, 4, 6, 8, 12, 16])
    HV = H * rng.choice([1, 1, 1, 2])
    if op == "step":
        B = _log(rng, 1, 256)
        T = 1 if rng.random() < 0.6 else rng.randint(2, 8)
        K, V = rng.choice([(64, 64), (128, 128), (128, 256), (96, 160), (256, 256)])
        B = max(1, min(B, 67108864 // (HV * K * V * T)))
        return dict(op=op, dtype=rng.choice(["bf16", "fp16", "fp32"]), B=B, T=T, H=H, HV=HV, K=K, V=V, docs=0)
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"])
    if dtype == "fp32":
        K, V, most = rng.choice([32, 64, 100]), rng.choice([32, 64, 128]), 8192
    else:
        K, V, most = rng.choice([64, 96, 128, 128]), rng.choice([64, 128, 128, 256]), 32768
    T = _log(rng, 1, min(most, 8192))
    B = _log(rng, 1, max(1, min(16, most * 16 * 128 // (T * HV * V))))
    docs = rng.randint(2, 16) if T >= 64 and rng.random() < 0.35 else 0
    return dict(op=op, dtype=dtype, B=1 if docs else B, T=T, H=H, HV=HV, K=K, V=V, docs=docs)


def _lens(case):
    """Document lengths of a packed case, the same for every seed: spread over their logarithm, one
    empty and one of a single token among them."""
    n, T = case["docs"], case["T"]
    rng = random.Random(n * 1000003 + T)
    w = [math.exp(rng.uniform(0.0, 4.0)) for _ in range(n)]
    lens = [int(T * x / sum(w)) for x in w]
    if n >= 3:
        lens[1], lens[2] = 0, 1
    lens[0] += T - sum(lens)
    return lens


def _unit(x):
    return x * torch.rsqrt((x * x).sum(-1, keepdim=True) + 1e-6)


def prepare(case, seed):
    dev = "cuda"
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    def rand(*shape):
        return torch.rand(*shape, generator=gen, device=dev)

    s = dict(case=case)
    if case["op"] == "norm":
        R, D = case["rows"], case["D"]
        s["x"] = (randn(R, D) * 1.5 + 0.3).to(dt)
        s["weight"] = 1.0 + 0.1 * randn(D)
        s["bias"] = 0.1 * randn(D) if case["form"] == "layer" else None
        s["residual"] = (randn(R, D) * 2.0).to(dt) if case["residual"] else None
        s["gate"] = randn(R, D).to(dt) if case["form"] == "gated" else None
        if case["grad"]:
            s["dy"] = randn(R, D).to(dt)
            s["dh"] = randn(R, D).to(dt) if case["residual"] else None
            for name in ("x", "weight", "bias", "residual", "gate"):
                if s[name] is not None:
                    s[name].requires_grad_(True)
        return s
    B, T, H, HV, K, V = (case[n] for n in ("B", "T", "H", "HV", "K", "V"))
    s["q"], s["k"] = (_unit(randn(B, T, H, K)).to(dt) for _ in range(2))
    s["v"] = randn(B, T, HV, V).to(dt)
    # gates as a layer makes them: decay -A softplus(a + bias), with A in 1..16 and steps of 0.001..0.1
    # by head, and a write strength from a sigmoid, both from a projection of the activations' type
    A, step = 1.0 + 15.0 * rand(HV), torch.exp(math.log(0.001) + rand(HV) * math.log(100.0))
    raw = randn(B, T, HV) + torch.log(torch.expm1(step))
    s["g"] = (-A * torch.log1p(torch.exp(raw))).to(dt)
    s["beta"] = torch.sigmoid(randn(B, T, HV)).to(dt)
    s["cu"] = None
    n = B
    if case["docs"]:
        ends = torch.tensor([0] + _lens(case)).cumsum(0)
        s["cu"], n = ends.to(dev), case["docs"]
    if case["op"] == "train":
        s["do"] = randn(B, T, HV, V).to(dt)
        for name in ("q", "k", "v", "g", "beta"):
            s[name].requires_grad_(True)
    else:
        s["state"] = 0.3 * randn(n, HV, K, V)
    return s


# ------------------------------------------------------------------------------------------------
# plain forms
# ------------------------------------------------------------------------------------------------
def _padding(case, dev):
    """For a packed case: the token of each [document, place], and which places hold one."""
    lens = torch.tensor(_lens(case))
    starts = lens.cumsum(0) - lens
    at = torch.arange(max(1, int(lens.max())))
    live = at[None, :] < lens[:, None]
    return torch.where(live, starts[:, None] + at[None, :], 0).to(dev), live.to(dev)


def _plain_chunked(q, k, v, g, beta, scale, state):
    """Chunks of 64 tokens: with G the running sum of g inside a chunk and D_ij = exp(G_i - G_j), j <= i,
    u solves (1 + strict(beta_i D_ij k_i.k_j)) u = beta (v - exp(G) S^T k)."""
    B, T, HV, K, V = *q.shape, v.shape[-1]
    n = (T + CHUNK - 1) // CHUNK

    def chunks(x):
        x = torch.nn.functional.pad(x, (0, 0) * (x.ndim - 2) + (0, n * CHUNK - T))
        return x.reshape(B, n, CHUNK, *x.shape[2:]).transpose(2, 3)

    q, k, v, g, beta = (chunks(x) for x in (q, k, v, g, beta))  # [B, n, HV, CHUNK, ...]
    G = g.cumsum(-1)
    row = torch.arange(CHUNK, device=q.device)
    low, strict = row[:, None] >= row[None, :], row[:, None] > row[None, :]
    D = torch.exp(torch.where(low, G[..., :, None] - G[..., None, :], float("-inf")))
    A = torch.where(strict, beta[..., None] * (k @ k.transpose(-1, -2)) * D, 0.0)
    inv, power = torch.eye(CHUNK, device=q.device) - A, A @ A
    for _ in range(5):  # 1/(1 + A) = (1 - A)(1 + A^2)(1 + A^4)..., A^64 = 0
        inv, power = inv + inv @ power, power @ power
    P = (q @ k.transpose(-1, -2)) * D * scale
    qg, kg = q * (scale * torch.exp(G))[..., None], k * torch.exp(G)[..., None]
    kd, last = (k * torch.exp(G[..., -1:] - G)[..., None]).transpose(-1, -2), torch.exp(G[..., -1])[..., None, None]
    S = state if state is not None else torch.zeros(B, HV, K, V, device=q.device)
    out = []
    for i in range(n):
        u = inv[:, i] @ (beta[:, i, ..., None] * (v[:, i] - kg[:, i] @ S))
        out.append(qg[:, i] @ S + P[:, i] @ u)
        S = last[:, i] * S + kd[:, i] @ u
    o = torch.stack(out, 1).transpose(2, 3).reshape(B, n * CHUNK, HV, V)[:, :T]
    return o, S


def _plain_rule(s, q, k, v, g, beta, state):
    case = s["case"]
    group = case["HV"] // case["H"]
    scale = case["K"] ** -0.5
    if group > 1:
        q, k = q.repeat_interleave(group, 2), k.repeat_interleave(group, 2)
    if not case["docs"]:
        return _plain_chunked(q, k, v, g, beta, scale, state)
    at, live = _padding(case, q.device)
    q, k, v, g, beta = (x[0][at] * live.reshape(*live.shape, *[1] * (x.ndim - 2)) for x in (q, k, v, g, beta))
    o, S = _plain_chunked(q, k, v, g, beta, scale, state)
    return o[live][None], S


def _plain(s):
    case = s["case"]
    if case["op"] == "norm":
        f = {n: None if s[n] is None else s[n].detach().float().requires_grad_(case["grad"])
             for n in ("x", "weight", "bias", "residual", "gate")}
        h = f["x"] if f["residual"] is None else f["x"] + f["residual"]
        c = h - h.mean(-1, keepdim=True) if case["form"] == "layer" else h
        y = c * torch.rsqrt((c * c).mean(-1, keepdim=True) + 1e-5) * f["weight"]
        y = y if f["bias"] is None else y + f["bias"]
        y = y if f["gate"] is None else y * f["gate"] / (1.0 + torch.exp(-f["gate"]))
        out = {"y": y.detach().to(s["x"].dtype)}
        if s["residual"] is not None:
            out["h"] = h.detach().to(s["x"].dtype)
        if case["grad"]:
            names = [n for n in f if f[n] is not None]
            outs, seen = ([y], [s["dy"].float()]) if s["dh"] is None else ([y, h], [s["dy"].float(), s["dh"].float()])
            for n, d in zip(names, torch.autograd.grad(outs, [f[n] for n in names], seen)):
                out["d" + n] = d.to(s[n].dtype)
        return out
    names = ("q", "k", "v", "g", "beta")
    if case["op"] == "train":
        f = [s[n].detach().float().requires_grad_(True) for n in names]
        o, _ = _plain_rule(s, *f, None)
        grads = torch.autograd.grad(o, f, s["do"].float())
        return {"o": o.detach().to(s["v"].dtype), **{"d" + n: d.to(s[n].dtype) for n, d in zip(names, grads)}}
    f = [s[n].float() for n in names]
    if case["op"] == "prefill":
        o, S = _plain_rule(s, *f, s["state"])
        return {"o": o.to(s["v"].dtype), "state": S}
    q, k, v, g, beta = f
    group = case["HV"] // case["H"]
    q, k = (x.repeat_interleave(group, 2) if group > 1 else x for x in (q, k))
    S, out = s["state"], []
    for t in range(case["T"]):
        S = S * torch.exp(g[:, t, :, None, None])
        u = beta[:, t, :, None] * (v[:, t] - (S * k[:, t, :, :, None]).sum(2))
        S = S + k[:, t, :, :, None] * u[:, :, None, :]
        out.append((S * q[:, t, :, :, None]).sum(2) * case["K"] ** -0.5)
    s["state"].copy_(S)
    return {"o": torch.stack(out, 1).to(s["v"].dtype), "state": s["state"]}


# ------------------------------------------------------------------------------------------------
# the framework's operators
# ------------------------------------------------------------------------------------------------
def _framework(s):
    import ccq_b200

    case = s["case"]
    if case["op"] == "norm":
        if case["form"] == "gated":
            y, h = ccq_b200.gated_rms_norm(s["x"], s["gate"], s["weight"], eps=1e-5), None
        else:
            norm = ccq_b200.layer_norm if case["form"] == "layer" else ccq_b200.rms_norm
            args = (s["x"], s["weight"], s["bias"]) if case["form"] == "layer" else (s["x"], s["weight"])
            y = norm(*args, eps=1e-5, residual=s["residual"])
            y, h = y if s["residual"] is not None else (y, None)
        out = {"y": y.detach()} if h is None else {"y": y.detach(), "h": h.detach()}
        if case["grad"]:
            names = [n for n in ("x", "weight", "bias", "residual", "gate") if s[n] is not None]
            outs, seen = ([y], [s["dy"]]) if h is None else ([y, h], [s["dy"], s["dh"]])
            out |= {"d" + n: d for n, d in zip(names, torch.autograd.grad(outs, [s[n] for n in names], seen))}
        return out
    names = ("q", "k", "v", "g", "beta")
    f = [s[n] for n in names]
    if case["op"] == "train":
        o, _ = ccq_b200.gated_delta_rule(*f, cu_seqlens=s["cu"])
        grads = torch.autograd.grad(o, f, s["do"])
        return {"o": o.detach(), **{"d" + n: d for n, d in zip(names, grads)}}
    if case["op"] == "prefill":
        o, S = ccq_b200.gated_delta_rule(*f, initial_state=s["state"], output_final_state=True, cu_seqlens=s["cu"])
        return {"o": o, "state": S}
    o, S = ccq_b200.gated_delta_step(*f, s["state"], inplace=True)
    return {"o": o, "state": S}


def run(state):
    return _framework(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------------
# work and 64-bit values
# ------------------------------------------------------------------------------------------------
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "norm":
        n, D = case["rows"] * case["D"], case["D"]
        params = 2 if case["form"] == "layer" else 1
        reads = 1 + case["residual"] + (case["form"] == "gated")
        moved = reads + 1 + case["residual"]  # inputs, y and the summed stream
        flops = 8 * n
        if case["grad"]:
            # output gradients in, input gradients out (x and the stream it is added to share one)
            moved += 1 + case["residual"] + 1 + (case["form"] == "gated")
            params *= 2
            flops += 12 * n
        return {"bytes": moved * n * size + params * D * 4, "flops": flops}
    B, T, H, HV, K, V = (case[n] for n in ("B", "T", "H", "HV", "K", "V"))
    qk, v, gates = B * T * H * K, B * T * HV * V, B * T * HV
    heads = B * T * HV
    if case["op"] == "train":
        return {"bytes": (2 * (2 * qk + v + 2 * gates) + 2 * v) * size, "flops": 18 * heads * K * V}
    n = case["docs"] or B
    return {"bytes": (2 * qk + 2 * v + 2 * gates) * size + 2 * 4 * n * HV * K * V, "flops": 6 * heads * K * V}


def _exact_norm(s, case):
    x, w = s["x"].detach().double(), s["weight"].detach().double()
    h = x if s["residual"] is None else x + s["residual"].detach().double()
    D = h.shape[-1]
    mu = h.sum(-1, keepdim=True) / D if case["form"] == "layer" else torch.zeros_like(h[:, :1])
    r = 1.0 / torch.sqrt(((h - mu) ** 2).sum(-1, keepdim=True) / D + 1e-5)
    n = (h - mu) * r
    core = n * w if s["bias"] is None else n * w + s["bias"].detach().double()
    gate = None if s["gate"] is None else s["gate"].detach().double()
    sig = None if gate is None else torch.sigmoid(gate)
    out = {"y": core if gate is None else core * gate * sig}
    if s["residual"] is not None:
        out["h"] = h
    if not case["grad"]:
        return out
    dy = s["dy"].double()
    dcore = dy if gate is None else dy * gate * sig
    if gate is not None:
        out["dgate"] = dy * core * sig * (1.0 + gate * (1.0 - sig))
    out["dweight"] = (dcore * n).sum(0)
    if s["bias"] is not None:
        out["dbias"] = dcore.sum(0)
    dn = dcore * w
    dh = r * (dn - n * (dn * n).sum(-1, keepdim=True) / D)
    if case["form"] == "layer":
        dh = dh - r * dn.sum(-1, keepdim=True) / D
    if s["dh"] is not None:
        dh = dh + s["dh"].double()
    out["dx"] = dh
    if s["residual"] is not None:
        out["dresidual"] = dh
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        return _exact_norm(s, case)
    if case["T"] > 20000 and not case["docs"]:
        return None
    H, HV, K, V = (case[n] for n in ("H", "HV", "K", "V"))
    f = [s[n].detach().double() for n in ("q", "k", "v", "g", "beta")] + ([s["do"].double()] if case["op"] == "train" else [])
    if case["docs"]:
        at, live = _padding(case, f[0].device)
        f = [x[0][at] * live.reshape(*live.shape, *[1] * (x.ndim - 2)) for x in f]
    q, k, v, g, beta = f[:5]
    q, k = (x.repeat_interleave(HV // H, 2) for x in (q, k))
    N, T = q.shape[:2]
    scale = K ** -0.5
    S = s["state"].double() if "state" in s else torch.zeros(N, HV, K, V, dtype=torch.float64, device=q.device)
    decay = torch.exp(g)[..., None, None]

    def token(S, t):
        Sd = S * decay[:, t]
        e = v[:, t] - torch.einsum("nhkv,nhk->nhv", Sd, k[:, t])
        u = beta[:, t, :, None] * e
        return Sd, e, u, Sd + torch.einsum("nhk,nhv->nhkv", k[:, t], u)

    o, kept = torch.empty_like(v), []
    for t in range(T):
        if t % CHUNK == 0 and case["op"] == "train":
            kept.append(S)
        S = token(S, t)[3]
        o[:, t] = scale * torch.einsum("nhkv,nhk->nhv", S, q[:, t])
    whole = (lambda x: x[live][None]) if case["docs"] else (lambda x: x)
    if case["op"] != "train":
        return {"o": whole(o), "state": S}
    do = f[5]
    dq, dk, dv, dg, dbeta = (torch.empty_like(x) for x in (q, k, v, g, beta))
    dS = torch.zeros_like(S)
    for c in range(len(kept) - 1, -1, -1):
        first, S, seen = c * CHUNK, kept.pop(), []
        for t in range(first, min(T, first + CHUNK)):
            seen.append(token(S, t))
            S = seen[-1][3]
        for t in range(min(T, first + CHUNK) - 1, first - 1, -1):
            Sd, e, u, S = seen.pop()
            dq[:, t] = scale * torch.einsum("nhkv,nhv->nhk", S, do[:, t])
            dS = dS + scale * torch.einsum("nhk,nhv->nhkv", q[:, t], do[:, t])
            du = torch.einsum("nhkv,nhk->nhv", dS, k[:, t])
            de = beta[:, t, :, None] * du
            dk[:, t] = torch.einsum("nhkv,nhv->nhk", dS, u) - torch.einsum("nhkv,nhv->nhk", Sd, de)
            dbeta[:, t] = (du * e).sum(-1)
            dv[:, t] = de
            dS = dS - torch.einsum("nhk,nhv->nhkv", k[:, t], de)
            dg[:, t] = (dS * Sd).sum((-1, -2))
            dS = dS * decay[:, t]
    dq, dk = (x.reshape(N, T, H, HV // H, K).sum(3) for x in (dq, dk))
    return {"o": whole(o), **{n: whole(x) for n, x in (("dq", dq), ("dk", dk), ("dv", dv), ("dg", dg), ("dbeta", dbeta))}}
