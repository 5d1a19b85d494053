"""Timed cases of three further training operators: linear attention with a
decay for each head, layer norm, and updates orthogonalised by Newton-Schulz
products.

Each operator has a plain form in elementary torch operations (32-bit
arithmetic whatever the inputs' type, rounded once at the end), the same call
through the framework, and its definition in 64 bits.  ``own`` selects between
the first two.

Linear attention (per row and head, scan order t; g is the log decay, of a head
or of every step and head, and a step that is ``reset`` forgets the state):

    S_t = exp(g_t) S_{t-1} + k_t v_t^T,   y_t = scale S_t^T q_t
    (steps past the row's length leave S and give y = 0)

Layer norm over the last dimension, with one weight for all rows or one for
each head:

    y = (x - mean(x)) / sqrt(var(x) + eps) * weight + bias

Muon over many matrices at once, on X = U / max(|U|, eps) of the shorter side first:

    m = beta m + (1 - beta) g,   U = beta m + (1 - beta) g
    five times:  A = X X^T,  X = a X + (b A + c A A) X
    p = p (1 - lr decay) - lr adjust X,   adjust = sqrt(max(1, rows / columns))
"""

import math

import torch

own = False

LN_EPS = 1e-5
COEFFICIENTS = (3.4445, -4.775, 2.0315)
NS_STEPS, NS_EPS = 5, 1e-7
LR, BETA, DECAY = 0.02, 0.95, 0.1
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
CHUNK = 64  # of the plain form


# ----------------------------------------------------------------------------------------------- cases


def listed():
    return [
        # one frame for each of 16 live streams: the latency of a streaming enhancer's attention
        attention("attention one frame, 16 streams", 16, 1, 8, 64, 64, "bf16"),
        # 8 utterances of 8 s at a hop of 256 samples, in inference
        attention("attention 8 x 8 s", 8, 500, 12, 64, 64, "bf16", packed=True),
        # one long recording at a short hop, in pieces that restart the state; few heads, odd widths
        attention("attention one long recording", 1, 65537, 4, 48, 33, "f32", gated=True, reset=True),
        # training on 64 clips of 8 s, a decay for every step
        attention("attention training 64 x 8 s", 64, 500, 14, 64, 64, "bf16", gated=True, train=True, packed=True),
        # training of a backward-in-time layer on clips of different lengths, wide heads
        attention("attention training ragged, reversed", 6, 4001, 5, 96, 128, "f16", train=True, reverse=True, ragged=True),
        # one frame for each of 16 live streams
        norm("layer norm one frame, 16 streams", 16, 1, 1, 512, "bf16", "bf16"),
        # training on 64 clips of 8 s, over all channels
        norm("layer norm training 64 x 8 s", 64, 500, 1, 896, "bf16", "bf16", train=True),
        # what follows the attention: every head normed by itself, a weight for each
        norm("layer norm of heads, training", 64, 500, 14, 64, "bf16", "bf16", bias=False, train=True),
        # a 32-bit residual stream of odd width normed for a 16-bit block
        norm("layer norm training, 32-bit stream", 6, 4001, 1, 1155, "f32", "f16", train=True),
        # a small enhancer's matrices
        muon("muon small model", 96, 6, "f32"),
        # a large one's, 16-bit gradients and working copies
        muon("muon large model", 1280, 4, "bf16", copies=True),
        # a stack of odd matrices orthogonalised by themselves
        orthogonal("orthogonalise a stack of odd matrices", 9, 385, 1155, "f32"),
    ]


def attention(name, batch, steps, heads, key, value, dtype, gated=False, reset=False, train=False, reverse=False,
              ragged=False, packed=False):
    return {"name": name, "op": "attention", "batch": batch, "steps": steps, "heads": heads, "key": key, "value": value,
            "dtype": dtype, "gated": gated, "reset": reset, "train": train, "reverse": reverse, "ragged": ragged,
            "packed": packed}


def norm(name, batch, steps, heads, width, dtype, out, bias=True, train=False):
    return {"name": name, "op": "norm", "batch": batch, "steps": steps, "heads": heads, "width": width, "dtype": dtype,
            "out": out, "bias": bias, "train": train}


def muon(name, width, layers, dtype, copies=False):
    return {"name": name, "op": "muon", "width": width, "layers": layers, "dtype": dtype, "copies": copies}


def orthogonal(name, count, rows, columns, dtype):
    return {"name": name, "op": "orthogonal", "count": count, "rows": rows, "columns": columns, "dtype": dtype}


def draw(rng):
    def size(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    op = rng.choice(("attention", "attention", "attention", "norm", "norm", "muon", "orthogonal"))
    if op == "attention":
        dtype = rng.choice(("f32", "bf16", "f16"))
        heads, key, value = rng.randint(1, 16), size(8, 128), size(8, 128)
        batch = size(1, 64)
        most = 14_000_000 // (heads * max(key, value) * batch)  # at most half the largest listed case's elements
        steps = 1 if rng.random() < 0.2 or most < 2 else size(2, min(most, 70000))
        case = attention("", batch, steps, heads, key, value, dtype, rng.random() < 0.5, rng.random() < 0.3,
                         rng.random() < 0.5, rng.random() < 0.3, rng.random() < 0.3, rng.random() < 0.5)
    elif op == "norm":
        dtype = rng.choice(("f32", "bf16", "f16"))
        heads = rng.randint(2, 16) if rng.random() < 0.4 else 1
        width = size(16, 128) if heads > 1 else size(16, 4096)
        batch = size(1, 64)
        steps = 1 if rng.random() < 0.2 else size(2, max(3, 14_000_000 // (heads * width * batch)))
        case = norm("", batch, steps, heads, width, dtype, rng.choice(("bf16", "f16")) if dtype == "f32" else dtype,
                    rng.random() < 0.7, rng.random() < 0.6)
    elif op == "muon":
        dtype = rng.choice(("f32", "bf16", "f16"))
        case = muon("", size(24, 900), rng.randint(1, 5), dtype, copies=dtype != "f32" and rng.random() < 0.5)
    else:
        case = orthogonal("", rng.randint(1, 9), size(8, 1100), size(8, 1100), rng.choice(("f32", "bf16", "f16")))
    del case["name"]
    return case


def shapes(case):
    """The matrices of an enhancer of `layers` blocks on 257 spectrum bins."""
    d = case["width"]
    return [(d, 257)] + [(3 * d, d), (d, d)] * case["layers"] + [(257, d)]


def newton_schulz_flops(rows, columns):
    n, m = min(rows, columns), max(rows, columns)
    return NS_STEPS * (n * (n + 1) * m + n * n * (n + 1) + 2 * n * n * m)  # of symmetric products one half


def work(case):
    if case["op"] == "attention":
        tokens = case["batch"] * case["steps"] * case["heads"]
        key, value, size = case["key"], case["value"], BYTES[case["dtype"]]
        state = 4 * case["batch"] * case["heads"] * key * value
        decay = 4 * tokens if case["gated"] else 4 * case["heads"]
        one = tokens * (2 * key + 2 * value) * size + decay + 2 * state  # q, k, v, state in; y, state out
        if not case["train"]:
            return {"bytes": one, "flops": 4 * tokens * key * value}
        # and dy, dlast in, the five gradients out
        return {"bytes": one + tokens * (2 * key + 2 * value) * size + decay + 2 * state, "flops": 12 * tokens * key * value}
    if case["op"] == "norm":
        n = case["batch"] * case["steps"] * case["heads"] * case["width"]
        vectors = 4 * case["heads"] * case["width"] * (2 if case["bias"] else 1)
        one = n * (BYTES[case["dtype"]] + BYTES[case["out"]])
        if not case["train"]:
            return {"bytes": one + vectors, "flops": 8 * n}
        return {"bytes": 2 * (one + vectors), "flops": 20 * n}
    if case["op"] == "orthogonal":
        n = case["count"] * case["rows"] * case["columns"]
        return {"bytes": 2 * n * BYTES[case["dtype"]],
                "flops": case["count"] * newton_schulz_flops(case["rows"], case["columns"])}
    n = sum(r * c for r, c in shapes(case))
    return {"bytes": n * (16 + BYTES[case["dtype"]] + (2 if case["copies"] else 0)),
            "flops": sum(newton_schulz_flops(r, c) for r, c in shapes(case))}


# ---------------------------------------------------------------------------------------------- inputs


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    return {"attention": _prepare_attention, "norm": _prepare_norm, "muon": _prepare_muon,
            "orthogonal": _prepare_orthogonal}[case["op"]](case, g, normal)


def _prepare_attention(case, g, normal):
    b, t, h, dk, dv = (case[k] for k in ("batch", "steps", "heads", "key", "value"))
    dt = TYPES[case["dtype"]]
    if case["packed"]:  # slices of one projection's output
        q, k, v = normal(b, t, h * (2 * dk + dv)).to(dt).split((h * dk, h * dk, h * dv), dim=2)
        q, k, v = q.view(b, t, h, dk), k.view(b, t, h, dk), v.view(b, t, h, dv)
    else:
        q, k, v = normal(b, t, h, dk).to(dt), normal(b, t, h, dk).to(dt), normal(b, t, h, dv).to(dt)
    if case["gated"]:  # -softplus of a projection, as far from zero as half-lives of 2 to 200 steps
        decay = -torch.nn.functional.softplus(1.5 * normal(b, t, h) - 3.0)
    else:
        decay = torch.log1p(-torch.exp2(-3.0 - 5.0 * torch.rand(h, device="cuda", generator=g)))
    s = {"case": case, "q": q, "k": k, "v": v, "decay": decay, "state": normal(b, h, dk, dv), "reset": None,
         "lengths": None, "scale": dk**-0.5}
    if case["reset"]:
        s["reset"] = torch.rand(b, t, device="cuda", generator=g) < 1.0 / 700
    if case["ragged"]:
        s["lengths"] = torch.randint(0, t + 1, (b,), device="cuda", generator=g)
    if case["train"]:
        s |= {"dy": normal(b, t, h, dv).to(dt), "dlast": normal(b, h, dk, dv)}
        for name in ("q", "k", "v", "decay", "state"):  # a training program's leaves
            s[name] = s[name].detach().requires_grad_(True)
    return s


def _prepare_norm(case, g, normal):
    b, t, h, d = (case[k] for k in ("batch", "steps", "heads", "width"))
    shape, vector = ((b, t, d), (d,)) if h == 1 else ((b, t, h, d), (h, d))
    s = {"case": case, "x": (0.3 + 1.5 * normal(*shape)).to(TYPES[case["dtype"]]), "weight": 1 + 0.1 * normal(*vector),
         "bias": 0.1 * normal(*vector) if case["bias"] else None}
    if case["train"]:
        s["dy"] = normal(*shape).to(TYPES[case["out"]])
        s["leaves"] = [k for k in ("x", "weight", "bias") if s[k] is not None]
        for k in s["leaves"]:
            s[k] = s[k].detach().requires_grad_(True)
    return s


def _prepare_muon(case, g, normal):
    dt = TYPES[case["dtype"]]
    s = {"case": case, "params": [], "grads": [], "momenta": [], "copies": [] if case["copies"] else None}
    for rows, columns in shapes(case):
        rank = max(1, min(rows, columns) // 8)  # a part of few directions, as gradients have, and noise
        few = normal(rows, rank) @ normal(rank, columns) * (2.0 / rank**0.5)
        s["params"].append(0.05 * normal(rows, columns))
        s["grads"].append((1e-3 * (few + normal(rows, columns))).to(dt))
        s["momenta"].append(5e-4 * (few + normal(rows, columns)))
        if case["copies"]:
            s["copies"].append(s["params"][-1].to(dt))
    return s


def _prepare_orthogonal(case, g, normal):
    return {"case": case, "x": normal(case["count"], case["rows"], case["columns"]).to(TYPES[case["dtype"]])}


# ------------------------------------------------------------------------------------------- one pass


def run(s):
    return {"attention": _run_attention, "norm": _run_norm, "muon": _run_muon,
            "orthogonal": _run_orthogonal}[s["case"]["op"]](s)


def _run_attention(s):
    c = s["case"]
    if not own:
        return _plain_attention(s, c)
    from triton_pesq_b200 import linear_attention

    y, last = linear_attention(s["q"], s["k"], s["v"], s["decay"], s["state"], reset=s["reset"], lengths=s["lengths"],
                               reverse=c["reverse"], scale=s["scale"])
    if not c["train"]:
        return {"y": y, "last": last}
    grads = torch.autograd.grad((y, last), [s[k] for k in ("q", "k", "v", "decay", "state")], (s["dy"], s["dlast"]))
    return {"y": y, "last": last, "grads": grads}


def _run_norm(s):
    c = s["case"]
    if not own:
        return _plain_norm(s, c)
    from triton_pesq_b200 import layer_norm

    y = layer_norm(s["x"], s["weight"], s["bias"], eps=LN_EPS, dtype=TYPES[c["out"]])
    if not c["train"]:
        return {"y": y}
    return {"y": y, "grads": torch.autograd.grad(y, [s[k] for k in s["leaves"]], s["dy"])}


def _run_muon(s):
    if not own:
        return _plain_muon(s, s["case"])
    from triton_pesq_b200 import muon_step

    muon_step(s["params"], s["grads"], s["momenta"], copies=s["copies"], lr=LR, momentum=BETA, weight_decay=DECAY,
              coefficients=COEFFICIENTS, eps=NS_EPS, steps=NS_STEPS)
    return {k: s[k] for k in ("params", "momenta", "copies")}


def _run_orthogonal(s):
    if not own:
        x = s["x"].float()
        return _newton_schulz(x).to(s["x"].dtype)
    from triton_pesq_b200 import orthogonalize

    return orthogonalize(s["x"], coefficients=COEFFICIENTS, eps=NS_EPS, steps=NS_STEPS)


# ----------------------------------------------------------------------------------------- plain forms


def _chunk(s, lo, hi, live, reverse):
    """Steps lo .. hi - 1 in scan order, [batch, head, step, ...] in 32 bits, and the decays between them."""
    n = s["q"].shape[1]

    def take(x):
        part = x[:, n - hi:n - lo].flip(1) if reverse else x[:, lo:hi]
        return part.transpose(1, 2)

    g = s["decay"].float()
    g = g[None, None].expand(s["q"].shape[0], n, -1) if g.dim() == 1 else g
    g = take(g).double()
    on = None if live is None else take(live[:, :, None]).expand(g.shape)
    if on is not None:
        g = torch.where(on, g, 0.0)
    cut = torch.zeros_like(g, dtype=torch.bool) if s["reset"] is None else take(s["reset"][:, :, None]).expand(g.shape)
    if on is not None:
        cut = cut & on
    g = torch.where(cut, 0.0, g)
    total, pieces = g.cumsum(2), cut.cumsum(2)
    order = torch.ones(hi - lo, hi - lo, dtype=torch.bool, device=g.device).tril()
    same = order & (pieces[:, :, :, None] == pieces[:, :, None, :])
    between = torch.where(same, torch.exp(torch.where(order, total[:, :, :, None] - total[:, :, None, :], 0.0)), 0.0).float()
    before = torch.where(pieces == 0, torch.exp(total), 0.0).float()
    after = torch.where(pieces == pieces[:, :, -1:], torch.exp(total[:, :, -1:] - total), 0.0).float()
    out = {"between": between, "before": before, "after": after, "live": on, "cut": cut}
    for k in ("q", "k", "v", "dy"):
        if k in s:
            x = take(s[k]).float()
            out[k] = x if on is None else torch.where(on[..., None], x, 0.0)
    return out


@torch.no_grad()
def _plain_attention(s, c):
    dt, n, scale = s["q"].dtype, s["q"].shape[1], s["scale"]
    live = None
    if s["lengths"] is not None:
        live = torch.arange(n, device="cuda")[None, :] < s["lengths"][:, None]
    state, starts, parts = s["state"], [], []
    edges = [(lo, min(lo + CHUNK, n)) for lo in range(0, n, CHUNK)]
    for lo, hi in edges:
        p = _chunk(s, lo, hi, live, c["reverse"])
        starts.append(state)
        y = ((p["q"] @ p["k"].transpose(2, 3)) * p["between"]) @ p["v"] + p["before"][..., None] * (p["q"] @ state)
        parts.append(y * scale if live is None else torch.where(p["live"][..., None], y * scale, 0.0))
        state = p["before"][:, :, -1, None, None] * state + (p["after"][..., None] * p["k"]).transpose(2, 3) @ p["v"]

    def whole(parts):
        x = torch.cat(parts, dim=2).transpose(1, 2)
        return x.flip(1) if c["reverse"] else x

    out = {"y": whole(parts).to(dt), "last": state.clone()}
    if not c["train"]:
        return out
    dstate, dq, dk, dv, dg = s["dlast"], [], [], [], []
    for (lo, hi), start in zip(reversed(edges), reversed(starts)):
        p = _chunk(s, lo, hi, live, c["reverse"])
        q, dy = p["q"] * scale, p["dy"]
        a = (q @ p["k"].transpose(2, 3)) * p["between"]
        d = (dy @ p["v"].transpose(2, 3)) * p["between"]
        dq_far = p["before"][..., None] * (dy @ start.transpose(2, 3))
        dk_far = p["after"][..., None] * (p["v"] @ dstate.transpose(2, 3))
        dq.append(scale * (d @ p["k"] + dq_far))
        dk.append(d.transpose(2, 3) @ q + dk_far)
        dv.append(a.transpose(2, 3) @ dy + p["after"][..., None] * (p["k"] @ dstate))
        # what the step's decay carries: from before it to it and later, within the chunk and across its ends
        w = ((a * (dy @ p["v"].transpose(2, 3)))).tril(-1)
        inside = torch.zeros_like(p["before"])
        w = w.flip(2).cumsum(2).flip(2)  # rows i >= t
        w = w.cumsum(3)                  # columns j <= t
        inside[:, :, 1:] = w.diagonal(offset=-1, dim1=2, dim2=3)
        from_start = (q * dq_far).sum(3).flip(2).cumsum(2).flip(2)
        to_end = (p["k"] * dk_far).sum(3).cumsum(2) - (p["k"] * dk_far).sum(3)
        through = p["before"][:, :, -1] * (start * dstate).sum((2, 3))
        t = inside + from_start + to_end + through[..., None]
        t = torch.where(p["cut"], 0.0, t)
        dg.append(t if live is None else torch.where(p["live"], t, 0.0))
        dstate = p["before"][:, :, -1, None, None] * dstate + (p["before"][..., None] * q).transpose(2, 3) @ dy
    for x in (dq, dk, dv, dg):
        x.reverse()
    ddecay = whole([x[..., None] for x in dg])[..., 0]
    if not c["gated"]:
        ddecay = ddecay.double().sum((0, 1)).float()
    out["grads"] = (whole(dq).to(dt), whole(dk).to(dt), whole(dv).to(dt), ddecay.contiguous(), dstate)
    return out


@torch.no_grad()
def _plain_norm(s, c):
    x, w = s["x"].float(), s["weight"]
    mean = x.mean(dim=-1, keepdim=True)
    x = x - mean
    r = torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + LN_EPS)
    h = x * r
    y = h * w if s["bias"] is None else h * w + s["bias"]
    out = {"y": y.to(TYPES[c["out"]])}
    if not c["train"]:
        return out
    dy = s["dy"].float()
    q = dy * w
    dx = r * (q - q.mean(dim=-1, keepdim=True) - h * (q * h).mean(dim=-1, keepdim=True))
    grads = [dx.to(s["x"].dtype), (dy * h).sum((0, 1))]
    if s["bias"] is not None:
        grads.append(dy.sum((0, 1)))
    return out | {"grads": tuple(grads)}


def _newton_schulz(u):
    a, b, c = COEFFICIENTS
    tall = u.shape[-2] > u.shape[-1]
    x = u.mT if tall else u
    x = x / x.square().sum((-2, -1), keepdim=True).sqrt().clamp_min(NS_EPS)
    for _ in range(NS_STEPS):
        gram = x @ x.mT
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.mT if tall else x


@torch.no_grad()
def _plain_muon(s, c):
    for i, (p, g, m) in enumerate(zip(s["params"], s["grads"], s["momenta"])):
        g = g.float()
        m.copy_(BETA * m + (1 - BETA) * g)
        x = _newton_schulz(BETA * m + (1 - BETA) * g)
        p.copy_(p * (1 - LR * DECAY) - LR * max(1.0, p.shape[0] / p.shape[1])**0.5 * x)
        if c["copies"]:
            s["copies"][i].copy_(p)
    return {k: s[k] for k in ("params", "momenta", "copies")}


# ------------------------------------------------------------------------------------ 64-bit definition


def exact(case, seed):
    s = prepare(case, seed)
    return {"attention": _exact_attention, "norm": _exact_norm, "muon": _exact_muon,
            "orthogonal": _exact_orthogonal}[case["op"]](case, s)


def _exact_attention(c, s):
    """Step by step.  What a step's decay carries is what its queries and keys from there on receive (the sum of
    q dq - k dk over the steps at and after it) and what the last state does."""
    if c["steps"] > 20000:
        return None
    n, scale = c["steps"], s["scale"]
    q, k, v, state = (s[x].detach().double() for x in ("q", "k", "v", "state"))
    g = s["decay"].detach().double()
    g = g.expand(c["batch"], n, c["heads"]) if g.dim() == 1 else g
    a = torch.exp(g)
    if s["reset"] is not None:
        a = a.masked_fill(s["reset"][:, :, None], 0.0)
    past = None
    if s["lengths"] is not None:
        past = torch.arange(n, device="cuda")[None, :] >= s["lengths"][:, None]
        a = a.masked_fill(past[:, :, None], 1.0)
        q, k, v = (x.masked_fill(past[:, :, None, None], 0.0) for x in (q, k, v))
    order = range(n - 1, -1, -1) if c["reverse"] else range(n)
    y, dq = torch.empty_like(v), torch.empty_like(q)
    train = c["train"]
    if train:
        dy = s["dy"].double()
        if past is not None:
            dy = dy.masked_fill(past[:, :, None, None], 0.0)
    for t in order:
        state = state * a[:, t, :, None, None] + k[:, t, :, :, None] * v[:, t, :, None, :]
        y[:, t] = scale * (q[:, t, :, None, :] @ state)[:, :, 0]
        if train:
            dq[:, t] = scale * (state @ dy[:, t, :, :, None])[..., 0]
    out = {"y": y, "last": state}
    if not train:
        return out
    ds, dk, dv, dg = s["dlast"].double(), torch.empty_like(k), torch.empty_like(v), torch.empty_like(a)
    carried = (state * ds).sum((2, 3))
    for t in reversed(order):
        ds = ds + scale * q[:, t, :, :, None] * dy[:, t, :, None, :]
        dk[:, t] = (ds @ v[:, t, :, :, None])[..., 0]
        dv[:, t] = (k[:, t, :, None, :] @ ds)[:, :, 0]
        ds = ds * a[:, t, :, None, None]
        carried = carried + (q[:, t] * dq[:, t]).sum(2) - (k[:, t] * dk[:, t]).sum(2)
        dg[:, t] = carried
    if s["reset"] is not None:
        dg = dg.masked_fill(s["reset"][:, :, None], 0.0)
    if past is not None:
        dg = dg.masked_fill(past[:, :, None], 0.0)
    out["grads"] = (dq, dk, dv, dg if c["gated"] else dg.sum((0, 1)), ds)
    return out


def _exact_norm(c, s):
    x, w = s["x"].detach().double().requires_grad_(c["train"]), s["weight"].detach().double().requires_grad_(c["train"])
    leaves = [x, w]
    var, mean = torch.var_mean(x, dim=-1, correction=0, keepdim=True)
    y = (x - mean) / (var + LN_EPS)**0.5 * w
    if c["bias"]:
        leaves.append(s["bias"].detach().double().requires_grad_(c["train"]))
        y = y + leaves[-1]
    out = {"y": y.detach()}
    if c["train"]:
        out["grads"] = torch.autograd.grad(y, leaves, s["dy"].double())
    return out


def _exact_polynomial(u):
    """The iteration acts on the singular values alone: an odd polynomial of each.  The singular vectors come from
    the Gram matrix of the shorter side, on which X = f(U U^T) U."""
    a, b, c = COEFFICIENTS
    tall = u.shape[-2] > u.shape[-1]
    u = u.mT if tall else u
    u = u / torch.linalg.matrix_norm(u, keepdim=True).clamp_min(NS_EPS)
    value, vector = torch.linalg.eigh(u @ u.mT)
    square, factor = value.clamp_min(0.0), torch.ones_like(value)
    for _ in range(NS_STEPS):
        step = a + b * square + c * square**2
        factor, square = factor * step, square * step**2
    x = (vector * factor[..., None, :]) @ (vector.mT @ u)
    return x.mT if tall else x


def _exact_muon(c, s):
    out = {"params": [], "momenta": [], "copies": [] if c["copies"] else None}
    for p, g, m in zip(s["params"], s["grads"], s["momenta"]):
        m = m.double() + (g.double() - m.double()) * (1 - BETA)
        x = _exact_polynomial(g.double() + (m - g.double()) * BETA)
        new = p.double() - LR * DECAY * p.double() - LR * max(1.0, p.shape[0] / p.shape[1])**0.5 * x
        out["params"].append(new)
        out["momenta"].append(m)
        if c["copies"]:
            out["copies"].append(new)
    return out


def _exact_orthogonal(c, s):
    return _exact_polynomial(s["x"].double())
