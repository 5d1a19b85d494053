"""Timed cases of the training operators: the gated linear recurrence, the
norm-gate-residual join and the AdamW step.

Each operator has a plain form in elementary torch operations (32-bit
arithmetic whatever the inputs' type, rounded once at the end), the same call
through the framework, and its definition in 64 bits.  ``own`` selects between
the first two.

Gated linear recurrence (per row b and channel d, scan order t):

    r = sigmoid(decay_gate),  i = sigmoid(input_gate)
    log a = -rate * softplus(decay) * r          (a = 0 where ``reset``)
    h_t = a_t h_{t-1} + sqrt(1 - a_t^2) i_t x_t  (steps past the row's length leave h and give y = 0)

Join of a block's output with the residual stream:

    stream' = stream + scale * act(gate) * rms(block) * post_weight
    normed  = rms(stream') * pre_weight,   rms(v) = v / sqrt(mean(v^2) + eps)

AdamW over many tensors at once, moments in 32 bits or as float8_e4m3fn in
blocks of 256 with a 32-bit scale each (the second moment as its root, rounded
stochastically with bits hashed from position, step and seed).
"""

import math

import torch

own = False

RATE = 8.0
EPS = 1e-6
BLOCK = 256
TOP = 448.0  # largest float8_e4m3fn
LR, BETA1, BETA2, ADAM_EPS, DECAY, SEED = 1e-3, 0.9, 0.999, 1e-8, 0.01, 7
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
ACTS = ("sigmoid", "silu")


# ----------------------------------------------------------------------------------------------- cases


def listed():
    return [
        # one frame for each of 16 live streams: the latency of a streaming enhancer's recurrence
        scan("scan one frame, 16 streams", 16, 1, 512, "bf16"),
        # 8 utterances of 8 s at a hop of 256 samples, in inference
        scan("scan 8 x 8 s", 8, 500, 768, "bf16", packed=True),
        # one long recording at a short hop, in pieces that restart the state, few channels wide
        scan("scan one long recording", 1, 65537, 129, "f32", reset=True),
        # training on 64 clips of 8 s: forward and backward
        scan("scan training 64 x 8 s", 64, 500, 896, "bf16", train=True, packed=True),
        # training of a backward-in-time layer on clips of different lengths, 32-bit streams, odd width
        scan("scan training ragged, reversed", 6, 4001, 385, "f32", train=True, reverse=True, ragged=True),
        # one frame for each of 16 live streams
        join("join one frame, 16 streams", 16, 1, 512, "bf16", "bf16"),
        # 8 utterances of 8 s in inference, 32-bit residual stream beside a 16-bit block
        join("join 8 x 8 s", 8, 500, 768, "f32", "bf16", act="silu"),
        # training on 64 clips of 8 s
        join("join training 64 x 8 s", 64, 500, 896, "bf16", "bf16", train=True),
        # training with one gate per clip for all its frames, 32 bits, odd width
        join("join training, shared gate", 6, 1500, 385, "f32", "f32", train=True, shared=True),
        # a small enhancer's optimiser step: many tensors, little in each
        adamw("adamw small model", 96, 6, 32, "f32"),
        # a large one, moments in 8 bits, 16-bit gradients and working copies
        adamw("adamw 8-bit large model", 1280, 16, 8, "bf16", copies=True),
        # the same sizes in 32 bits
        adamw("adamw 32-bit model", 1040, 8, 32, "f32"),
    ]


def scan(name, batch, steps, width, dtype, train=False, reverse=False, reset=False, ragged=False, packed=False):
    return {"name": name, "op": "scan", "batch": batch, "steps": steps, "width": width, "dtype": dtype, "train": train,
            "reverse": reverse, "reset": reset, "ragged": ragged, "packed": packed}


def join(name, batch, steps, width, stream, dtype, act="sigmoid", train=False, shared=False):
    return {"name": name, "op": "join", "batch": batch, "steps": steps, "width": width, "stream": stream, "dtype": dtype,
            "act": act, "train": train, "shared": shared}


def adamw(name, width, layers, bits, dtype, copies=False):
    return {"name": name, "op": "adamw", "width": width, "layers": layers, "bits": bits, "dtype": dtype, "copies": copies}


def draw(rng):
    def size(low, high):
        n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
        return n - 1 if n in (1024, 3072) else n

    op = rng.choice(("scan", "scan", "join", "join", "adamw"))
    if op == "adamw":
        bits = rng.choice((8, 32))
        dtype = rng.choice(("f32", "bf16"))
        case = adamw("", size(24, 1024), rng.randint(1, 12), bits, dtype, copies=dtype == "bf16" and rng.random() < 0.5)
    else:
        dtype = rng.choice(("f32", "bf16", "f16"))
        width = size(16, 2048)
        batch = size(1, 64)
        most = 16_000_000 // (width * batch)  # at most half the largest listed case's elements, in 32 bits its bytes
        steps = 1 if rng.random() < 0.2 or most < 2 else size(2, min(most, 70000))
        train = rng.random() < 0.5
        if op == "scan":
            case = scan("", batch, steps, width, dtype, train, rng.random() < 0.3, rng.random() < 0.3, rng.random() < 0.3,
                        rng.random() < 0.5)
        else:
            case = join("", batch, steps, width, rng.choice(("f32", dtype)), dtype, rng.choice(ACTS), train,
                        rng.random() < 0.3)
    del case["name"]
    return case


def shapes(case):
    """Parameters of an enhancer of `layers` blocks on 257 spectrum bins: projections, and the vectors beside them."""
    d = case["width"]
    block = [(3 * d, d), (d, d), (3 * d,), (d,), (d,), (d,), (d,), (d,)]
    return [(d, 257), (d,)] + block * case["layers"] + [(257, d), (257,)]


def work(case):
    if case["op"] == "adamw":
        n = sum(math.prod(s) for s in shapes(case))
        moments = 16 if case["bits"] == 32 else 4 + 16 / BLOCK
        return {"bytes": n * (8 + BYTES[case["dtype"]] + moments + (2 if case["copies"] else 0)), "flops": n * 16}
    n = case["batch"] * case["steps"] * case["width"]
    if case["op"] == "scan":
        state = 8 * case["batch"] * case["width"] + 4 * case["width"]
        if not case["train"]:
            return {"bytes": 4 * n * BYTES[case["dtype"]] + state, "flops": 20 * n}
        return {"bytes": 8 * n * BYTES[case["dtype"]] + 2 * state, "flops": 60 * n}
    s, b = BYTES[case["stream"]], BYTES[case["dtype"]]
    gate = b * (case["batch"] * case["width"] if case["shared"] else n)
    flops = (16 if not case["train"] else 56) * n
    if not case["train"]:  # stream, block, gate in; stream, normed out
        return {"bytes": n * (2 * s + 2 * b) + gate + 12 * case["width"], "flops": flops}
    # and both upstream gradients in; the three inputs' gradients out
    return {"bytes": n * (4 * s + 4 * b) + 2 * gate + 24 * case["width"], "flops": flops}


# ---------------------------------------------------------------------------------------------- inputs


def prepare(case, seed):
    return {"scan": _prepare_scan, "join": _prepare_join, "adamw": _prepare_adamw}[case["op"]](case, seed)


def _source(seed):
    return torch.Generator("cuda").manual_seed(seed)


def _prepare_scan(case, seed):
    g = _source(seed)
    b, t, d, dt = case["batch"], case["steps"], case["width"], TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    if case["packed"]:  # slices of one projection's output
        x, ig, rg = normal(b, t, 3 * d).to(dt).chunk(3, dim=2)
    else:
        x, ig, rg = normal(b, t, d).to(dt), (1.5 * normal(b, t, d)).to(dt), (1.5 * normal(b, t, d)).to(dt)
    slow = 0.9 + 0.099 * torch.rand(d, device="cuda", generator=g)  # a at an open decay gate
    s = {"case": case, "x": x, "ig": ig, "rg": rg, "decay": torch.log(torch.expm1(-torch.log(slow) / RATE)),
         "state": normal(b, d), "reset": None, "lengths": None}
    if case["reset"]:
        s["reset"] = torch.rand(b, t, device="cuda", generator=g) < 1.0 / 700
    if case["ragged"]:
        s["lengths"] = torch.randint(0, t + 1, (b,), device="cuda", generator=g)
    if case["train"]:
        s |= {"dy": normal(b, t, d).to(dt), "dlast": normal(b, d)}
        for k in ("x", "ig", "rg", "decay", "state"):  # a training program's leaves
            s[k] = s[k].detach().requires_grad_(True)
    return s


def _prepare_join(case, seed):
    g = _source(seed)
    b, t, d = case["batch"], case["steps"], case["width"]
    ds, dt = TYPES[case["stream"]], TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    s = {"case": case, "stream": (2 * normal(b, t, d)).to(ds), "block": (0.5 * normal(b, t, d)).to(dt),
         "gate": normal(b, 1 if case["shared"] else t, d).to(dt), "post": 1 + 0.1 * normal(d), "pre": 1 + 0.1 * normal(d),
         "scale": 0.5 + 0.1 * normal(d)}
    if case["train"]:
        s |= {"dstream": normal(b, t, d).to(ds), "dnormed": normal(b, t, d).to(dt)}
        for k in ("stream", "block", "gate", "post", "pre", "scale"):
            s[k] = s[k].detach().requires_grad_(True)
    return s


def _prepare_adamw(case, seed):
    """Every buffer is flat, a tensor's part beginning at a multiple of 256 values; the tensors are views of it."""
    g = _source(seed)
    at, total = [], 0
    for s in shapes(case):
        at.append((total, math.prod(s), s))
        total += -(-math.prod(s) // BLOCK) * BLOCK
    live = torch.zeros(total, device="cuda")
    for o, n, _ in at:
        live[o:o + n] = 1

    def normal():
        return torch.randn(total, device="cuda", generator=g) * live

    param, grad = 0.05 * normal(), (1e-3 * normal()).to(TYPES[case["dtype"]])
    m, v = 3e-4 * normal(), (1e-3 * normal()).square() * torch.rand(total, device="cuda", generator=g)
    s = {"case": case, "param": param, "grad": grad, "scales": None, "copy": None, "copies": None,
         "step": torch.tensor([99, 0], device="cuda")}
    s["params"] = [param[o:o + n].view(z) for o, n, z in at]
    s["grads"] = [grad[o:o + n].view(z) for o, n, z in at]
    if case["copies"]:
        s["copy"] = param.to(TYPES[case["dtype"]])
        s["copies"] = [s["copy"][o:o + n].view(z) for o, n, z in at]
    if case["bits"] == 32:
        s["m"], s["v"] = m, v
    else:
        both = torch.stack([m, v.sqrt()]).view(2, -1, BLOCK)
        s["scales"] = both.abs().amax(dim=2) / TOP
        code = (both / s["scales"].clamp_min(1e-30)[:, :, None]).to(torch.float8_e4m3fn).view(2, -1)
        s["m"], s["v"] = code[0].clone(), code[1].clone()
    return s


# ------------------------------------------------------------------------------------------- one pass


def run(s):
    return {"scan": _run_scan, "join": _run_join, "adamw": _run_adamw}[s["case"]["op"]](s)


def _run_scan(s):
    c = s["case"]
    if not own:
        return _plain_scan(s, c)
    from triton_pesq_b200 import gated_scan

    y, last = gated_scan(s["x"], s["ig"], s["rg"], s["decay"], s["state"], reset=s["reset"], lengths=s["lengths"],
                         reverse=c["reverse"], rate=RATE)
    if not c["train"]:
        return {"y": y, "last": last}
    grads = torch.autograd.grad((y, last), (s["x"], s["ig"], s["rg"], s["decay"], s["state"]), (s["dy"], s["dlast"]))
    return {"y": y, "last": last, "grads": grads}


def _run_join(s):
    c = s["case"]
    if not own:
        return _plain_join(s, c)
    from triton_pesq_b200 import norm_join

    stream, normed = norm_join(s["stream"], s["block"], s["post"], s["pre"], gate=s["gate"], scale=s["scale"], eps=EPS,
                               activation=c["act"])
    if not c["train"]:
        return {"stream": stream, "normed": normed}
    grads = torch.autograd.grad((stream, normed), [s[k] for k in ("stream", "block", "gate", "post", "pre", "scale")],
                                (s["dstream"], s["dnormed"]))
    return {"stream": stream, "normed": normed, "grads": grads}


def _run_adamw(s):
    if not own:
        return _plain_adamw(s, s["case"])
    from triton_pesq_b200 import adamw_step

    adamw_step(s["params"], s["grads"], s["m"], s["v"], s["step"], scales=s["scales"], copies=s["copies"], lr=LR,
               betas=(BETA1, BETA2), eps=ADAM_EPS, weight_decay=DECAY, seed=SEED)
    return {k: s[k] for k in ("param", "m", "v", "scales", "copy", "step")}


# ----------------------------------------------------------------------------------------- plain forms


def _doubling(a, b):
    """All h_t = a_t h_{t-1} + b_t along dimension 1, by doubling the span that each step covers."""
    k = 1
    while k < a.shape[1]:
        b = torch.cat([b[:, :k], b[:, k:] + a[:, k:] * b[:, :-k]], dim=1)
        a = torch.cat([a[:, :k], a[:, k:] * a[:, :-k]], dim=1)
        k *= 2
    return b


@torch.no_grad()
def _plain_scan(s, c):
    dt = s["x"].dtype
    x, i, r = s["x"].float(), torch.sigmoid(s["ig"].float()), torch.sigmoid(s["rg"].float())
    soft = torch.log1p(torch.exp(s["decay"]))
    la = -RATE * soft * r
    a = torch.exp(la)
    beta = torch.sqrt(-torch.expm1(2 * la))
    slope = torch.where(beta > 0, a * a / beta, torch.zeros_like(beta))  # -d beta / d log a
    if s["reset"] is not None:
        keep = ~s["reset"][:, :, None]
        a, slope = a * keep, slope * keep
        beta = torch.where(keep, beta, torch.ones_like(beta))
    live = None
    if s["lengths"] is not None:
        live = (torch.arange(x.shape[1], device=x.device)[None, :] < s["lengths"][:, None])[:, :, None]
        a = torch.where(live, a, torch.ones_like(a))
        beta = beta * live
        slope = slope * live
    b = beta * i * x
    if c["reverse"]:
        a, b = a.flip(1), b.flip(1)
    b = torch.cat([b[:, :1] + a[:, :1] * s["state"][:, None], b[:, 1:]], dim=1)
    h = _doubling(a, b)
    last = h[:, -1]
    y = h.flip(1) if c["reverse"] else h
    if live is not None:
        y = y * live
    if not c["train"]:
        return {"y": y.to(dt), "last": last.clone()}
    dy = s["dy"].float()
    if live is not None:
        dy = dy * live
    if c["reverse"]:
        dy = dy.flip(1)
    dy = torch.cat([dy[:, :-1], dy[:, -1:] + s["dlast"][:, None]], dim=1)
    after = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], dim=1)
    g = _doubling(after.flip(1), dy.flip(1)).flip(1)  # g_t = dy_t + a_{t+1} g_{t+1}
    dstate = a[:, 0] * g[:, 0]
    before = torch.cat([s["state"][:, None], h[:, :-1]], dim=1)
    through = g * a * before
    if c["reverse"]:
        g, through = g.flip(1), through.flip(1)
    if live is not None:
        through = through * live
    dx = g * beta * i
    dig = dx * x * (1 - i)
    dla = through - g * slope * i * x
    drg = dla * la * (1 - r)
    ddecay = (dla * r).sum(dim=(0, 1)) * (-RATE * torch.sigmoid(s["decay"]))
    return {"y": y.to(dt), "last": last.clone(), "grads": (dx.to(dt), dig.to(dt), drg.to(dt), ddecay, dstate)}


@torch.no_grad()
def _plain_join(s, c):
    x, z, g = s["stream"].float(), s["block"].float(), s["gate"].float()
    rz = torch.rsqrt((z * z).mean(dim=2, keepdim=True) + EPS)
    zh = z * rz
    n = zh * s["post"]
    sig = torch.sigmoid(g)
    act = sig if c["act"] == "sigmoid" else g * sig
    r = x + s["scale"] * act * n
    rr = torch.rsqrt((r * r).mean(dim=2, keepdim=True) + EPS)
    rh = r * rr
    y = rh * s["pre"]
    out = {"stream": r.to(s["stream"].dtype), "normed": y.to(s["block"].dtype)}
    if not c["train"]:
        return out
    dy = s["dnormed"].float()
    q = dy * s["pre"]
    dr = s["dstream"].float() + rr * (q - rh * (q * rh).mean(dim=2, keepdim=True))
    dpre = (dy * rh).sum(dim=(0, 1))
    dscale = (dr * act * n).sum(dim=(0, 1))
    slope = sig * (1 - sig) if c["act"] == "sigmoid" else sig * (1 + g * (1 - sig))
    dg = dr * s["scale"] * n * slope
    if c["shared"]:
        dg = dg.sum(dim=1, keepdim=True)
    dn = dr * s["scale"] * act
    dpost = (dn * zh).sum(dim=(0, 1))
    q = dn * s["post"]
    dz = rz * (q - zh * (q * zh).mean(dim=2, keepdim=True))
    out["grads"] = (dr.to(s["stream"].dtype), dz.to(s["block"].dtype), dg.to(s["gate"].dtype), dpost, dpre, dscale)
    return out


def _hash(n, step):
    """32 bits for each position: a multiply-xorshift finaliser over position, step and seed."""
    word = 0xFFFFFFFF
    h = (torch.arange(n, device="cuda") + step * 0x9E3779B9 + SEED * 0x85EBCA6B) & word
    h = ((h ^ (h >> 16)) * 0x7FEB352D) & word
    h = ((h ^ (h >> 15)) * 0x846CA68B) & word
    return h ^ (h >> 16)


@torch.no_grad()
def _plain_adamw(s, c):
    p, g = s["param"], s["grad"].float()
    s["step"][0] += 1
    t = s["step"][0].double()
    c1, c2 = (1 - BETA1 ** t).float(), (1 - BETA2 ** t).float()
    m, v = s["m"].float(), s["v"].float()
    if c["bits"] == 8:
        m = (m.view(-1, BLOCK) * s["scales"][0][:, None]).view(-1)
        v = (v.view(-1, BLOCK) * s["scales"][1][:, None]).view(-1).square()
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * g * g
    root = torch.sqrt(v)
    p.copy_(p * (1 - LR * DECAY) - LR / c1 * m / (root / torch.sqrt(c2) + ADAM_EPS))
    if c["copies"]:
        s["copy"].copy_(p)
    if c["bits"] == 32:
        s["m"].copy_(m)
        s["v"].copy_(v)
    else:
        both = torch.stack([m, root]).view(2, -1, BLOCK)
        s["scales"].copy_(both.abs().amax(dim=2) * (1 / TOP))
        both = (both * torch.where(s["scales"] > 0, 1 / s["scales"], s["scales"])[:, :, None]).view(2, -1)
        s["m"].copy_(both[0].clamp(-TOP, TOP))
        # stochastic rounding to 3 mantissa bits (steps of 2^-9 below 2^-6), never to zero from above
        u = both[1].clamp(0, TOP)
        bits = _hash(u.numel(), s["step"][0]) & 0xFFFFF
        normal = ((u.view(torch.int32) + bits.int()) & ~0xFFFFF).view(torch.float32)
        small = torch.floor(u * 512 + bits.float() * 2.0**-20).clamp_min(1) / 512
        s["v"].copy_(torch.where(u >= 2.0**-6, normal, torch.where(u > 0, small, u)))
    return {k: s[k] for k in ("param", "m", "v", "scales", "copy", "step")}


# ------------------------------------------------------------------------------------ 64-bit definition


def exact(case, seed):
    made = {k: v.detach() if isinstance(v, torch.Tensor) else v for k, v in prepare(case, seed).items()}
    return {"scan": _exact_scan, "join": _exact_join, "adamw": _exact_adamw}[case["op"]](case, made)


def _exact_scan(c, s):
    names = ("x", "ig", "rg", "decay", "state")
    x, ig, rg, decay, state = (s[k].double().requires_grad_(c["train"]) for k in names)
    n = x.shape[1]
    la = -RATE * torch.nn.functional.softplus(decay, threshold=1000.0) * torch.sigmoid(rg)
    a = torch.exp(la)
    beta = torch.sqrt(-torch.expm1(2 * la))
    if s["reset"] is not None:
        cut = s["reset"][:, :, None]
        a = torch.where(cut, 0.0, a)
        beta = torch.where(cut, 1.0, beta)
    b = beta * torch.sigmoid(ig) * x
    if s["lengths"] is not None:
        past = (torch.arange(n, device="cuda")[None, :] >= s["lengths"][:, None])[:, :, None]
        a = torch.where(past, 1.0, a)
        b = torch.where(past, 0.0, b)
    order = range(n - 1, -1, -1) if c["reverse"] else range(n)
    with torch.no_grad():
        h, seen, before = state.detach(), torch.empty_like(b), torch.empty_like(b)
        for t in order:
            before[:, t] = h
            h = torch.addcmul(b[:, t], a[:, t], h)
            seen[:, t] = h
        if s["lengths"] is not None:
            seen = torch.where(past, 0.0, seen)
        if not c["train"]:
            return {"y": seen, "last": h}
        g, da, db = s["dlast"].double(), before, torch.empty_like(b)
        dy = s["dy"].double()
        if s["lengths"] is not None:
            dy = torch.where(past, 0.0, dy)
        for t in reversed(order):
            g = g + dy[:, t]
            db[:, t] = g
            da[:, t] *= g
            g = g * a[:, t]
    dx, dig, drg, ddecay = torch.autograd.grad((a, b), (x, ig, rg, decay), (da, db))
    return {"y": seen, "last": h, "grads": (dx, dig, drg, ddecay, g)}


def _exact_join(c, s):
    names = ("stream", "block", "gate", "post", "pre", "scale")
    leaf = [s[k].double().requires_grad_(c["train"]) for k in names]
    x, z, g, post, pre, scale = leaf

    def rms(v):
        return v / torch.sqrt(v.pow(2).mean(dim=-1, keepdim=True) + EPS)

    act = torch.nn.functional.silu(g) if c["act"] == "silu" else torch.sigmoid(g)
    stream = x + scale * act * (rms(z) * post)
    normed = rms(stream) * pre
    out = {"stream": stream.detach(), "normed": normed.detach()}
    if c["train"]:
        out["grads"] = torch.autograd.grad((stream, normed), leaf, (s["dstream"].double(), s["dnormed"].double()))
    return out


def _exact_adamw(c, s):
    """The 8-bit moments' values before their rounding, in units of their block's scale."""
    p, g, t = s["param"].double(), s["grad"].double(), int(s["step"][0]) + 1
    m, v = s["m"].double(), s["v"].double()
    if c["bits"] == 8:
        spread = s["scales"].double().repeat_interleave(BLOCK, dim=1)
        m, v = m * spread[0], (v * spread[1]) ** 2
    m = m + (g - m) * (1 - BETA1)
    v = v + (g**2 - v) * (1 - BETA2)
    new = p - LR * DECAY * p - LR * (m / (1 - BETA1**t)) / ((v / (1 - BETA2**t)) ** 0.5 + ADAM_EPS)
    out = {"param": new, "m": m, "v": v, "scales": None, "copy": new if c["copies"] else None, "step": None}
    if c["bits"] == 8:
        both = torch.stack([m, v**0.5]).reshape(2, -1, BLOCK)
        scales = both.abs().amax(dim=2) / TOP
        unit = (both / scales.clamp_min(1e-300)[:, :, None]).reshape(2, -1)
        out |= {"m": unit[0], "v": unit[1], "scales": scales}
    return out
