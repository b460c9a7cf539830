"""The token-encoder operators next to MaxSim, as cases to time and to compare.

Four operators of one path -- the encoder block in front of the late-interaction
scores, its training step and its INT8 serving form:

  gated_ffn      h = a(x Wg^T) * (x Wu^T) and its gradients
  norm_residual  z = scale x + gate * N(h), y = N(z) and their gradients
  int8_linear    y = (sx sw) * (codes_x codes_w^T) + b, x quantised per token
  adamw_step     AdamW over many tensors, moments in 32 bits or in 8 (e4m3 codes
                 with one scale per 256 values, stochastic rounding by a seed)

With `own` false `run` computes them in elementary torch operations in 32 bits,
rounded once at the end; with `own` true it calls this repository's package.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
EPS = 1e-6
BLOCK = 256  # values per scale of an 8-bit moment
HYPER = {"lr": 1e-3, "betas": (0.9, 0.999), "eps": 1e-8, "weight_decay": 0.01}
SEED = 20  # of the stochastic rounding


# --------------------------------------------------------------------------- cases

def listed():
    return [
        # one new token through the block while a query is typed: weights are all there is to read
        dict(name="ffn one token", op="gated_ffn", rows=1, dim=768, hidden=2048, dtype="bfloat16",
             act="silu", train=False),
        # encoding a ragged pack of documents for the index; sizes that no tile divides
        dict(name="ffn ragged documents", op="gated_ffn", rows=4099, dim=1000, hidden=2730,
             dtype="float16", act="gelu", train=False),
        # the queries of an in-batch training step: 256 queries of 32 tokens
        dict(name="ffn queries train", op="gated_ffn", rows=8192, dim=768, hidden=2048,
             dtype="bfloat16", act="silu", train=True),
        # the documents of that step: 256 documents of 180 tokens
        dict(name="ffn documents train", op="gated_ffn", rows=46080, dim=768, hidden=2048,
             dtype="float16", act="gelu", train=True),
        # one query of 32 tokens between two blocks
        dict(name="norm one query", op="norm_residual", batch=1, tokens=32, dim=768,
             dtype="bfloat16", kind="rms", gate="dim", scale=1.0, train=False),
        # the documents of the training step, each with its own gate
        dict(name="norm documents train", op="norm_residual", batch=256, tokens=180, dim=768,
             dtype="bfloat16", kind="layer", gate="sequence", scale=1.0, train=True),
        # a packed batch in 32 bits at an odd width
        dict(name="norm packed odd train", op="norm_residual", batch=1, tokens=16411, dim=1001,
             dtype="float32", kind="rms", gate="dim", scale=0.7, train=True),
        # one token through a serving projection
        dict(name="int8 one token", op="int8_linear", rows=1, dim=768, out=2048, dtype="bfloat16",
             bias=False),
        # documents projected to the width that the index keeps
        dict(name="int8 project documents", op="int8_linear", rows=46080, dim=768, out=128,
             dtype="float16", bias=True),
        # a wide layer over a large batch: matrix-product bound
        dict(name="int8 wide", op="int8_linear", rows=8192, dim=4096, out=8192, dtype="bfloat16",
             bias=False),
        # only the projection is trained: launch latency
        dict(name="adamw projection", op="adamw", bits=32, mode="float32", blocks=0, dim=768,
             hidden=2048, out=128),
        # all blocks of an encoder, 32-bit weights with 16-bit copies and 8-bit moments
        dict(name="adamw blocks 8 bits", op="adamw", bits=8, mode="mixed", blocks=24, dim=768,
             hidden=2048, out=128),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    def width(lo, hi):
        n = log(lo, hi)
        step = rng.choice([1, 8, 64])
        n = max(step, n // step * step)
        return n + step if n == 3 * 1024 else n

    op = rng.choice(["gated_ffn", "norm_residual", "int8_linear", "adamw"])
    if op == "gated_ffn":
        return dict(op=op, rows=log(1, 46080), dim=width(64, 768), hidden=width(128, 2048),
                    dtype=rng.choice(["float16", "bfloat16"]),
                    act=rng.choice(["silu", "gelu", "gelu_tanh", "relu"]),
                    train=rng.random() < 0.6)
    if op == "norm_residual":
        return dict(op=op, batch=log(1, 256), tokens=log(1, 180), dim=width(64, 768),
                    dtype=rng.choice(["float32", "float16", "bfloat16"]),
                    kind=rng.choice(["rms", "layer"]),
                    gate=rng.choice(["none", "dim", "sequence"]),
                    scale=rng.choice([1.0, 0.5, 1.25]), train=rng.random() < 0.6)
    if op == "int8_linear":
        return dict(op=op, rows=log(1, 8192), dim=width(64, 4096), out=width(64, 8192),
                    dtype=rng.choice(["float32", "float16", "bfloat16"]),
                    bias=rng.random() < 0.5)
    return dict(op=op, bits=rng.choice([8, 32]), mode=rng.choice(["float32", "bfloat16", "mixed"]),
                blocks=rng.randint(0, 16), dim=width(64, 768), hidden=width(128, 2048),
                out=width(32, 256))


# --------------------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _optimizer_shapes(c):
    d, f = c["dim"], c["hidden"]
    block = [(f, d), (f, d), (d, f), (d,), (d,), (d,)]
    return block * c["blocks"] + [(c["out"], d), (c["out"],)]


def _views(flat, shapes):
    """Views of `shapes` into a flat buffer, each starting on a multiple of 256 values."""
    out, at = [], 0
    for s in shapes:
        n = math.prod(s)
        out.append(flat[at:at + n].view(s))
        at += -(-n // BLOCK) * BLOCK
    return out


def _flat_numel(shapes):
    return sum(-(-math.prod(s) // BLOCK) * BLOCK for s in shapes)


def prepare(case, seed):
    g = _gen(seed)
    c = dict(case)
    if c["op"] == "gated_ffn":
        T, R, D, F = DTYPES[c["dtype"]], c["rows"], c["dim"], c["hidden"]
        s = {"case": c,
             "x": _randn(g, R, D).to(T),
             "w_gate": (_randn(g, F, D) / math.sqrt(D)).to(T),
             "w_up": (_randn(g, F, D) / math.sqrt(D)).to(T)}
        if c["train"]:
            s["dh"] = _randn(g, R, F).to(T)
            for k in ("x", "w_gate", "w_up"):
                s[k].requires_grad_()
        return s
    if c["op"] == "norm_residual":
        T, B, N, D = DTYPES[c["dtype"]], c["batch"], c["tokens"], c["dim"]
        s = {"case": c,
             "x": (2.0 * _randn(g, B, N, D)).to(T),
             "h": (0.5 * _randn(g, B, N, D) + 0.1).to(T),
             "w_post": (1.0 + 0.1 * _randn(g, D)).to(T),
             "w_pre": (1.0 + 0.1 * _randn(g, D)).to(T)}
        if c["kind"] == "layer":
            s["b_post"] = (0.1 * _randn(g, D)).to(T)
            s["b_pre"] = (0.1 * _randn(g, D)).to(T)
        if c["gate"] != "none":
            s["gate"] = (0.5 + 0.2 * _randn(g, *((D,) if c["gate"] == "dim" else (B, D)))).to(T)
        if c["train"]:
            for k in ("x", "h", "w_post", "w_pre", "b_post", "b_pre", "gate"):
                if k in s:
                    s[k].requires_grad_()
            s["dz"] = _randn(g, B, N, D).to(T)
            s["dy"] = _randn(g, B, N, D).to(T)
        return s
    if c["op"] == "int8_linear":
        T, R, K, C = DTYPES[c["dtype"]], c["rows"], c["dim"], c["out"]
        w = _randn(g, C, K) / math.sqrt(K)
        ws = w.abs().amax(1).clamp(min=1e-8) / 127.0
        return {"case": c, "x": _randn(g, R, K).to(T),
                "w_codes": torch.round(w / ws[:, None]).clamp(-127, 127).to(torch.int8),
                "w_scales": ws,
                "bias": (0.1 * _randn(g, C)).to(T) if c["bias"] else None}
    shapes = _optimizer_shapes(c)
    n = _flat_numel(shapes)
    P = torch.float32 if c["mode"] in ("float32", "mixed") else torch.bfloat16
    G = torch.float32 if c["mode"] == "float32" else torch.bfloat16
    s = {"case": c, "step": 100, "p": (0.05 * _randn(g, n)).to(P),
         "g": (1e-3 * _randn(g, n)).to(G)}
    s["params"], s["grads"] = _views(s["p"], shapes), _views(s["g"], shapes)
    s["copies"] = None
    if c["mode"] == "mixed":
        s["copy"] = s["p"].to(torch.bfloat16)
        s["copies"] = _views(s["copy"], shapes)
    m, r = 3e-4 * _randn(g, n), (1e-3 * _randn(g, n)).abs() + 1e-4
    if c["bits"] == 32:
        s["m"], s["v"] = m, r * r
        s["exp_avgs"], s["exp_avg_sqs"] = _views(s["m"], shapes), _views(s["v"], shapes)
        return s
    for name, x in (("m", m), ("v", r)):
        sc = x.view(-1, BLOCK).abs().amax(1) / 448.0
        s[name] = (x.view(-1, BLOCK) / sc[:, None]).view(-1).clamp(-448, 448).to(torch.float8_e4m3fn)
        s[name + "_scales"] = sc
        blocks = [(-(-math.prod(t) // BLOCK),) for t in shapes]
        at, views = 0, []
        for (b,) in blocks:
            views.append(sc[at:at + b])
            at += b
        s["exp_avgs" if name == "m" else "exp_avg_sqs"] = list(zip(_views(s[name], shapes), views))
    return s


# --------------------------------------------------------------------------- run

def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    import flashmaxsim_b200 as fms
    c = s["case"]
    if c["op"] == "gated_ffn":
        h = fms.gated_ffn(s["x"], s["w_gate"], s["w_up"], act=c["act"])
        if not c["train"]:
            return {"h": h}
        dx, dg, du = torch.autograd.grad(h, (s["x"], s["w_gate"], s["w_up"]), s["dh"])
        return {"h": h, "dx": dx, "dw_gate": dg, "dw_up": du}
    if c["op"] == "norm_residual":
        z, y = fms.norm_residual(s["x"], s["h"], s["w_post"], s["w_pre"], gate=s.get("gate"),
                                 b_post=s.get("b_post"), b_pre=s.get("b_pre"), scale=c["scale"],
                                 kind=c["kind"], eps=EPS)
        out = {"z": z, "y": y}
        if c["train"]:
            names = [k for k in ("x", "h", "w_post", "w_pre", "b_post", "b_pre", "gate") if k in s]
            grads = torch.autograd.grad((z, y), [s[k] for k in names], (s["dz"], s["dy"]))
            out.update(zip(["d" + k for k in names], grads))
        return out
    if c["op"] == "int8_linear":
        return {"y": fms.int8_linear(s["x"], fms.Int8Index(s["w_codes"], s["w_scales"]),
                                     bias=s["bias"])}
    s["step"] += 1
    fms.adamw_step(s["params"], s["grads"], s["exp_avgs"], s["exp_avg_sqs"], step=s["step"],
                   seed=SEED, copies=s["copies"], **HYPER)
    return _optimizer_outputs(s)


def _optimizer_outputs(s):
    return {k: s[k] for k in ("p", "copy", "m", "v", "m_scales", "v_scales") if k in s}


def _act(g, act):
    """a(g) and a'(g)."""
    if act == "silu":
        sig = 1.0 / (1.0 + torch.exp(-g))
        return g * sig, sig * (1.0 + g * (1.0 - sig))
    if act == "relu":
        on = (g > 0).to(g.dtype)
        return g * on, on
    if act == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(g * (1.0 / math.sqrt(2.0))))
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))
    k = math.sqrt(2.0 / math.pi)
    t = torch.tanh(k * (g + 0.044715 * g * g * g))
    return 0.5 * g * (1.0 + t), \
        0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * k * (1.0 + 3.0 * 0.044715 * g * g)


def _norm(v, w, b, kind):
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt((v * v).mean(-1, keepdim=True) + EPS)
    hat = v * rstd
    out = hat * w
    return (out if b is None else out + b), hat, rstd


def _norm_grad(dout, w, hat, rstd, kind):
    d = dout * w
    e = d - hat * (d * hat).mean(-1, keepdim=True)
    if kind == "layer":
        e = e - d.mean(-1, keepdim=True)
    return e * rstd


def _run_plain(s):
    c = s["case"]
    if c["op"] == "gated_ffn":
        return _ffn_plain(s, c)
    if c["op"] == "norm_residual":
        return _norm_plain(s, c)
    if c["op"] == "int8_linear":
        x = s["x"].float()
        sx = x.abs().amax(1).clamp(min=1e-8) / 127.0
        codes = torch.round((x / sx[:, None]).clamp(-127.0, 127.0))
        y = (sx[:, None] * s["w_scales"][None, :]) * (codes @ s["w_codes"].float().T)
        return {"y": (y if s["bias"] is None else y + s["bias"].float()).to(s["x"].dtype)}
    s["step"] += 1
    h = _host_constants(s["step"])
    ones = [None] * len(s["params"])
    [_adamw_plain(k, *t, h) for k, t in enumerate(
        zip(s["params"], s["grads"], s["exp_avgs"], s["exp_avg_sqs"], s["copies"] or ones))]
    return _optimizer_outputs(s)


@torch.no_grad()
def _ffn_plain(s, c):
    T = s["x"].dtype
    x, wg, wu = s["x"].float(), s["w_gate"].float(), s["w_up"].float()
    g, u = x @ wg.T, x @ wu.T
    a, da = _act(g, c["act"])
    out = {"h": (a * u).to(T)}
    if c["train"]:
        dh = s["dh"].float()
        dg, du = dh * u * da, dh * a
        out.update(dx=(dg @ wg + du @ wu).to(T), dw_gate=(dg.T @ x).to(T), dw_up=(du.T @ x).to(T))
    return out


@torch.no_grad()
def _norm_plain(s, c):
    T = s["x"].dtype
    f = {k: s[k].float() for k in ("x", "h", "w_post", "w_pre", "b_post", "b_pre", "gate") if k in s}
    gate = 1.0 if c["gate"] == "none" else f["gate"] if c["gate"] == "dim" else f["gate"][:, None, :]
    p, hhat, hr = _norm(f["h"], f["w_post"], f.get("b_post"), c["kind"])
    z = c["scale"] * f["x"] + gate * p
    y, zhat, zr = _norm(z, f["w_pre"], f.get("b_pre"), c["kind"])
    out = {"z": z.to(T), "y": y.to(T)}
    if c["train"]:
        dy = s["dy"].float()
        dz = s["dz"].float() + _norm_grad(dy, f["w_pre"], zhat, zr, c["kind"])
        dp = dz * gate
        out.update(dx=(c["scale"] * dz).to(T),
                   dh=_norm_grad(dp, f["w_post"], hhat, hr, c["kind"]).to(T),
                   dw_post=(dp * hhat).sum((0, 1)).to(T), dw_pre=(dy * zhat).sum((0, 1)).to(T))
        if c["kind"] == "layer":
            out.update(db_post=dp.sum((0, 1)).to(T), db_pre=dy.sum((0, 1)).to(T))
        if c["gate"] != "none":
            out["dgate"] = (dz * p).sum((0, 1) if c["gate"] == "dim" else 1).to(T)
    return out


# The random numbers of the stochastic rounding, an input of the step: 32 bits for
# each value from the seed, the step, the tensor's place in the list and the value's.

MASK = 0xFFFFFFFF


def _mix(h):
    h = h ^ (h >> 16)
    h = (h * 0x6A09E667) & MASK
    h = h ^ (h >> 15)
    h = (h * 0xBB67AE85) & MASK
    return h ^ (h >> 16)


def _random16(step, k, n):
    """Two 16-bit random whole numbers for each of the n values of tensor k."""
    key = _mix((_mix((SEED + step * 0x9E3779B1) & MASK) + k * 0x3C6EF373) & MASK)
    r = _mix(torch.arange(n, dtype=torch.int64, device=DEV) ^ key)
    return r & 0xFFFF, r >> 16


def _host_constants(step):
    b1, b2 = HYPER["betas"]
    return {"t": step, "b1": b1, "a1": 1.0 - b1, "b2": b2, "a2": 1.0 - b2,
            "size": HYPER["lr"] / (1.0 - b1 ** step), "rc2": 1.0 / math.sqrt(1.0 - b2 ** step),
            "eps": HYPER["eps"], "keep": 1.0 - HYPER["lr"] * HYPER["weight_decay"]}


def _blocks(x):
    return torch.nn.functional.pad(x, (0, -x.numel() % BLOCK)).view(-1, BLOCK)


def _decode(state, n):
    codes, scales = state
    return (_blocks(codes.reshape(-1).float()) * scales[:, None]).view(-1)[:n]


def _encode(x, r16, state, positive):
    """e4m3 codes of x with one scale per block of 256, rounded up with the probability of
    the part that is cut off (r16 / 65536 against it); a positive moment keeps a code over 0."""
    codes, scales = state
    n = x.numel()
    a = _blocks(x.abs())
    top = a.amax(1)
    sc = torch.where(top < 1e-30, torch.full_like(top, 1e-30), top) / 448.0
    a = (a * (1.0 / sc)[:, None]).clamp(max=448.0).view(-1)[:n]
    r16 = r16.to(torch.int32)
    big = ((a.view(torch.int32) + (r16 << 4)) >> 20) - 960
    small = (a * 512.0 + r16.float() * (1.0 / 65536.0)).to(torch.int32)
    k = torch.where(a < 0.015625, small, big).clamp(max=126)
    if positive:
        k = torch.where(x > 0, k.clamp(min=1), k)
    else:
        k = k + 128 * (x < 0)
    codes.view(-1).copy_(k.to(torch.uint8).view(torch.float8_e4m3fn))
    scales.copy_(sc)


@torch.no_grad()
def _adamw_plain(k, p, g, m_state, v_state, copy, h):
    n = p.numel()
    eight = isinstance(m_state, tuple)
    g = g.reshape(-1).float()
    if eight:
        m, r = _decode(m_state, n), _decode(v_state, n)
        v = r * r
    else:
        m, v = m_state.view(-1), v_state.view(-1)
    m = m * h["b1"] + g * h["a1"]
    v = v * h["b2"] + (g * g) * h["a2"]
    root = torch.sqrt(v)
    w = p.view(-1).float() * h["keep"] - (m * h["size"]) / (root * h["rc2"] + h["eps"])
    p.view(-1).copy_(w)
    if copy is not None:
        copy.view(-1).copy_(w)
    if eight:
        rm, rv = _random16(h["t"], k, n)
        _encode(m, rm, m_state, False)
        _encode(root, rv, v_state, True)
    else:
        m_state.view(-1).copy_(m)
        v_state.view(-1).copy_(v)


# --------------------------------------------------------------------------- work

def work(case):
    c = case
    if c["op"] == "gated_ffn":
        R, D, F = c["rows"], c["dim"], c["hidden"]
        b = R * D + 2 * F * D + R * F
        if c["train"]:
            b += R * F + R * D + 2 * F * D
        return {"bytes": 2 * b, "flops": (12 if c["train"] else 4) * R * D * F}
    if c["op"] == "norm_residual":
        e = 4 if c["dtype"] == "float32" else 2
        n = c["batch"] * c["tokens"] * c["dim"]
        # the gradients' pass reads x and h again: z and y stand between the two passes
        return {"bytes": e * n * (10 if c["train"] else 4), "flops": n * (40 if c["train"] else 15)}
    if c["op"] == "int8_linear":
        e = 4 if c["dtype"] == "float32" else 2
        R, K, C = c["rows"], c["dim"], c["out"]
        return {"bytes": e * R * K + C * K + 4 * C + e * R * C, "flops": 2 * R * K * C}
    n = sum(math.prod(s) for s in _optimizer_shapes(c))
    per = {"float32": 4 + 8, "bfloat16": 2 + 4, "mixed": 2 + 8 + 2}[c["mode"]]
    per += 16 if c["bits"] == 32 else 4 + 16 / BLOCK
    return {"bytes": int(n * per), "flops": 20 * n}


# --------------------------------------------------------------------------- 64 bits

@torch.no_grad()
def exact(case, seed):
    """The definitions in 64 bits, the gradients by torch's own differentiation of them."""
    s = prepare(case, seed)
    c = s["case"]
    if c["op"] == "gated_ffn":
        with torch.enable_grad():
            v = [s[k].detach().double().requires_grad_(c["train"]) for k in ("x", "w_gate", "w_up")]
            g, u = v[0] @ v[1].T, v[0] @ v[2].T
            if c["act"] == "silu":
                h = g * torch.sigmoid(g) * u
            elif c["act"] == "relu":
                h = torch.clamp(g, min=0) * u
            elif c["act"] == "gelu":
                h = g * torch.special.ndtr(g) * u
            else:
                h = g * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)) * u
            out = {"h": h.detach()}
            if c["train"]:
                d = torch.autograd.grad(h, v, s["dh"].double())
                out.update(dx=d[0], dw_gate=d[1], dw_up=d[2])
        return out
    if c["op"] == "norm_residual":
        names = [k for k in ("x", "h", "w_post", "w_pre", "b_post", "b_pre", "gate") if k in s]
        with torch.enable_grad():
            v = {k: s[k].detach().double().requires_grad_(c["train"]) for k in names}

            def norm(t, w, b):
                if c["kind"] == "rms":
                    return t * torch.rsqrt(t.pow(2).mean(-1, keepdim=True) + EPS) * w
                var, mean = torch.var_mean(t, -1, keepdim=True, correction=0)
                return (t - mean) * torch.rsqrt(var + EPS) * w + b

            p = norm(v["h"], v["w_post"], v.get("b_post"))
            if c["gate"] == "dim":
                p = p * v["gate"]
            elif c["gate"] == "sequence":
                p = p * v["gate"].unsqueeze(1)
            z = v["x"] * c["scale"] + p
            y = norm(z, v["w_pre"], v.get("b_pre"))
            out = {"z": z.detach(), "y": y.detach()}
            if c["train"]:
                d = torch.autograd.grad((z, y), [v[k] for k in names],
                                        (s["dz"].double(), s["dy"].double()))
                out.update(zip(["d" + k for k in names], d))
        return out
    if c["op"] == "int8_linear":
        x = s["x"].double()
        sx = torch.clamp(x.abs().max(dim=1).values, min=1e-8) / 127
        q = torch.clamp(x / sx.unsqueeze(1), -127, 127).round()
        y = torch.einsum("tk,ck->tc", q * sx.unsqueeze(1), s["w_codes"].double() * s["w_scales"].double().unsqueeze(1))
        return {"y": y if s["bias"] is None else y + s["bias"].double()}
    return _adamw_exact(s)


def _adamw_exact(s):
    b1, b2 = HYPER["betas"]
    t = s["step"] + 1
    out = {k: s[k].double() if k in s else None for k in ("p", "copy", "m", "v", "m_scales", "v_scales")}
    shapes = _optimizer_shapes(s["case"])
    at = 0
    for k, shape in enumerate(shapes):
        n = math.prod(shape)
        here, blocks = slice(at, at + n), slice(at // BLOCK, -(-(at + n) // BLOCK))
        at += -(-n // BLOCK) * BLOCK
        g = s["g"][here].double()
        m, v = out["m"][here], out["v"][here]
        if s["case"]["bits"] == 8:
            spread = lambda sc: sc[blocks].repeat_interleave(BLOCK)[:n]  # noqa: E731
            m, v = m * spread(out["m_scales"]), (v * spread(out["v_scales"])) ** 2
        m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g ** 2
        p = out["p"][here]
        p = p - HYPER["lr"] * HYPER["weight_decay"] * p \
            - HYPER["lr"] * (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + HYPER["eps"])
        out["p"][here] = p
        if out["copy"] is not None:
            out["copy"][here] = p
        if s["case"]["bits"] == 32:
            out["m"][here], out["v"][here] = m, v
            continue
        for name, x, r in zip("mv", (m, torch.sqrt(v)), _random16(t, k, n)):
            top = torch.stack([b.abs().max() for b in x.split(BLOCK)]) if n < 16 * BLOCK else \
                torch.cat([x, x.new_zeros(-n % BLOCK)]).reshape(-1, BLOCK).abs().max(dim=1).values
            sc = top / 448
            a = (x / sc.repeat_interleave(BLOCK)[:n]).abs()
            q = torch.exp2(torch.clamp(torch.floor(torch.log2(a)), min=-6.0) - 3)
            a = torch.floor(a / q + r.double() / 65536) * q
            out[name][here] = torch.clamp(a, max=448.0) * torch.sign(x)
            out[name + "_scales"][blocks] = sc
    return {k: v for k, v in out.items() if v is not None}
