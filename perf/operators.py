"""The transformer-block operators: layer norm, rotary positions and the gated feed-forward block, as cases to measure.

`run` computes a case in plain torch operations (`own` false) or through diffusion_model_amd (`own` true); `exact` gives
the same outputs from the definitions in 64 bits."""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZEOF = {"fp32": 4, "bf16": 2, "fp16": 2}


def listed():
    return [
        # one token of a decode loop, or one image's pooled vector: launch latency
        {"name": "norm token", "op": "norm", "rows": 1, "width": 4096, "dtype": "bf16", "affine": "same", "train": False},
        # the 16x16 tokens of 1024 images at the attention width of the widened model
        {"name": "norm image tokens", "op": "norm", "rows": 262144, "width": 256, "dtype": "fp32", "affine": "same", "train": False},
        # a training step on a ragged batch: odd row count, a width that fills no power of two, fp32 parameters
        {"name": "norm train ragged", "op": "norm", "rows": 8191, "width": 1000, "dtype": "fp16", "affine": "fp32", "train": True},
        # a training step at the width of a large model
        {"name": "norm train wide", "op": "norm", "rows": 32768, "width": 4096, "dtype": "bf16", "affine": "same", "train": True},
        # one new token for each of 64 requests, far into long contexts
        {"name": "rotary token", "op": "rotary", "batch": 64, "tokens": 1, "heads": 32, "kv_heads": 8, "head_dim": 128,
         "rotary_dim": 128, "layout": "half", "axes": 1, "scaling": "yarn", "far": 1000000, "dtype": "bf16", "packed": True, "inverse": False},
        # prompts: query and key heads are views of one projection's output
        {"name": "rotary prompt", "op": "rotary", "batch": 4, "tokens": 8192, "heads": 32, "kv_heads": 8, "head_dim": 128,
         "rotary_dim": 128, "layout": "half", "axes": 1, "scaling": "none", "far": 0, "dtype": "bf16", "packed": True, "inverse": False},
        # the gradient for image tokens: rows and columns as two axes, three quarters of the head rotated
        {"name": "rotary image gradient", "op": "rotary", "batch": 256, "tokens": 256, "heads": 4, "kv_heads": 4, "head_dim": 64,
         "rotary_dim": 48, "layout": "interleaved", "axes": 2, "scaling": "none", "far": 0, "dtype": "fp32", "packed": False, "inverse": True},
        # one token through a large block: the weights' bandwidth
        {"name": "ffn token", "op": "ffn", "rows": 1, "width": 4096, "hidden": 11008, "dtype": "bf16", "activation": "silu", "bias": False, "train": False},
        # a decode batch
        {"name": "ffn decode batch", "op": "ffn", "rows": 48, "width": 2048, "hidden": 5504, "dtype": "fp16", "activation": "gelu", "bias": True, "train": False},
        # image tokens of the widened model in the framework's own type, a training step
        {"name": "ffn train image tokens", "op": "ffn", "rows": 65536, "width": 256, "hidden": 1024, "dtype": "fp32", "activation": "gelu_tanh", "bias": True, "train": True},
        # a ragged training batch at sizes that no tile divides
        {"name": "ffn train ragged", "op": "ffn", "rows": 1999, "width": 1001, "hidden": 2731, "dtype": "bf16", "activation": "silu", "bias": True, "train": True},
        # a training step of a large block
        {"name": "ffn train wide", "op": "ffn", "rows": 8192, "width": 4096, "hidden": 11008, "dtype": "bf16", "activation": "silu", "bias": False, "train": True},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "rotary", "ffn", "ffn"])
    dtype = rng.choice(["fp32", "bf16", "bf16", "fp16"])
    if op == "norm":
        width = _log(rng, 32, 16384)
        rows = _log(rng, 1, max(1, min(262144, (1 << 27) // width)))
        return {"op": "norm", "rows": rows, "width": width, "dtype": dtype,
                "affine": rng.choice(["same", "fp32", "none"]), "train": rng.random() < 0.5}
    if op == "rotary":
        head_dim = rng.choice([32, 48, 64, 80, 96, 128, 256])
        axes = rng.choice([1, 1, 2])
        rotary_dim = rng.choice([head_dim, head_dim // 2 // (2 * axes) * (2 * axes)])
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 4])
        tokens = 1 if rng.random() < 0.3 else _log(rng, 2, 16384)
        batch = _log(rng, 1, max(1, min(256, (1 << 27) // (tokens * (heads + kv_heads) * head_dim))))
        return {"op": "rotary", "batch": batch, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
                "rotary_dim": rotary_dim, "layout": rng.choice(["half", "interleaved"]), "axes": axes,
                "scaling": rng.choice(["none", "linear", "ntk", "yarn"]), "far": rng.choice([0, 0, 100000, 1000000]), "dtype": dtype,
                "packed": rng.random() < 0.5, "inverse": rng.random() < 0.3}
    train = rng.random() < 0.5
    width = _log(rng, 64, 4096)
    hidden = _log(rng, width, min(11008, 4 * width))
    if rng.random() < 0.6:  # most models' widths fill whole vectors
        width, hidden = (width + 31) // 32 * 32, (hidden + 31) // 32 * 32
    rows = _log(rng, 1, max(1, min(65536, 8192 * 4096 * 11008 // (4 if dtype == "fp32" else 1) // (width * hidden))))
    return {"op": "ffn", "rows": rows, "width": width, "hidden": hidden, "dtype": dtype,
            "activation": rng.choice(["silu", "gelu", "gelu_tanh", "relu", "sigmoid"]), "bias": rng.random() < 0.5, "train": train}


def _frequencies(case):
    """Angle per position of each pair, 64 bits, and the factor on the rotated values (base 10000, trained to 8192 positions,
    stretched by 16 where scaled). With two axes each half of the pairs has the whole range of frequencies."""
    pairs = case["rotary_dim"] // 2 // case["axes"]
    base, factor, trained = 10000.0, 16.0, 8192
    i = torch.arange(pairs, dtype=torch.float64)
    span = max(1, pairs)
    scale = 1.0
    if case["scaling"] == "ntk":
        base = base * factor ** (span / max(1, span - 1))
    inv = base ** (-i / span)
    if case["scaling"] == "linear":
        inv = inv / factor
    if case["scaling"] == "yarn":
        turn = lambda n: span * math.log(trained / (n * 2 * math.pi)) / math.log(base)  # noqa: E731
        low, high = max(math.floor(turn(32.0)), 0), min(math.ceil(turn(1.0)), span - 1)
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        inv = inv / factor * ramp + inv * (1 - ramp)
        scale = 0.1 * math.log(factor) + 1.0
    return inv.repeat(case["axes"]), scale


def prepare(case, seed):
    dt = DTYPES[case["dtype"]]
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    if case["op"] == "norm":
        n, c = case["rows"], case["width"]
        st = {"case": case, "x": (rand(n, c) * 1.5 + 0.3 * rand(c)).to(dt), "weight": None, "bias": None, "eps": 1e-5}
        if case["affine"] != "none":
            wt = torch.float32 if case["affine"] == "fp32" else dt
            st["weight"], st["bias"] = (1 + 0.1 * rand(c)).to(wt), (0.1 * rand(c)).to(wt)
        if case["train"]:
            st["grad"] = rand(n, c).to(dt)
        return st
    if case["op"] == "rotary":
        b, t, h, k, d = case["batch"], case["tokens"], case["heads"], case["kv_heads"], case["head_dim"]
        if case["packed"]:
            qkv = rand(b, t, (h + 2 * k) * d).to(dt)
            q, kk = qkv[..., : h * d].unflatten(-1, (h, d)), qkv[..., h * d: (h + k) * d].unflatten(-1, (k, d))
        else:
            q, kk = rand(b, t, h, d).to(dt), rand(b, t, k, d).to(dt)
        at = torch.arange(t, device="cuda")
        begin = torch.randint(0, case["far"] + 1, (b, 1), device="cuda", generator=g)
        if case["axes"] == 1:
            pos = begin + at
        else:
            side = math.isqrt(t - 1) + 1
            pos = torch.stack([begin + at // side, begin + at % side])
        inv, scale = _frequencies(case)
        return {"case": case, "q": q, "k": kk, "positions": pos, "inv_freq": inv.cuda(), "scale": scale}
    n, d, f = case["rows"], case["width"], case["hidden"]
    st = {"case": case, "x": rand(n, d).to(dt), "w_gate": (rand(f, d) / d ** 0.5).to(dt), "w_up": (rand(f, d) / d ** 0.5).to(dt),
          "w_down": (rand(d, f) / f ** 0.5).to(dt), "b_gate": None, "b_up": None, "b_down": None}
    if case["bias"]:
        st.update(b_gate=(0.1 * rand(f)).to(dt), b_up=(0.1 * rand(f)).to(dt), b_down=(0.1 * rand(d)).to(dt))
    if case["train"]:
        st["grad"] = rand(n, d).to(dt)
    return st


# ---------------------------------------------------------------- plain forms, 32 bits

def _plain_norm(st):
    x, dt = st["x"].float(), st["x"].dtype
    mean = x.mean(-1, keepdim=True)
    xc = x - mean
    rstd = (xc.square().mean(-1, keepdim=True) + st["eps"]).rsqrt()
    xh = xc * rstd
    y = xh
    if st["weight"] is not None:
        y = xh * st["weight"].float() + st["bias"].float()
    if not st["case"]["train"]:
        return {"y": y.to(dt)}
    g = st["grad"].float()
    gw = g if st["weight"] is None else g * st["weight"].float()
    dx = rstd * (gw - gw.mean(-1, keepdim=True) - xh * (gw * xh).mean(-1, keepdim=True))
    res = {"y": y.to(dt), "dx": dx.to(dt)}
    if st["weight"] is not None:
        res["dweight"], res["dbias"] = (g * xh).sum(0).to(st["weight"].dtype), g.sum(0).to(st["bias"].dtype)
    return res


def _plain_rotary(st):
    c = st["case"]
    rd, pairs = c["rotary_dim"], c["rotary_dim"] // 2
    pos = st["positions"].double()
    if c["axes"] == 1:
        ang = pos[..., None] * st["inv_freq"]
    else:
        ang = pos.repeat_interleave(pairs // c["axes"], 0).movedim(0, -1) * st["inv_freq"]
    cos, sin = (ang.cos() * st["scale"]).float()[:, :, None], (ang.sin() * st["scale"]).float()[:, :, None]
    if c["inverse"]:
        sin = -sin

    def turned(x):
        v = x[..., :rd].float()
        a, b = (v[..., :pairs], v[..., pairs:]) if c["layout"] == "half" else (v[..., 0::2], v[..., 1::2])
        ra, rb = a * cos - b * sin, a * sin + b * cos
        r = torch.cat([ra, rb], -1) if c["layout"] == "half" else torch.stack([ra, rb], -1).flatten(-2)
        return torch.cat([r.to(x.dtype), x[..., rd:]], -1)

    return {"q": turned(st["q"]), "k": turned(st["k"])}


def _act(name, v):
    """The activation of v and its derivative."""
    if name == "relu":
        return v.clamp_min(0), (v > 0).to(v.dtype)
    if name == "gelu":
        cdf = 0.5 * (1 + torch.erf(v * 0.5 ** 0.5))
        return v * cdf, cdf + v * torch.exp(-0.5 * v * v) * (0.5 / math.pi) ** 0.5
    if name == "gelu_tanh":
        k = (2 / math.pi) ** 0.5
        t = torch.tanh(k * (v + 0.044715 * v * v * v))
        return 0.5 * v * (1 + t), 0.5 * (1 + t) + 0.5 * v * (1 - t * t) * k * (1 + 3 * 0.044715 * v * v)
    s = 1 / (1 + torch.exp(-v))
    return (s, s * (1 - s)) if name == "sigmoid" else (v * s, s * (1 + v * (1 - s)))


def _plain_ffn(st):
    c, dt = st["case"], st["x"].dtype
    x, wg, wu, wd = (st[k].float() for k in ("x", "w_gate", "w_up", "w_down"))
    g, u = x @ wg.T, x @ wu.T
    if c["bias"]:
        g, u = g + st["b_gate"].float(), u + st["b_up"].float()
    a, da = _act(c["activation"], g)
    h = a * u
    y = h @ wd.T
    if c["bias"]:
        y = y + st["b_down"].float()
    if not c["train"]:
        return {"y": y.to(dt)}
    dy = st["grad"].float()
    dh = dy @ wd
    dg, du = dh * u * da, dh * a
    res = {"y": y, "dx": dg @ wg + du @ wu, "dw_gate": dg.T @ x, "dw_up": du.T @ x, "dw_down": dy.T @ h}
    if c["bias"]:
        res.update(db_gate=dg.sum(0), db_up=du.sum(0), db_down=dy.sum(0))
    return {k: v.to(dt) for k, v in res.items()}


# ---------------------------------------------------------------- the framework's operators

def _own_norm(st):
    import diffusion_model_amd as d
    if not st["case"]["train"]:
        return {"y": d.layer_norm(st["x"], st["weight"], st["bias"], eps=st["eps"])}
    y, mean, rstd = d.layer_norm(st["x"], st["weight"], st["bias"], eps=st["eps"], return_stats=True)
    dx, dw, db = d.layer_norm_backward(st["grad"], st["x"], st["weight"], mean, rstd)
    res = {"y": y, "dx": dx}
    if st["weight"] is not None:
        res["dweight"], res["dbias"] = dw, db
    return res


def _own_rotary(st):
    import diffusion_model_amd as d
    c = st["case"]
    q, k = d.apply_rotary(st["q"], st["k"], st["inv_freq"], st["positions"], layout=c["layout"], scale=st["scale"], inverse=c["inverse"])
    return {"q": q, "k": k}


def _own_ffn(st):
    import diffusion_model_amd as d
    c = st["case"]
    w = (st["w_gate"], st["w_up"], st["w_down"])
    biases = {k: st[k] for k in ("b_gate", "b_up", "b_down")}
    if not c["train"]:
        return {"y": d.gated_ffn(st["x"], *w, **biases, activation=c["activation"])}
    y, saved = d.gated_ffn(st["x"], *w, **biases, activation=c["activation"], save=True)
    grads = d.gated_ffn_backward(st["grad"], st["x"], *w, saved, activation=c["activation"], bias=c["bias"])
    names = ("dx", "dw_gate", "dw_up", "dw_down") + (("db_gate", "db_up", "db_down") if c["bias"] else ())
    return {"y": y, **dict(zip(names, grads))}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": _own_norm, "rotary": _own_rotary, "ffn": _own_ffn}[op](state)
    return {"norm": _plain_norm, "rotary": _plain_rotary, "ffn": _plain_ffn}[op](state)


def work(case):
    s = SIZEOF[case["dtype"]]
    if case["op"] == "norm":
        n, c = case["rows"], case["width"]
        p = {"same": s, "fp32": 4, "none": 0}[case["affine"]] * 2 * c
        if not case["train"]:
            return {"bytes": 2 * n * c * s + p, "flops": 7 * n * c}
        # x and the output's gradient in; y, dx and the parameters' gradients out
        return {"bytes": 4 * n * c * s + 2 * p, "flops": 20 * n * c}
    if case["op"] == "rotary":
        rows = case["batch"] * case["tokens"]
        vals = rows * (case["heads"] + case["kv_heads"])
        return {"bytes": 2 * vals * case["head_dim"] * s + rows * case["axes"] * 8 + case["rotary_dim"] * 4, "flops": 3 * vals * case["rotary_dim"]}
    n, d, f = case["rows"], case["width"], case["hidden"]
    w, b = 3 * d * f * s, (2 * f + d) * s if case["bias"] else 0
    if not case["train"]:
        return {"bytes": 2 * n * d * s + w + b, "flops": 6 * n * d * f}
    return {"bytes": 4 * n * d * s + 2 * w + 2 * b, "flops": 18 * n * d * f}


# ---------------------------------------------------------------- the definitions in 64 bits

def exact(case, seed):
    st = prepare(case, seed)
    st = {k: v.double() if torch.is_tensor(v) and v.is_floating_point() else v for k, v in st.items()}
    if case["op"] == "norm":
        x, n = st["x"], case["width"]
        mu = x.sum(1, keepdim=True) / n
        sd = (((x - mu) ** 2).sum(1, keepdim=True) / n + st["eps"]).sqrt()
        z = (x - mu) / sd
        w = st["weight"] if st["weight"] is not None else torch.ones(n, dtype=torch.float64, device=x.device)
        y = z * w + (st["bias"] if st["bias"] is not None else 0)
        if not case["train"]:
            return {"y": y}
        gz = st["grad"] * w  # gradient of the normalised row; its projection on (1, z) is what normalising takes out
        res = {"y": y, "dx": (gz - gz.sum(1, keepdim=True) / n - z * ((gz * z).sum(1, keepdim=True) / n)) / sd}
        if st["weight"] is not None:
            res.update(dweight=torch.einsum("nc,nc->c", st["grad"], z), dbias=st["grad"].sum(0))
        return res
    if case["op"] == "rotary":
        rd, half = case["rotary_dim"], case["layout"] == "half"
        pos = st["positions"].double().reshape(case["axes"], case["batch"], case["tokens"])
        per = rd // 2 // case["axes"]
        sign = -1.0 if case["inverse"] else 1.0
        res = {}
        for name in ("q", "k"):
            out = st[name].clone()
            for i in range(rd // 2):
                a, b = (i, i + rd // 2) if half else (2 * i, 2 * i + 1)
                turn = torch.polar(torch.full_like(pos[0], st["scale"]), sign * pos[i // per] * st["inv_freq"][i])
                z = torch.complex(st[name][..., a], st[name][..., b]) * turn[:, :, None]
                out[..., a], out[..., b] = z.real, z.imag
            res[name] = out
        return res
    x, wg, wu, wd = st["x"], st["w_gate"], st["w_up"], st["w_down"]
    bg, bu, bd = (st[k] if case["bias"] else 0.0 for k in ("b_gate", "b_up", "b_down"))
    gate, up = x.mm(wg.t()) + bg, x.mm(wu.t()) + bu
    name = case["activation"]
    if name == "relu":
        value, slope = torch.where(gate > 0, gate, 0.0), torch.where(gate > 0, 1.0, 0.0)
    elif name == "gelu":
        phi = torch.special.ndtr(gate)
        value, slope = gate * phi, phi + gate * torch.exp(-gate ** 2 / 2) / math.sqrt(2 * math.pi)
    elif name == "gelu_tanh":
        inner = math.sqrt(2 / math.pi) * (gate + 0.044715 * gate ** 3)
        sech2 = 1 / torch.cosh(inner) ** 2
        value = gate / 2 * (1 + torch.tanh(inner))
        slope = (1 + torch.tanh(inner)) / 2 + gate / 2 * sech2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * gate ** 2)
    else:
        sig = torch.sigmoid(gate)
        value, slope = (sig, sig * torch.sigmoid(-gate)) if name == "sigmoid" else (gate * sig, sig + gate * sig * torch.sigmoid(-gate))
    y = (value * up).mm(wd.t()) + bd
    if not case["train"]:
        return {"y": y}
    dy = st["grad"]
    dhid = dy.mm(wd)
    dgate, dup = dhid * up * slope, dhid * value
    res = {"y": y, "dx": dgate.mm(wg) + dup.mm(wu), "dw_gate": dgate.t().mm(x), "dw_up": dup.t().mm(x), "dw_down": dy.t().mm(value * up)}
    if case["bias"]:
        ones = torch.ones(1, x.shape[0], dtype=torch.float64, device=x.device)
        res.update(db_gate=ones.mm(dgate)[0], db_up=ones.mm(dup)[0], db_down=ones.mm(dy)[0])
    return res
