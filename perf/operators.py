"""What is timed of the operators for per-pixel and per-token networks: the root-mean-square norm with its residual, the product
with a fused epilogue, and the AdamW step.  `own` chooses between the plain form (elementary torch operations) and the kernels."""
import math

import torch

own = False

BLOCK = 256                      # values that share one scale of an 8-bit optimizer state
HYPER = {"lr": 2e-4, "beta1": 0.9, "beta2": 0.999, "eps": 1e-8, "weight_decay": 0.01, "step": 100, "seed": 0x5EED}
EPS = 1e-6
E4M3_MAX = 448.0
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
ACTS = ("none", "relu", "lrelu", "gelu", "silu")


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # a single feed-forward layer's five tensors: the launch itself
        {"name": "step32_layer", "op": "adamw", "bits": 32, "dtype": "f32", "layers": 1, "width": 64},
        # 350 tensors with 3.3 M values in all, as many as the large rescaling network has; odd sizes
        {"name": "step32_net", "op": "adamw", "bits": 32, "dtype": "f32", "layers": 70, "width": 77},
        {"name": "step8_net", "op": "adamw", "bits": 8, "dtype": "f32", "layers": 70, "width": 77},
        # 134 M values in 20 tensors: memory traffic alone
        {"name": "step32_wide", "op": "adamw", "bits": 32, "dtype": "f32", "layers": 4, "width": 2048},
        {"name": "step8_wide", "op": "adamw", "bits": 8, "dtype": "bf16", "layers": 4, "width": 2048},
        # a few new tokens in front of an 8-bit product
        {"name": "norm_q8_rows", "op": "norm", "kind": "q8", "dtype": "bf16", "rows": 8, "cols": 4096, "residual": True},
        # every pixel of four septuplets' latents (28 x 64 x 112) over the conditioner's 64 channels, trained
        {"name": "norm_train_pixels", "op": "norm", "kind": "train", "dtype": "f16", "rows": 200704, "cols": 64, "residual": True},
        # long rows, trained
        {"name": "norm_train_rows", "op": "norm", "kind": "train", "dtype": "bf16", "rows": 8192, "cols": 4096, "residual": True},
        # one new token through a wide layer: the weights are read once
        {"name": "product_one", "op": "product", "kind": "forward", "dtype": "bf16", "rows": 1, "k": 4096, "n": 4096, "act": "silu", "residual": True},
        # the 36 x 36 latents of eight 144 x 144 training septuplets, 51 channels in, 204 out: nothing is a multiple of 8 but the pixels
        {"name": "product_train_pixels", "op": "product", "kind": "train", "dtype": "f16", "rows": 72576, "k": 51, "n": 204, "act": "lrelu", "residual": False},
        # a wide layer, trained
        {"name": "product_train", "op": "product", "kind": "train", "dtype": "bf16", "rows": 8192, "k": 2048, "n": 8192, "act": "gelu", "residual": False},
        # the layer that leads back into the stream of rows, served in 8 bits
        {"name": "product_q8", "op": "product", "kind": "q8", "dtype": "bf16", "rows": 4096, "k": 8192, "n": 2048, "act": "none", "residual": True},
    ]


def _between(rng, lo, hi):
    """A whole number spread over the logarithm of lo..hi; as often a multiple of 16 as not."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if v >= 32 and rng.random() < 0.5:
        v -= v % 16
    return v


def draw(rng):
    op = rng.choice(("adamw", "adamw", "norm", "product", "product"))
    if op == "adamw":
        layers = _between(rng, 1, 70)
        width = _between(rng, 16, 2048)
        while layers * width * width > 4 * 2048 * 2048:
            layers, width = max(1, layers // 2), max(16, int(width / 1.3))
        return {"op": op, "bits": rng.choice((8, 32)), "dtype": rng.choice(("f32", "bf16")), "layers": layers, "width": width}
    if op == "norm":
        cols = _between(rng, 3, 8192)
        rows = _between(rng, 1, 200704)
        rows = max(1, min(rows, 8192 * 4096 // cols))
        return {"op": op, "kind": rng.choice(("q8", "train")), "dtype": rng.choice(("bf16", "f16")), "rows": rows, "cols": cols,
                "residual": rng.random() < 0.7}
    kind = rng.choice(("forward", "train", "q8"))
    rows, k, n = _between(rng, 1, 72576), _between(rng, 16, 8192), _between(rng, 16, 8192)
    while rows * k * n > 8192 * 2048 * 8192:
        rows, k, n = max(1, int(rows / 1.5)), max(16, int(k / 1.2)), max(16, int(n / 1.2))
    return {"op": op, "kind": kind, "dtype": rng.choice(("bf16", "f16")), "rows": rows, "k": k, "n": n, "act": rng.choice(ACTS),
            "residual": rng.random() < 0.5}


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _sizes(case):
    """The tensors of `layers` feed-forward layers: both weights, both biases and the norm's weight."""
    w = case["width"]
    return [n for _ in range(case["layers"]) for n in (w, 4 * w * w, 4 * w, 4 * w * w, w)]


def _padded(n):
    return -(-n // BLOCK) * BLOCK


def _prepare_adamw(case, gen, dev):
    sizes, dt = _sizes(case), TYPES[case["dtype"]]
    total, padded = sum(sizes), [_padded(n) for n in sizes]
    f = lambda scale: torch.randn(total, generator=gen, device=dev).mul_(scale)  # noqa: E731
    state = {"params": [t.clone() for t in f(0.02).to(dt).split(sizes)], "grads": [t.clone() for t in f(1e-3).to(dt).split(sizes)]}
    inside = torch.cat([torch.arange(p, device=dev) < n for n, p in zip(sizes, padded)])
    m = torch.randn(sum(padded), generator=gen, device=dev).mul_(3e-4).mul_(inside)
    v = torch.randn(sum(padded), generator=gen, device=dev).mul_(0.5).exp_().mul_(1e-6).mul_(inside)
    if case["bits"] == 8:
        def held(x, top, kind):      # the block's largest value lies in [2^top, 2^(top + 1)) steps of its scale
            x = x.view(-1, BLOCK)
            s = torch.ldexp(torch.ones_like(x[:, 0]), torch.frexp(x.abs().amax(1)).exponent - 1 - top)
            return (x / s[:, None]).to(kind).view(-1), s
        m, state["m_scale"] = held(m, 7, torch.float8_e4m3fn)
        v, state["v_scale"] = held(v, 14, torch.float8_e5m2)
    state.update(m=m, v=v, inside=inside.nonzero().view(-1), sizes=sizes)
    return state


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device()) if torch.cuda.is_available() else torch.device("cpu")
    gen = torch.Generator(device=dev).manual_seed(seed)
    if case["op"] == "adamw":
        return {"case": case, **_prepare_adamw(case, gen, dev)}
    dt = TYPES[case["dtype"]]
    f = lambda *s, scale=1.0: torch.randn(*s, generator=gen, device=dev).mul_(scale).to(dt)  # noqa: E731
    st = {"case": case}
    if case["op"] == "norm":
        rows, cols = case["rows"], case["cols"]
        st["x"], st["weight"] = f(rows, cols), f(cols, scale=0.2) + 1
        if case["residual"]:
            st["residual"] = f(rows, cols)
        if case["kind"] == "train":
            st["dy"] = f(rows, cols)
            if case["residual"]:
                st["dh"] = f(rows, cols)
            st["x"].requires_grad_(True)
            st["weight"].requires_grad_(True)
        return st
    rows, k, n = case["rows"], case["k"], case["n"]
    st["bias"] = f(n, scale=0.5)
    if case["residual"]:
        st["residual"] = f(rows, n)
    if case["kind"] == "q8":
        for name, r in (("x", rows), ("weight", n)):
            t = torch.randn(r, k, generator=gen, device=dev).mul_(1.0 if name == "x" else k ** -0.5)
            st[name + "_scale"] = t.abs().amax(1) / E4M3_MAX
            st[name] = (t / st[name + "_scale"][:, None]).to(torch.float8_e4m3fn)
        return st
    st["x"], st["weight"] = f(rows, k), f(n, k, scale=k ** -0.5)
    if case["kind"] == "train":
        st["dy"] = f(rows, n)
        for name in ("x", "weight", "bias"):
            st[name].requires_grad_(True)
    return st


def work(case):
    b = BYTES[case["dtype"]]
    if case["op"] == "adamw":
        n = sum(_sizes(case))
        return {"bytes": n * (3 * b + (16 if case["bits"] == 32 else 4 + 16 / BLOCK)), "flops": 16 * n}
    r = case["residual"]
    if case["op"] == "norm":
        rows, cols = case["rows"], case["cols"]
        if case["kind"] == "q8":
            return {"bytes": rows * cols * (b * (1 + 2 * r) + 1) + 4 * rows + cols * b, "flops": 6 * rows * cols}
        return {"bytes": rows * cols * b * (4 + 3 * r) + 2 * cols * b, "flops": 16 * rows * cols}
    rows, k, n = case["rows"], case["k"], case["n"]
    if case["kind"] == "q8":
        return {"bytes": (rows + n) * (k + 4) + rows * n * b * (1 + r) + n * b, "flops": 2 * rows * k * n}
    once = (rows * k + n * k + n + rows * n * (1 + r)) * b
    if case["kind"] == "forward":
        return {"bytes": once, "flops": 2 * rows * k * n}
    return {"bytes": once + (rows * n + rows * k + n * k + n) * b, "flops": 6 * rows * k * n}


# ---------------------------------------------------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------------------------------------------------
def _mix(x):
    """The dither's integer mixing of 32-bit numbers held in int64."""
    for shift, mul in ((16, 0x85A308D3), (15, 0x13198A2F)):
        x = x ^ (x >> shift)
        low = (mul & 0xFFFF) * x
        x = (low + ((((mul >> 16) * x) & 0xFFFF) << 16)) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _mix_int(x):
    return int(_mix(torch.tensor([x & 0xFFFFFFFF], dtype=torch.int64)))


def _dither(sizes, dev):
    """Two numbers in [0, 1) for each value of the padded layout: from the seed, the step, the tensor's place and the value's."""
    key = _mix_int(HYPER["seed"] ^ _mix_int(HYPER["step"]))
    place = torch.arange(len(sizes), device=dev)
    keys = _mix(key ^ _mix(place))
    padded = torch.tensor([_padded(n) for n in sizes], device=dev)
    starts = padded.cumsum(0) - padded
    owner = torch.repeat_interleave(place, padded)
    x = _mix((torch.arange(owner.numel(), device=dev) - starts[owner]) ^ keys[owner])
    return (x & 0xFFFF).float() / 65536, (x >> 16).float() / 65536


def _hold(x, u, top, least, digits, floor):
    """x in 8 bits: a power of two per block, and the value of x over it rounded down after adding u steps."""
    x = x.view(-1, BLOCK)
    most = x.abs().amax(1)
    s = torch.ldexp(torch.ones_like(most), (torch.frexp(most).exponent - 1 - top).clamp_(min=-126))
    s = torch.where(most > 0, s, torch.ones_like(s))
    y = x / s[:, None]
    q = torch.ldexp(torch.ones_like(y), (torch.frexp(y).exponent - 1).clamp_(min=least) - digits)
    k = torch.floor(y.abs() / q + u.view(-1, BLOCK))
    if floor:
        k = torch.where(y > 0, k.clamp(min=1), k)
    return (k * q * y.sign()).view(-1), s


def _plain_adamw(st):
    c, h = st["case"], HYPER
    dt, inside = TYPES[c["dtype"]], st["inside"]
    p = torch.cat([t.view(-1) for t in st["params"]]).float()
    g = torch.cat([t.view(-1) for t in st["grads"]]).float()
    m, v = st["m"], st["v"]
    if c["bits"] == 8:
        m = (m.float().view(-1, BLOCK) * st["m_scale"][:, None]).view(-1)
        v = (v.float().view(-1, BLOCK) * st["v_scale"][:, None]).view(-1)
    wide = torch.zeros_like(m)
    wide[inside] = g
    m = h["beta1"] * m + (1 - h["beta1"]) * wide
    v = h["beta2"] * v + (1 - h["beta2"]) * (wide * wide)
    den = v[inside].sqrt() / math.sqrt(1 - h["beta2"] ** h["step"]) + h["eps"]
    p = p * (1 - h["lr"] * h["weight_decay"]) - h["lr"] / (1 - h["beta1"] ** h["step"]) * (m[inside] / den)
    torch._foreach_copy_(st["params"], list(p.to(dt).split(st["sizes"])))
    if c["bits"] == 8:
        um, uv = _dither(st["sizes"], m.device)
        m, s = _hold(m, um, 7, -6, 3, False)
        st["m_scale"].copy_(s)
        v, s = _hold(v, uv, 14, -14, 2, True)
        st["v_scale"].copy_(s)
    st["m"].copy_(m.to(st["m"].dtype))
    st["v"].copy_(v.to(st["v"].dtype))
    return _adamw_outputs(st)


def _adamw_outputs(st):
    """All that the step updates: the tensors (joined where they are many) and the state."""
    held = {k: st[k] for k in ("m", "v", "m_scale", "v_scale") if k in st}
    return {"params": st["params"] if len(st["params"]) <= 50 else torch.cat([t.view(-1) for t in st["params"]]), **held}


def _plain_norm(st):
    c, dt = st["case"], TYPES[st["case"]["dtype"]]
    x, w = st["x"].detach(), st["weight"].detach().float()
    out = {}
    if c["residual"]:
        x = out["h"] = (x.float() + st["residual"].float()).to(dt)       # the sum is an output; the norm is that of the output
    x = x.float()
    r = torch.rsqrt((x * x).mean(1, keepdim=True) + EPS)
    n = x * r
    y = n * w
    if c["kind"] == "q8":
        out["scale"] = y.abs().amax(1) / E4M3_MAX
        out["q"] = (y / out["scale"][:, None]).to(torch.float8_e4m3fn)
        return out
    out["y"] = y.to(dt)
    dy = st["dy"].float()
    dn = dy * w
    dx = r * (dn - n * (dn * n).mean(1, keepdim=True))
    if c["residual"]:
        dx = dx + st["dh"].float()
    out["dx"], out["dw"] = dx.to(dt), (dy * n).sum(0).to(dt)
    return out


def _act(z, act):
    """The activation's value and derivative."""
    if act == "none":
        return z, torch.ones_like(z)
    if act in ("relu", "lrelu"):
        d = torch.where(z > 0, 1.0, 0.0 if act == "relu" else 0.2).to(z.dtype)
        return z * d, d
    if act == "gelu":
        phi = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * phi, phi + z * torch.exp(-0.5 * z * z) * math.sqrt(0.5 / math.pi)
    s = torch.sigmoid(z)
    return z * s, s * (1 + z * (1 - s))


def _plain_product(st):
    c, dt = st["case"], TYPES[st["case"]["dtype"]]
    x, w = st["x"].detach().float(), st["weight"].detach().float()
    if c["kind"] == "q8":
        z = (x @ w.t()) * st["x_scale"][:, None] * st["weight_scale"]
    else:
        z = x @ w.t()
    y, d = _act(z + st["bias"].detach().float(), c["act"])
    if c["residual"]:
        y = y + st["residual"].float()
    out = {"y": y.to(dt)}
    if c["kind"] == "train":
        dz = st["dy"].float() * d
        out.update(dx=(dz @ w).to(dt), dw=(dz.t() @ x).to(dt), db=dz.sum(0).to(dt))
    return out


# ---------------------------------------------------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------------------------------------------------
def _own(st):
    c = st["case"]
    if c["op"] == "adamw":
        from selfc_amd import optim
        optim.adamw_step(st["params"], st["grads"], st["m"], st["v"], st.get("m_scale"), st.get("v_scale"), **HYPER)
        return _adamw_outputs(st)
    from selfc_amd import pointwise as pw
    if c["op"] == "norm":
        if c["kind"] == "q8":
            q, scale, h = pw.rms_norm_q8(st["x"], st["weight"], residual=st.get("residual"), eps=EPS)
            return {"q": q, "scale": scale, **({"h": h} if c["residual"] else {})}
        y, h = pw.rms_norm(st["x"], st["weight"], residual=st.get("residual"), eps=EPS)
        if not c["residual"]:
            dx, dw = torch.autograd.grad(y, (st["x"], st["weight"]), st["dy"])
            return {"y": y, "dx": dx, "dw": dw}
        dx, dw = torch.autograd.grad((y, h), (st["x"], st["weight"]), (st["dy"], st["dh"]))
        return {"y": y, "h": h, "dx": dx, "dw": dw}
    if c["kind"] == "q8":
        return {"y": pw.linear_q8(st["x"], st["x_scale"], st["weight"], st["weight_scale"], bias=st["bias"], act=c["act"],
                                  residual=st.get("residual"), out_dtype=TYPES[c["dtype"]])}
    y = pw.linear(st["x"], st["weight"], bias=st["bias"], act=c["act"], residual=st.get("residual"))
    if c["kind"] == "forward":
        return {"y": y}
    dx, dw, db = torch.autograd.grad(y, (st["x"], st["weight"], st["bias"]), st["dy"])
    return {"y": y, "dx": dx, "dw": dw, "db": db}


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return {"adamw": _plain_adamw, "norm": _plain_norm, "product": _plain_product}[state["case"]["op"]](state)


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def _exact_round(x, u, top, least, digits, floor):
    """What _hold does, from the definition: the two neighbours in 8 bits, and the upper one where the rest and u reach a step."""
    x = x.reshape(-1, BLOCK)
    most = x.abs().max(dim=1).values
    expo = torch.floor(torch.log2(most.clamp(min=2.0 ** -149)))
    expo = expo + (2.0 ** (expo + 1) <= most).double() - (2.0 ** expo > most).double()       # log2 next to a power of two
    s = torch.where(most > 0, 2.0 ** (expo - top).clamp(min=-126), torch.ones_like(most))
    y = x.abs() / s[:, None]
    e = torch.floor(torch.log2(y.clamp(min=2.0 ** -300)))
    e = e + (2.0 ** (e + 1) <= y).double() - (2.0 ** e > y).double()
    step = 2.0 ** (e.clamp(min=least) - digits)
    below = torch.floor(y / step)
    k = below + ((y / step - below) + u.reshape(-1, BLOCK) >= 1).double()
    if floor:
        k = torch.where((y > 0) & (k == 0), torch.ones_like(k), k)
    return (k * step * torch.sign(x)).reshape(-1), s


def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "adamw":
            b1, b2, t, lr = HYPER["beta1"], HYPER["beta2"], HYPER["step"], HYPER["lr"]
            ms, vs, out_p, out_m, out_v = st["m"].double(), st["v"].double(), [], [], []
            if case["bits"] == 8:
                ms = ms * st["m_scale"].double().repeat_interleave(BLOCK)
                vs = vs * st["v_scale"].double().repeat_interleave(BLOCK)
            at = 0
            for p, g in zip(st["params"], st["grads"]):
                n, p, g = p.numel(), p.double(), g.double()
                m, v = ms[at:at + n] * b1 + (1 - b1) * g, vs[at:at + n] * b2 + (1 - b2) * g ** 2
                out_p.append(p * (1 - lr * HYPER["weight_decay"]) - lr * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)) ** 0.5 + HYPER["eps"]))
                zeros = m.new_zeros(_padded(n) - n)
                out_m += [m, zeros]
                out_v += [v, zeros]
                at += _padded(n)
            m, v = torch.cat(out_m), torch.cat(out_v)
            out = {"params": out_p if len(out_p) <= 50 else torch.cat(out_p), "m": m, "v": v}
            if case["bits"] == 8:
                um, uv = _dither(st["sizes"], m.device)
                out["m"], _ = _exact_round(m, um.double(), 7, -6, 3, False)
                out["v"], _ = _exact_round(v, uv.double(), 14, -14, 2, True)
                # a scale is the power of two below the largest of the 32-bit moments: where that is a power of two itself, as moments
                # on a coarse grid often are, its last bit decides, and 64 bits have no say
                out["m_scale"] = out["v_scale"] = None
            return out
        if case["op"] == "norm":
            dt, out = TYPES[case["dtype"]], {}
            h = st["x"].detach().double()
            if case["residual"]:
                out["h"] = h = (h + st["residual"].double()).to(dt).double()
            w = st["weight"].detach().double()
            rms = (h.pow(2).sum(1) / case["cols"] + EPS).sqrt().unsqueeze(1)
            y = h / rms * w
            if case["kind"] == "q8":
                out["scale"] = y.abs().max(dim=1).values / 448
                out["q"] = y / out["scale"].unsqueeze(1)
                return out
            dy = st["dy"].double()
            inner = (dy * w * h).sum(1, keepdim=True)
            dx = dy * w / rms - h * inner / (case["cols"] * rms ** 3)
            out.update(y=y, dx=dx + st["dh"].double() if case["residual"] else dx, dw=(dy * h / rms).sum(0))
            return out
        x, w, b = st["x"].detach().double(), st["weight"].detach().double(), st["bias"].detach().double()
        if case["kind"] == "q8":
            x, w = x * st["x_scale"].double().unsqueeze(1), w * st["weight_scale"].double().unsqueeze(1)
        z = torch.addmm(b, x, w.t())
        if case["act"] == "relu":
            y, d = z.clamp(min=0), (z > 0).double()
        elif case["act"] == "lrelu":
            y, d = torch.maximum(z, 0.2 * z), 0.2 + 0.8 * (z > 0).double()
        elif case["act"] == "gelu":
            cdf = 0.5 * torch.special.erfc(-z / 2 ** 0.5)
            y, d = z * cdf, cdf + z * torch.exp(-z ** 2 / 2) / (2 * math.pi) ** 0.5
        elif case["act"] == "silu":
            s = 1 / (1 + torch.exp(-z))
            y, d = z * s, s + z * s * (1 - s)
        else:
            y, d = z, torch.ones_like(z)
        if case["residual"]:
            y = y + st["residual"].double()
        if case["kind"] != "train":
            return {"y": y}
        dz = st["dy"].double() * d
        return {"y": y, "dx": torch.mm(dz, w), "dw": torch.mm(dz.t().contiguous(), x), "db": dz.sum(0)}
