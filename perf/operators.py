"""The operators between two layers, as measurable cases: block norms (with the
block's gate and residual scale), quantisation to 8-bit floating point in blocks
of 128, products of such blocks, and a linear layer's training step on them.

Sizes come from this repository's configurations, tests and benchmark: hidden
2048, 16 heads of 128 or 256, the fused q/k/v/a/b projection's 6176 or 8224
columns, batches up to 4 x 4096 tokens, with odd and ragged ones beside them.
``run`` computes in plain torch in 32 bits, or, where ``own`` is true, calls the
framework.
"""

import math

import torch

own = False

DEV = "cuda"
BLK = 128
EPS = 1e-6
E4M3, E5M2, E8M0 = torch.float8_e4m3fn, torch.float8_e5m2, torch.float8_e8m0fnu
FORMATS = {"e4m3": E4M3, "e5m2": E5M2}
TOP = {E4M3: 8, E5M2: 15}  # the largest code is 1.75 * 2^TOP


# ---------------------------------------------------------------------------
# The cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # One user's next token between two layers: the block's output joins the
        # residual stream, and the next projection gets its codes.
        dict(name="norm_token", kind="norm", B=1, T=1, H=0, D=2048, types="bf16", residual=True, post=True, pre=True,
             gate="token", act="silu", scale=True, rs=1.0, quant=True),
        # The recurrence's heads of a prompt, normalised and gated before the
        # output projection (no residual; dv = 256).
        dict(name="norm_heads", kind="norm", B=1, T=1500, H=16, D=256, types="bf16", residual=False, post=True, pre=False,
             gate="token", act="silu", scale=False, rs=1.0, quant=False),
        # A full training-sized batch between two layers, one gate a sequence.
        dict(name="norm_batch", kind="norm", B=4, T=4096, H=0, D=2048, types="bf16", residual=True, post=True, pre=True,
             gate="sequence", act="tanh", scale=False, rs=0.5, quant=False),
        # Backward over a small odd batch, all in 32 bits.
        dict(name="norm_backward_odd", kind="norm_backward", B=3, T=111, H=0, D=1001, types="fp32", residual=True,
             post=True, pre=True, gate="channel", act="none", scale=True, rs=1.0),
        # Backward of the training-sized batch with a gate for each token.
        dict(name="norm_backward_batch", kind="norm_backward", B=4, T=4096, H=0, D=2048, types="bf16", residual=True,
             post=True, pre=True, gate="token", act="silu", scale=True, rs=1.0),
        # A prompt's activations on their way into a projection.
        dict(name="quantize_prompt", kind="quantize", M=1500, K=2048, block=1, fmt="e4m3", rows=True, columns=False),
        # A weight matrix, laid out for both directions of training.
        dict(name="quantize_weight", kind="quantize", M=8224, K=2048, block=128, fmt="e4m3", rows=True, columns=True),
        # One user's token through the fused projection: the weights' bytes.
        dict(name="product_token", kind="product", M=1, N=8224, K=2048, a="e4m3", b="e4m3", bscale="e8m0", brows=128,
             out="bf16"),
        # A serving batch, not a round number, through the output projection,
        # weights with 32-bit scales.
        dict(name="product_serving", kind="product", M=48, N=2048, K=4096, a="e4m3", b="e4m3", bscale="fp32", brows=128,
             out="bf16"),
        # A prompt through the fused projection.
        dict(name="product_prompt", kind="product", M=1500, N=8224, K=2048, a="e4m3", b="e4m3", bscale="e8m0", brows=128,
             out="bf16"),
        # The training-sized batch through the fused projection: the largest.
        dict(name="product_batch", kind="product", M=16384, N=6176, K=2048, a="e4m3", b="e4m3", bscale="e8m0", brows=128,
             out="bf16"),
        # Forward and backward of a projection over packed prompts (2683
        # tokens), gradients in the wider-ranged format, weight gradient in fp32.
        dict(name="train_step", kind="train", M=2683, N=2048, K=2048),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "norm_backward", "norm_backward", "quantize", "product", "product", "product", "train"])
    if kind in ("norm", "norm_backward"):
        types = rng.choice(["bf16", "bf16", "bf16", "fp32", "mixed"])
        heads = rng.random() < 0.25
        H = rng.choice([4, 16, 32]) if heads else 0
        D = rng.choice([128, 256]) if heads else rng.choice([2048, 4096, 8 * _log_int(rng, 8, 1024), _log_int(rng, 33, 5000)])
        most = (1 << 25) // (D * max(H, 1))
        T = _log_int(rng, 1, min(8192, most))
        B = _log_int(rng, 1, max(1, min(16, most // T)))
        residual = not heads or rng.random() < 0.3
        pre = rng.random() < 0.75 if residual else False
        post = rng.random() < 0.75 or not (residual or pre)
        gate = rng.choice(["none", "token", "sequence", "channel"]) if not heads else "token"
        case = dict(kind=kind, B=B, T=T, H=H, D=D, types=types, residual=residual, post=post, pre=pre, gate=gate,
                    act=rng.choice(["none", "sigmoid", "silu", "tanh"]) if gate != "none" else "none",
                    scale=rng.random() < 0.5, rs=rng.choice([1.0, 0.25, 0.7071]))
        if kind == "norm":
            case["quant"] = rng.random() < 0.4
        return case
    if kind == "quantize":
        M = _log_int(rng, 1, 16384)
        rows, columns = rng.choice([(True, False), (False, True), (True, True)])
        return dict(kind=kind, M=M, K=_log_int(rng, 16, min(16384, (1 << 25) // M)), block=rng.choice([1, 1, 128]),
                    fmt=rng.choice(["e4m3", "e4m3", "e5m2"]), rows=rows, columns=columns)
    if kind == "product":
        M, N = _log_int(rng, 1, 16384), _log_int(rng, 16, 8224)
        K = BLK * _log_int(rng, 1, max(1, min(64, (1 << 37) // (M * N * BLK))))
        return dict(kind=kind, M=M, N=N, K=K, a=rng.choice(["e4m3", "e4m3", "e5m2"]), b=rng.choice(["e4m3", "e4m3", "e5m2"]),
                    bscale=rng.choice(["e8m0", "e8m0", "fp32"]), brows=rng.choice([128, 128, 1]),
                    out=rng.choice(["bf16", "bf16", "fp32"]))
    M = _log_int(rng, 64, 8192)
    return dict(kind=kind, M=M, N=16 * _log_int(rng, 8, 256), K=16 * _log_int(rng, 8, 256))


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _shape(c):
    return (c["B"], c["T"], c["H"], c["D"]) if c["H"] else (c["B"], c["T"], c["D"])


def _gate_shape(c):
    return {"none": None, "token": _shape(c), "sequence": (c["B"], c["D"]), "channel": (c["D"],)}[c["gate"]]


def _exponents(amax, top):
    """The least e with amax / 2^e <= 1.75 * 2^top (0 where amax is 0)."""
    m, e = torch.frexp(amax)
    e = e - (top + 1) + (m > 0.875).int()
    return torch.where(amax > 0, e.clamp(min=-127), 0)


def _pow2(e):
    """2^e in 32 bits, exactly (a power function may round)."""
    half = torch.div(e, 2, rounding_mode="floor")
    bits = lambda k: ((k + 127) << 23).to(torch.int32).view(torch.float32)  # noqa: E731
    return bits(half) * bits(e - half)


def _quantize_rows(x, block, fmt):
    """Codes [M, Kp] and exponents [M or M / block, Kp / 128] of x [M, K] in fp32, one scale for `block` x 128 values."""
    M, K = x.shape
    KB, MB = -(-K // BLK), -(-M // block)
    p = torch.nn.functional.pad(x, (0, KB * BLK - K, 0, MB * block - M))
    t = p.view(MB, block, KB, BLK)
    e = _exponents(t.abs().amax(dim=(1, 3)), TOP[fmt])
    codes = (t * _pow2(-e)[:, None, :, None]).view(MB * block, KB * BLK)[:M].to(fmt)
    return codes.contiguous(), e


def _values(codes, e, block):
    """What codes and exponents stand for, in 32 bits."""
    M = codes.shape[0]
    s = _pow2(e).repeat_interleave(block, 0)[:M]
    return (codes.float().view(M, -1, BLK) * s[:, :, None]).view(M, -1)


def _e8m0(e):
    return (e + 127).to(torch.uint8).view(E8M0)


def _down_columns(t):
    """[M, KB] as the framework keeps scales: a K block's scales adjacent, columns 16 apart at least."""
    M, KB = t.shape
    whole = t.view(torch.uint8) if t.dtype == E8M0 else t
    buf = torch.zeros(KB, -(-M // 16) * 16, dtype=whole.dtype, device=t.device)
    buf[:, :M] = whole.t()
    return buf.view(t.dtype)[:, :M].t()


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)

    def randn(*shape, dtype=torch.float32, std=1.0, mean=0.0):
        return (torch.randn(shape, generator=g, device=DEV) * std + mean).to(dtype)

    st = {"case": case}
    c = case
    if c["kind"] in ("norm", "norm_backward"):
        T = torch.float32 if c["types"] == "fp32" else torch.bfloat16
        R = torch.bfloat16 if c["types"] == "bf16" else torch.float32
        sh, D = _shape(c), c["D"]
        st["y"] = randn(*sh, dtype=T, std=0.7)
        st["residual"] = randn(*sh, dtype=R, std=2.0) if c["residual"] else None
        gs = _gate_shape(c)
        st["gate"] = randn(*gs, dtype=T) if gs else None
        P = torch.float32 if c["types"] != "bf16" else torch.bfloat16
        for name, there in (("post_gamma", c["post"]), ("gamma", c["pre"]), ("scale", c["scale"])):
            st[name] = randn(D, dtype=P, std=0.1, mean=1.0) if there else None
        if c["kind"] == "norm_backward":
            st["dh"] = randn(*sh, dtype=R if c["residual"] else T)
            st["dn"] = randn(*sh, dtype=T) if c["pre"] else None
            # what the forward pass of a training step keeps: 1 / rms of y and of h, a row
            y, h = _h32(st)
            st["rstd_y"] = torch.rsqrt(y.square().mean(-1) + EPS).reshape(-1) if c["post"] else None
            st["rstd_h"] = torch.rsqrt(h.square().mean(-1) + EPS).reshape(-1) if c["pre"] else None
    elif c["kind"] == "quantize":
        # rows of different magnitude, as activations have them
        st["x"] = (randn(c["M"], c["K"]) * torch.exp(randn(c["M"], 1))).to(torch.bfloat16)
    elif c["kind"] == "product":
        M, N, K = c["M"], c["N"], c["K"]
        a, ea = _quantize_rows(randn(M, K, dtype=torch.bfloat16).float(), 1, FORMATS[c["a"]])
        b, eb = _quantize_rows(randn(N, K, dtype=torch.bfloat16, std=0.02).float(), c["brows"], FORMATS[c["b"]])
        st["a"], st["a_scale"], st["b"] = a, _down_columns(_e8m0(ea)), b
        if c["bscale"] == "fp32":  # scales of a checkpoint, any 32-bit number
            bs = (1.0 + 0.9 * torch.rand(eb.shape, generator=g, device=DEV)) * _pow2(eb)
        else:
            bs = _e8m0(eb)
        st["b_scale"] = _down_columns(bs) if c["brows"] == 1 else bs.contiguous()
    else:
        M, N, K = c["M"], c["N"], c["K"]
        st["x"] = randn(M, K, dtype=torch.bfloat16)
        st["w"] = randn(N, K, dtype=torch.bfloat16, std=0.02)
        st["dy"] = randn(M, N, dtype=torch.bfloat16, std=1e-3)
    if own:
        from gdn_18646_amd import compile_kernels
        st["exts"] = compile_kernels()
    return st


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------
def _act(x, name):
    return {"none": lambda: x, "sigmoid": lambda: torch.sigmoid(x), "silu": lambda: x * torch.sigmoid(x),
            "tanh": lambda: torch.tanh(x)}[name]()


def _act_grad(x, name):
    s = torch.sigmoid(x)
    return {"none": lambda: torch.ones_like(x), "sigmoid": lambda: s * (1 - s), "silu": lambda: s * (1 + x * (1 - s)),
            "tanh": lambda: 1 - torch.tanh(x).square()}[name]()


def _spread(gate, y):
    """The gate over y's rows: its own shape, one a sequence, or one for all."""
    if gate.dim() == 2 and y.dim() > 2:
        return gate.view(gate.shape[0], *([1] * (y.dim() - 2)), gate.shape[1])
    return gate


def _h32(st):
    c = st["case"]
    y = st["y"].float()
    u = y
    if st["post_gamma"] is not None:
        u = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * st["post_gamma"].float()
    f = c["rs"] if st["scale"] is None else c["rs"] * st["scale"].float()
    if st["gate"] is not None:
        f = f * _act(_spread(st["gate"].float(), y), c["act"])
    h = f * u
    if st["residual"] is not None:
        h = st["residual"].float() + h
    return y, h


def _plain_norm(st):
    c = st["case"]
    _, h = _h32(st)
    n = None
    if st["gamma"] is not None:
        n = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * st["gamma"].float()
    hout = h.to(st["residual"].dtype if st["residual"] is not None else st["y"].dtype)
    if not c["quant"]:
        return hout, None if n is None else n.to(st["y"].dtype)
    codes, e = _quantize_rows((h if n is None else n).reshape(-1, c["D"]), 1, E4M3)
    return hout, codes, _e8m0(e)


def _plain_norm_backward(st):
    c = st["case"]
    y, h = _h32(st)
    dh = st["dh"].float()
    if st["gamma"] is not None:
        hn = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS)
        dn = st["dn"].float()
        t = dn * st["gamma"].float()
        dh = dh + torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * (t - hn * (t * hn).mean(-1, keepdim=True))
        dgamma = (dn * hn).reshape(-1, c["D"]).sum(0).to(st["gamma"].dtype)
    else:
        dgamma = None
    rstd, yn = None, y
    if st["post_gamma"] is not None:
        rstd = torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS)
        yn = y * rstd
    pg = 1.0 if st["post_gamma"] is None else st["post_gamma"].float()
    sc = 1.0 if st["scale"] is None else st["scale"].float()
    a = 1.0
    if st["gate"] is not None:
        gate = _spread(st["gate"].float(), y)
        a = _act(gate, c["act"])
    e = dh * yn * c["rs"]  # d / d (scale act(gate) post_gamma)
    dgate = None
    if st["gate"] is not None:
        dgate = e * (pg * sc) * _act_grad(gate, c["act"])
        if c["gate"] == "sequence":
            dgate = dgate.reshape(c["B"], -1, c["D"]).sum(1)
        elif c["gate"] == "channel":
            dgate = dgate.reshape(-1, c["D"]).sum(0)
        dgate = dgate.to(st["gate"].dtype)
    ea = (e * a).reshape(-1, c["D"]).sum(0)
    dpost = (ea * sc).to(st["post_gamma"].dtype) if st["post_gamma"] is not None else None
    dscale = (ea * pg).to(st["scale"].dtype) if st["scale"] is not None else None
    dyn = dh * (c["rs"] * sc * a) * pg
    dy = dyn if rstd is None else rstd * (dyn - yn * (dyn * yn).mean(-1, keepdim=True))
    dres = dh.to(st["residual"].dtype) if st["residual"] is not None else None
    return dres, dy.to(st["y"].dtype), dgate, dpost, dgamma, dscale


def _plain_quantize(st):
    c = st["case"]
    x, out = st["x"].float(), []
    for there, t in ((c["rows"], x), (c["columns"], x.t())):
        if there:
            codes, e = _quantize_rows(t, c["block"], FORMATS[c["fmt"]])
            out += [codes, _e8m0(e)]
    return out


def _plain_product(st):
    c = st["case"]
    a = st["a"].float().view(c["M"], -1, BLK) * st["a_scale"].float()[:, :, None]
    bs = st["b_scale"].float().repeat_interleave(c["brows"], 0)[:c["N"]]
    b = st["b"].float().view(c["N"], -1, BLK) * bs[:, :, None]
    y = a.view(c["M"], -1) @ b.view(c["N"], -1).t()
    return y.to(torch.bfloat16 if c["out"] == "bf16" else torch.float32)


def _plain_train(st):
    x, w, dy = st["x"].float(), st["w"].float(), st["dy"].float()
    K, N = x.shape[1], w.shape[0]
    y = _values(*_quantize_rows(x, 1, E4M3), 1) @ _values(*_quantize_rows(w, BLK, E4M3), BLK).t()
    dx = _values(*_quantize_rows(dy, 1, E5M2), 1) @ _values(*_quantize_rows(w.t(), BLK, E4M3), BLK).t()
    dw = _values(*_quantize_rows(dy.t(), 1, E5M2), 1) @ _values(*_quantize_rows(x.t(), 1, E4M3), 1).t()
    return y.to(torch.bfloat16), dx[:, :K].to(torch.bfloat16), dw[:N, :K]


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(st):
    c = st["case"]
    if not own:
        return {"norm": _plain_norm, "norm_backward": _plain_norm_backward, "quantize": _plain_quantize,
                "product": _plain_product, "train": _plain_train}[c["kind"]](st)
    rmsnorm, proj = st["exts"]["rmsnorm"], st["exts"]["proj"]
    if c["kind"] == "norm":
        h, n, codes, scales = rmsnorm.block_norm(st["y"], residual=st["residual"], gate=st["gate"],
                                                 post_gamma=st["post_gamma"], gamma=st["gamma"], scale=st["scale"],
                                                 residual_scale=c["rs"], act=c["act"], eps=EPS, quantize=c["quant"])
        return (h, codes, scales) if c["quant"] else (h, n)
    if c["kind"] == "norm_backward":
        return rmsnorm.block_norm_backward(st["dh"], st["dn"], st["y"], residual=st["residual"], gate=st["gate"],
                                           post_gamma=st["post_gamma"], gamma=st["gamma"], scale=st["scale"],
                                           residual_scale=c["rs"], act=c["act"], rstd_y=st["rstd_y"],
                                           rstd_h=st["rstd_h"])
    if c["kind"] == "quantize":
        return proj.fp8_quantize(st["x"], block_rows=c["block"], dtype=FORMATS[c["fmt"]], rows=c["rows"],
                                 columns=c["columns"])
    if c["kind"] == "product":
        return proj.fp8_matmul(st["a"], st["a_scale"], st["b"], st["b_scale"],
                               out_dtype=torch.bfloat16 if c["out"] == "bf16" else torch.float32)
    x, xs, xt, xts = proj.fp8_quantize(st["x"], rows=True, columns=True)
    w, ws, wt, wts = proj.fp8_quantize(st["w"], block_rows=BLK, rows=True, columns=True)
    y = proj.fp8_matmul(x, xs, w, ws)
    d, ds, dt, dts = proj.fp8_quantize(st["dy"], dtype=E5M2, rows=True, columns=True)
    return y, proj.fp8_matmul(d, ds, wt, wts), proj.fp8_matmul(dt, dts, xt, xts, out_dtype=torch.float32)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    c = case
    if c["kind"] in ("norm", "norm_backward"):
        n = c["B"] * c["T"] * max(c["H"], 1) * c["D"]
        t = 4 if c["types"] == "fp32" else 2
        r = 2 if c["types"] == "bf16" else 4
        gs = _gate_shape(c)
        gate = math.prod(gs) * t if gs else 0
        if c["kind"] == "norm":
            b = n * t + (n * r if c["residual"] else 0) + gate + n * (r if c["residual"] else t)
            b += n if c["quant"] else (n * t if c["pre"] else 0)
            return {"bytes": b, "flops": 12 * n}
        b = n * (t + (r if c["residual"] else t)) + n * t + (n * t if c["pre"] else 0) + (2 * n * r if c["residual"] else 0)
        b += 2 * gate
        return {"bytes": b, "flops": 30 * n}
    if c["kind"] == "quantize":
        return {"bytes": c["M"] * c["K"] * (2 + c["rows"] + c["columns"]), "flops": 3 * c["M"] * c["K"]}
    M, N, K = c["M"], c["N"], c["K"]
    if c["kind"] == "product":
        return {"bytes": M * K + N * K + M * N * (2 if c["out"] == "bf16" else 4), "flops": 2 * M * N * K}
    return {"bytes": 2 * (M * K + N * K + M * N) + 2 * (M * N + M * K) + 4 * N * K, "flops": 6 * M * N * K}


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------
def _two64(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _grid64(v, mantissa, least):
    """v to the nearest number of `mantissa` bits after the point, ties to even, steps no finer than at 2^least."""
    _, e = torch.frexp(v)
    step = _two64((e - 1).clamp(min=least) - mantissa)
    return torch.round(v / step) * step


def _blocks64(x, rows, fmt):
    """Codes and scales of x [M, K] in float64 by definition: one power of two for rows x 128 values."""
    mantissa, least, most = (3, -6, 448.0) if fmt == E4M3 else (2, -14, 57344.0)
    M, K = x.shape
    Kp, Mp = -(-K // BLK) * BLK, -(-M // rows) * rows
    p = x.new_zeros(Mp, Kp)
    p[:M, :K] = x
    big = torch.nn.functional.max_pool2d(p.abs()[None, None], (rows, BLK))[0, 0]
    s = _two64(torch.ceil(torch.log2(big / most)).clamp(min=-200))
    s = torch.where(big / s > most, 2 * s, s)          # the logarithm may have
    s = torch.where(big / (s / 2) <= most, s / 2, s)   # rounded past a border
    s = torch.where(big > 0, s.clamp(min=2.0 ** -127), 1.0)
    wide = torch.kron(s, s.new_ones(rows, BLK))
    return _grid64(p / wide, mantissa, least)[:M], s, wide[:M]


def _forward64(st, c):
    """(leaves, h, n) by the definition, with a gradient tape."""
    names = ["y", "residual", "gate", "post_gamma", "gamma", "scale"]
    v = {k: None if st[k] is None else st[k].double().requires_grad_() for k in names}
    u = v["y"]
    if c["post"]:
        u = u / (u.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * v["post_gamma"]
    if c["gate"] != "none":
        z = v["gate"]
        if c["gate"] == "sequence":
            z = z[:, None, :]
        u = u * {"none": lambda z: z, "sigmoid": torch.sigmoid, "silu": lambda z: z / (1 + torch.exp(-z)),
                 "tanh": torch.tanh}[c["act"]](z)
    if c["scale"]:
        u = u * v["scale"]
    h = c["rs"] * u if v["residual"] is None else v["residual"] + c["rs"] * u
    n = h / (h.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * v["gamma"] if c["pre"] else None
    return v, h, n


def exact(case, seed):
    c = case
    st = prepare(case, seed)
    if c["kind"] == "norm":
        with torch.no_grad():
            _, h, n = _forward64(st, c)
            if not c["quant"]:
                return h, n
            codes, s, _ = _blocks64((h if n is None else n).reshape(-1, c["D"]), 1, E4M3)
            return h, codes, s
    if c["kind"] == "norm_backward":
        v, h, n = _forward64(st, c)
        loss = (h * st["dh"].double()).sum()
        if n is not None:
            loss = loss + (n * st["dn"].double()).sum()
        names = [k for k in ("residual", "y", "gate", "post_gamma", "gamma", "scale")]
        grads = dict(zip([k for k in names if v[k] is not None],
                         torch.autograd.grad(loss, [v[k] for k in names if v[k] is not None])))
        return tuple(grads.get(k) for k in names)
    if c["kind"] == "quantize":
        x, out = st["x"].double(), []
        for there, t in ((c["rows"], x), (c["columns"], x.t())):
            if there:
                out += list(_blocks64(t, c["block"], FORMATS[c["fmt"]])[:2])
        return out
    if c["kind"] == "product":
        N, K = c["N"], c["K"]
        of_a = torch.arange(K, device=DEV) // BLK
        a = st["a"].double() * st["a_scale"].double().index_select(1, of_a)
        b = st["b"].double() * st["b_scale"].double()[torch.arange(N, device=DEV) // c["brows"]].index_select(1, of_a)
        return torch.mm(a, b.t())
    def value(t, rows, fmt):
        codes, _, wide = _blocks64(t, rows, fmt)
        return codes * wide
    x, w, dy = st["x"].double(), st["w"].double(), st["dy"].double()
    y = torch.mm(value(x, 1, E4M3), value(w, BLK, E4M3).t())
    dx = torch.mm(value(dy, 1, E5M2), value(w.t(), BLK, E4M3).t())
    dw = torch.mm(value(dy.t(), 1, E5M2), value(x.t(), 1, E4M3).t())
    return y, dx[:, :c["K"]], dw[:c["N"], :c["K"]]
