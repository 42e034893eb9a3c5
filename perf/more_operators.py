"""Projections in 4-bit microscaled floating point and the clipping of gradients,
as measurable cases: quantisation to e2m1 codes with a power-of-two scale for each
32 of them and back, products of such weights with 4-bit or 8-bit activations, a
linear layer's training step on them, and the global norm of a model's gradients
with their clipping.

Sizes come from this repository's configurations, tests and benchmark: hidden
2048, 16 heads of 128 or 256, the fused q/k/v/a/b projection's 6176 or 8224
columns, batches up to 4 x 4096 tokens, a layer's twelve weights, with odd and
ragged ones beside them.  ``run`` computes in plain torch in 32 bits, or, where
``own`` is true, calls the framework.
"""

import math

import torch

own = False

DEV = "cuda"
E2M1X2, E4M3, E5M2, E8M0 = torch.float4_e2m1fn_x2, torch.float8_e4m3fn, torch.float8_e5m2, torch.float8_e8m0fnu
# a block's length, and the largest code as m 2^e with 1/2 <= m < 1
FORMATS = {"e2m1": (32, 0.75, 3), "e4m3": (128, 0.875, 9), "e5m2": (128, 0.875, 16)}
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
VALUES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
EPS = 1e-6


# ---------------------------------------------------------------------------
# The cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # One token's activations to 4 bits and back: a call's latency.
        dict(name="codes_token", kind="codes", M=1, K=2048, type="bf16", block=1, rows=True, columns=False),
        # The fused projection's weight, laid out for both directions of
        # training, and read back (an export, a check of what it became).
        dict(name="codes_weight", kind="codes", M=8224, K=2048, type="bf16", block=32, rows=True, columns=True),
        # One user's token through the fused projection: the weights' bytes.
        dict(name="product_token", kind="product", M=1, N=8224, K=2048, a="e4m3", block=1, out="bf16"),
        # A serving batch, not a round number, 4 bits on both sides.
        dict(name="product_serving", kind="product", M=48, N=2048, K=4096, a="e2m1", block=1, out="fp32"),
        # A prompt through the fused projection, 8-bit activations.
        dict(name="product_prompt", kind="product", M=1500, N=8224, K=2048, a="e4m3", block=32, out="bf16"),
        # The training-sized batch through the fused projection, 4 bits on both
        # sides: the largest.
        dict(name="product_batch", kind="product", M=16384, N=6176, K=2048, a="e2m1", block=32, out="bf16"),
        # Forward and backward of a projection over packed prompts.
        dict(name="train_prompts", kind="train", M=2683, N=2048, K=2048, a="e4m3", weight="fp32"),
        # The same of the output projection over two sequences of 4096.
        dict(name="train_batch", kind="train", M=8192, N=2048, K=4096, a="e2m1", weight="bf16"),
        # The gradients of one small layer: launches.
        dict(name="norm_layer", kind="norm", layers=1, D=256, H=2, dv=128, types="mixed", odd=False, spread=1.0, most=0.0),
        # The gradients of an eight-layer model, 96 tensors.
        dict(name="norm_model", kind="norm", layers=8, D=2048, H=16, dv=256, types="bf16", odd=False, spread=1.0, most=0.0),
        # One layer's gradients, 32-bit ones and odd lengths among them, clipped.
        dict(name="clip_layer", kind="clip", layers=1, D=1000, H=4, dv=128, types="mixed", odd=True, spread=1.0, most=1.0),
        # The gradients of a four-layer model, clipped for a 32-bit optimiser's
        # step: 48 tensors.
        dict(name="clip_model", kind="clip", layers=4, D=2048, H=16, dv=256, types="bf16", odd=False, spread=1.0, most=1.0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["codes", "codes", "product", "product", "product", "product", "train", "norm", "clip"])
    if kind == "codes":
        M = _log_int(rng, 1, 16384)
        rows, columns = rng.choice([(True, False), (False, True), (True, True)])
        return dict(kind=kind, M=M, K=_log_int(rng, 16, min(16384, (1 << 25) // M)), type=rng.choice(["bf16", "bf16", "fp32"]),
                    block=rng.choice([1, 1, 32]), rows=rows, columns=columns)
    if kind == "product":
        M, N = _log_int(rng, 1, 16384), _log_int(rng, 16, 8224)
        K = 128 * _log_int(rng, 1, max(1, min(64, (1 << 37) // (M * N * 128))))
        return dict(kind=kind, M=M, N=N, K=K, a=rng.choice(["e2m1", "e2m1", "e4m3", "e4m3", "e5m2"]), block=rng.choice([1, 32]),
                    out=rng.choice(["bf16", "bf16", "fp32"]))
    if kind == "train":
        return dict(kind=kind, M=_log_int(rng, 64, 8192), N=16 * _log_int(rng, 8, 256), K=16 * _log_int(rng, 8, 256),
                    a=rng.choice(["e4m3", "e2m1"]), weight=rng.choice(["bf16", "fp32"]))
    D = rng.choice([128, 333, 512, 1000, 2048])
    layers = _log_int(rng, 1, 4 if kind == "clip" else 24 if D < 2048 else 8)
    return dict(kind=kind, layers=layers, D=D, H=rng.choice([2, 4, 16]), dv=rng.choice([128, 256]),
                types=rng.choice(["bf16", "fp32", "mixed"]), odd=rng.random() < 0.5, spread=rng.choice([1.0, 30.0]),
                most=rng.choice([0.1, 1.0, 1e4]) if kind == "clip" else 0.0)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _pow2(e):
    """2^e in 32 bits, exactly (a power function may round)."""
    half = torch.div(e, 2, rounding_mode="floor")
    bits = lambda k: ((k + 127) << 23).to(torch.int32).view(torch.float32)  # noqa: E731
    return bits(half) * bits(e - half)


def _exponents(amax, fmt):
    """The least e >= -127 with amax / 2^e no larger than the format's largest code (0 where amax is 0)."""
    _, m_top, e_top = FORMATS[fmt]
    m, e = torch.frexp(amax)
    e = e - e_top + (m > m_top).int()
    return torch.where(amax > 0, e.clamp(min=-127), 0)


def _round4(v):
    """v, no larger than 6, to the nearest of 0, 1/2, 1, 3/2, 2, 3, 4, 6 and their negatives, ties to the even code."""
    a = v.abs()
    step = torch.where(a >= 4, 2.0, torch.where(a >= 2, 1.0, 0.5))
    return torch.round(v / step) * step


def _blocks(x, rows, fmt):
    """x [M, K] in fp32 as what its codes stand for over their scales, and the scales' exponents spread over them,
    [M, K padded to 128] each; one scale for `rows` x a block's length."""
    n = FORMATS[fmt][0]
    M, K = x.shape
    Kp, Mp = -(-K // 128) * 128, -(-M // rows) * rows
    t = torch.nn.functional.pad(x, (0, Kp - K, 0, Mp - M)).view(Mp // rows, rows, Kp // n, n)
    e = _exponents(t.abs().amax(dim=(1, 3)), fmt)[:, None, :, None]
    t = t * _pow2(-e)
    codes = _round4(t) if fmt == "e2m1" else t.to(E4M3 if fmt == "e4m3" else E5M2).float()
    return codes.reshape(Mp, Kp)[:M], e.expand(t.shape).reshape(Mp, Kp)[:M]


def _quantized(x, rows, fmt):
    """What x's codes and scales stand for, [M, K]."""
    codes, e = _blocks(x, rows, fmt)
    return (codes * _pow2(e))[:, :x.shape[1]]


def _packed(codes):
    """Values of e2m1 codes [M, K] as the codes, two a byte, the earlier one low."""
    c = torch.bucketize(codes.abs(), torch.tensor(VALUES, device=codes.device)).to(torch.uint8)
    c = c + 8 * torch.signbit(codes).to(torch.uint8)
    return (c[:, 0::2] | c[:, 1::2] << 4).contiguous().view(E2M1X2)


def _operand(x, rows, fmt):
    """(codes, scales) of x as the framework keeps them: 4-bit ones in rows of whole 256 values with scales [M, K / 128,
    4], 8-bit ones with scales [M, K / 128], both by blocks of 128 first and then by rows, 16 rows at a time."""
    n, M = FORMATS[fmt][0], x.shape[0]
    if fmt == "e2m1":
        x = torch.nn.functional.pad(x, (0, -x.shape[1] % 256))
    codes, e = _blocks(x, rows, fmt)
    s = (e[:, ::n] + 127).to(torch.uint8).view(M, -1, 128 // n)
    buf = torch.zeros(s.shape[1], -(-M // 16) * 16, 128 // n, dtype=torch.uint8, device=x.device)
    buf[:, :M] = s.transpose(0, 1)
    s = buf[:, :M].transpose(0, 1).view(E8M0)
    return (_packed(codes), s) if fmt == "e2m1" else (codes.to(E4M3 if fmt == "e4m3" else E5M2), s[:, :, 0])


def _shapes(c):
    """The weights of the case's layers (projections, convolutions, norm, gates), and with `odd` one of no round size."""
    D, K, V, H = c["D"], c["H"] * 128, c["H"] * c["dv"], c["H"]
    layer = [(D,), (K, D), (K, 4), (K, D), (K, 4), (V, D), (V, 4), (H, D), (H, D), (H,), (1,), (D, V)]
    return layer * c["layers"] + ([(D + 7, 3)] if c["odd"] else [])


def _gradient_types(c):
    n = len(_shapes(c))
    return [TYPES[c["types"]]] * n if c["types"] != "mixed" else [torch.float32 if i % 12 in (0, 4, 9, 10, 11) else torch.bfloat16 for i in range(n)]


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)

    def randn(*shape, dtype=torch.float32, std=1.0):
        return (torch.randn(shape, generator=g, device=DEV) * std).to(dtype)

    c = case
    st = {"case": case}
    if c["kind"] == "codes":  # rows of different magnitude, as activations have them
        st["x"] = (randn(c["M"], c["K"]) * torch.exp(randn(c["M"], 1))).to(TYPES[c["type"]])
    elif c["kind"] == "product":
        st["a"], st["a_scale"] = _operand(randn(c["M"], c["K"], dtype=torch.bfloat16).float(), 1, c["a"])
        st["b"], st["b_scale"] = _operand(randn(c["N"], c["K"], dtype=torch.bfloat16, std=0.02).float(), c["block"], "e2m1")
    elif c["kind"] == "train":
        st["x"] = randn(c["M"], c["K"], dtype=torch.bfloat16).requires_grad_()
        st["w"] = randn(c["N"], c["K"], dtype=TYPES[c["weight"]], std=0.02).requires_grad_()
        st["dy"] = randn(c["M"], c["N"], dtype=torch.bfloat16, std=1e-3)
    else:  # tensors of different magnitude, as a model's gradients are
        st["grads"] = [randn(*s, dtype=t, std=1e-3 * c["spread"] ** math.sin(i)) for i, (s, t) in enumerate(zip(_shapes(c), _gradient_types(c)))]
        if c["kind"] == "clip":  # where the optimiser reads them
            st["out"] = [torch.empty_like(t) for t in st["grads"]]
    return st


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------
def _plain_codes(st):
    c, x = st["case"], st["x"].float()
    return [_quantized(t, c["block"], "e2m1").to(st["x"].dtype) for there, t in ((c["rows"], x), (c["columns"], x.t())) if there]


def _values(codes, scales):
    """What codes with scales stand for, in 32 bits."""
    if codes.dtype == E2M1X2:
        bytes_ = codes.view(torch.uint8)
        table = torch.tensor(VALUES + [-v for v in VALUES], device=codes.device)
        v = table[torch.stack((bytes_ & 15, bytes_ >> 4), -1).view(codes.shape[0], -1).int()]
    else:
        v = codes.float()
    s = scales.float().reshape(v.shape[0], -1)
    return (v.view(v.shape[0], s.shape[1], -1) * s[:, :, None]).view(v.shape)


def _plain_product(st):
    a, b = _values(st["a"], st["a_scale"]), _values(st["b"], st["b_scale"])
    y = a @ b[:, :a.shape[1]].t()
    return y.to(TYPES[st["case"]["out"]])


def _plain_train(st):
    c = st["case"]
    x, w, dy = st["x"].detach().float(), st["w"].detach().float(), st["dy"].float()
    w4 = _quantized(w, 32, "e2m1")
    y = _quantized(x, 1, c["a"]) @ w4.t()
    dx = _quantized(dy, 1, "e5m2") @ w4
    dw = _quantized(dy.t(), 1, "e5m2") @ _quantized(x.t(), 1, "e4m3").t()
    return y.to(torch.bfloat16), dx.to(torch.bfloat16), dw.to(st["w"].dtype)


def _plain_norm(grads):
    return torch.stack([t.float().square().sum(dtype=torch.float64) for t in grads]).sum().sqrt().float()


def _plain_clip(st):
    norm = _plain_norm(st["grads"])
    f = (st["case"]["most"] / (norm + EPS)).clamp(max=1.0)
    return norm, [(t.float() * f).to(t.dtype) for t in st["grads"]]


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(st):
    c = st["case"]
    if not own:
        if c["kind"] == "norm":
            return _plain_norm(st["grads"])
        return {"codes": _plain_codes, "product": _plain_product, "train": _plain_train, "clip": _plain_clip}[c["kind"]](st)
    from gdn_18646_amd import blocks, compile_kernels
    proj = compile_kernels()["proj"]
    if c["kind"] == "codes":
        x = st["x"]
        q = proj.fp4_quantize(x, block_rows=c["block"], rows=c["rows"], columns=c["columns"])
        sizes = [n for there, n in ((c["rows"], c["K"]), (c["columns"], c["M"])) if there]
        return [proj.fp4_dequantize(q[2 * i], q[2 * i + 1], columns=n, dtype=x.dtype) for i, n in enumerate(sizes)]
    if c["kind"] == "product":
        return proj.fp4_matmul(st["a"], st["a_scale"], st["b"], st["b_scale"], out_dtype=TYPES[c["out"]])
    if c["kind"] == "train":
        y = blocks.fp4_linear(st["x"], st["w"], activations=E2M1X2 if c["a"] == "e2m1" else E4M3)
        return (y.detach(), *torch.autograd.grad(y, (st["x"], st["w"]), st["dy"]))
    if c["kind"] == "norm":
        return blocks.grad_norm(st["grads"])
    return blocks.clip_grad_norm(st["grads"], c["most"], out=st["out"]), st["out"]


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    c = case
    coded = lambda n, fmt: n * ((0.5 if fmt == "e2m1" else 1.0) + 1.0 / FORMATS[fmt][0])  # noqa: E731
    if c["kind"] == "codes":  # values in, codes out; codes in, values out
        n, t, ways = c["M"] * c["K"], 2 if c["type"] == "bf16" else 4, c["rows"] + c["columns"]
        return {"bytes": n * t + ways * (2 * coded(n, "e2m1") + n * t), "flops": 4 * n * ways}
    if c["kind"] in ("norm", "clip"):
        sizes = [(math.prod(s), 2 if t == torch.bfloat16 else 4) for s, t in zip(_shapes(c), _gradient_types(c))]
        b = sum(n * t for n, t in sizes)
        return {"bytes": b if c["kind"] == "norm" else 2 * b, "flops": (2 if c["kind"] == "norm" else 3) * sum(n for n, _ in sizes)}
    M, N, K = c["M"], c["N"], c["K"]
    if c["kind"] == "product":
        return {"bytes": coded(M * K, c["a"]) + coded(N * K, "e2m1") + M * N * (2 if c["out"] == "bf16" else 4), "flops": 2 * M * N * K}
    w = 2 if c["weight"] == "bf16" else 4
    return {"bytes": 4 * M * K + 4 * M * N + 2 * w * N * K, "flops": 6 * M * N * K}


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------
def _two64(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _standing_for(x, rows, n, mantissa, least, most):
    """x [M, K] in float64 as the format of `mantissa` bits, exponents from `least` on and largest number `most` has it,
    by definition: one power of two for rows x n values, codes to the nearest, ties to even."""
    M, K = x.shape
    p = x.new_zeros(-(-M // rows) * rows, -(-K // n) * n)
    p[:M, :K] = x
    big = torch.nn.functional.max_pool2d(p.abs()[None, None], (rows, n))[0, 0]
    s = _two64(torch.ceil(torch.log2(big / most)).clamp(min=-200))
    s = torch.where(big / s > most, 2 * s, s)          # the logarithm may have
    s = torch.where(big / (s / 2) <= most, s / 2, s)   # rounded past a border
    s = torch.where(big > 0, s.clamp(min=2.0 ** -127), 1.0)
    wide = torch.kron(s, s.new_ones(rows, n))
    v = p / wide
    step = _two64((torch.frexp(v)[1] - 1).clamp(min=least) - mantissa)
    return (torch.round(v / step) * step * wide)[:M, :K]


def _as4(x, rows):
    return _standing_for(x, rows, 32, 1, 0, 6.0)


def _as8(x, fmt):
    return _standing_for(x, 1, 128, 3, -6, 448.0) if fmt == "e4m3" else _standing_for(x, 1, 128, 2, -14, 57344.0)


def _decoded64(codes, scales):
    """What codes with scales stand for: a 4-bit code of sign s, exponent e and mantissa m is (-1)^s 2^(e - 1) (1 + m / 2),
    and m / 2 where e is 0."""
    if codes.dtype == E2M1X2:
        b = codes.view(torch.uint8)
        q = b.new_empty(b.shape[0], 2 * b.shape[1])
        q[:, 0::2], q[:, 1::2] = b % 16, torch.div(b, 16, rounding_mode="floor")
        s, e, m = (q & 8).double() / 8, (q & 6).double() / 2, (q & 1).double()
        v = (1 - 2 * s) * torch.where(e > 0, torch.exp2(e - 1) * (1 + m / 2), m / 2)
        n = 32
    else:
        v, n = codes.double(), 128
    return v * scales.double().flatten(1).index_select(1, torch.arange(v.shape[1], device=v.device) // n)


def exact(case, seed):
    c = case
    st = prepare(case, seed)
    if c["kind"] == "codes":
        x = st["x"].double()
        return [_as4(t, c["block"]) for there, t in ((c["rows"], x), (c["columns"], x.t())) if there]
    if c["kind"] == "product":
        return torch.mm(_decoded64(st["a"], st["a_scale"])[:, :c["K"]], _decoded64(st["b"], st["b_scale"])[:, :c["K"]].t())
    if c["kind"] == "train":
        x, w, dy = st["x"].detach().double(), st["w"].detach().double(), st["dy"].double()
        w4 = _as4(w, 32)
        y = torch.mm(_as4(x, 1) if c["a"] == "e2m1" else _as8(x, "e4m3"), w4.t())
        return y, torch.mm(_as8(dy, "e5m2"), w4), torch.mm(_as8(dy.t(), "e5m2"), _as8(x.t(), "e4m3").t())
    norm = math.sqrt(math.fsum(torch.linalg.vector_norm(t.double()).item() ** 2 for t in st["grads"]))
    if c["kind"] == "norm":
        return torch.tensor(norm, dtype=torch.float64)
    f = min(1.0, c["most"] / (norm + EPS))
    return torch.tensor(norm, dtype=torch.float64), [t.double() * f for t in st["grads"]]
