"""Block norms (rmsnorm.block_norm and its backward) on the GPU against their
definition in float64.

Tolerances count roundings.  A value written in bf16 is off by at most half a
step of the fp32 value (eps / 2 = 2^-8 of it); the fp32 value itself carries at
most some tens of roundings of 2^-24 (a product of up to seven factors, each rounded
once, and 1 / sqrt of a mean whose sum of D positive terms is off by no more
than the depth of its tree, at most 8 + 6 + 4 additions a path), so 64 * 2^-24
relative to the sum of the magnitudes that enter a value covers it.
"""

import pytest
import torch

from tests.test_fp8_gpu import _quantize64

pytestmark = pytest.mark.gpu

EPS = 1e-6
F32 = 64 * 2.0 ** -24


def _act(x, name):
    return {"none": lambda: x, "sigmoid": lambda: torch.sigmoid(x), "silu": lambda: x * torch.sigmoid(x),
            "tanh": lambda: torch.tanh(x)}[name]()


def _inputs(shape, types="bf16", gate="token", residual=True, post=True, pre=True, scale=True, seed=0, dev="cuda"):
    g = torch.Generator().manual_seed(seed)
    T = torch.float32 if types == "fp32" else torch.bfloat16
    R = torch.bfloat16 if types in ("bf16", "bf16_f32") else torch.float32
    P = torch.bfloat16 if types == "bf16" else torch.float32
    D = shape[-1]
    rnd = lambda s, t, std=1.0, mean=0.0: (torch.randn(s, generator=g) * std + mean).to(t).to(dev)  # noqa: E731
    gs = {"none": None, "token": shape, "sequence": (shape[0], D), "channel": (D,)}[gate]
    return dict(y=rnd(shape, T, 0.7), residual=rnd(shape, R, 2.0) if residual else None,
                gate=rnd(gs, T) if gs else None, post_gamma=rnd((D,), P, 0.1, 1.0) if post else None,
                gamma=rnd((D,), P, 0.1, 1.0) if pre else None, scale=rnd((D,), P, 0.1, 1.0) if scale else None)


def _reference(v, rs, act):
    """(float64 leaves, h, n, magnitude of h's terms)."""
    v = {k: None if t is None else t.double().cpu().requires_grad_() for k, t in v.items()}
    u = v["y"]
    if v["post_gamma"] is not None:
        u = u * (u.pow(2).mean(-1, keepdim=True) + EPS).rsqrt() * v["post_gamma"]
    if v["gate"] is not None:
        z = v["gate"]
        if z.dim() == 2 and v["y"].dim() > 2:
            z = z.reshape(z.shape[0], *([1] * (v["y"].dim() - 2)), z.shape[1])
        u = u * _act(z, act)
    if v["scale"] is not None:
        u = u * v["scale"]
    h = rs * u if v["residual"] is None else v["residual"] + rs * u
    mag = (rs * u).abs() + (0 if v["residual"] is None else v["residual"].abs())
    n = None
    if v["gamma"] is not None:
        n = h * (h.pow(2).mean(-1, keepdim=True) + EPS).rsqrt() * v["gamma"]
    return v, h, n, mag.detach()


def _close(x, ref, mag, what):
    """x is ref within one rounding to its type and F32 of the magnitudes mag."""
    eps = torch.finfo(x.dtype).eps / 2
    x, ref = x.detach().double().cpu(), ref.detach().double().cpu()
    assert x.shape == ref.shape, what
    far = (x - ref).abs() - (eps * ref.abs() + (1 + eps) * F32 * mag.double().cpu() + 1e-30)
    assert not (far > 0).any(), f"{what}: {(far > 0).sum().item()} values, the worst {far.max().item():.3g} past its bound"


SHAPES = [(1, 1, 2048), (2, 3, 128), (5, 7, 16, 256), (3, 5, 8), (2, 9, 1000), (4, 33, 2048), (2, 3, 2056), (3, 4096), (1, 2, 8192),
          (2, 16384), (3, 5, 1), (2, 5, 127), (3, 3, 2049), (2, 2, 5001)]


@pytest.mark.parametrize("types", ["bf16", "bf16_f32", "mixed", "fp32"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward(exts, dev, shape, types):
    gate = "token" if len(shape) != 3 else {1: "channel", 2: "sequence", 3: "token", 4: "sequence"}.get(shape[0], "token")
    act = ["none", "sigmoid", "silu", "tanh"][sum(shape) % 4]
    v = _inputs(shape, types, gate)
    h, n, codes, scales, ry, rh = exts["rmsnorm"].block_norm(**v, residual_scale=0.7, act=act, eps=EPS, stats=True)
    r, h64, n64, mag = _reference(v, 0.7, act)
    assert codes is None and scales is None
    assert h.dtype == v["residual"].dtype and n.dtype == v["y"].dtype
    _close(h, h64, mag, "h")
    # n's error: that of h over h's rms, times gamma
    rms = (h64.pow(2).mean(-1, keepdim=True) + EPS).sqrt()
    _close(n, n64, mag / rms * r["gamma"].abs(), "n")
    _close(ry, (r["y"].pow(2).mean(-1) + EPS).rsqrt().reshape(-1), (r["y"].pow(2).mean(-1) + EPS).rsqrt().reshape(-1), "rstd_y")
    _close(rh, 1 / rms.reshape(-1), (mag.pow(2).mean(-1).sqrt() / rms.squeeze(-1) ** 2).reshape(-1), "rstd_h")


@pytest.mark.parametrize("absent", ["residual", "gate", "post_gamma", "gamma", "scale"])
def test_forward_without(exts, dev, absent):
    v = _inputs((3, 5, 512))
    v[absent] = None
    h, n, _, _ = exts["rmsnorm"].block_norm(**v, act="silu" if absent != "gate" else "none")
    r, h64, n64, mag = _reference(v, 1.0, "silu")
    _close(h, h64, mag, "h")
    if absent == "gamma":
        assert n is None
    else:
        rms = (h64.pow(2).mean(-1, keepdim=True) + EPS).sqrt()
        _close(n, n64, mag / rms * r["gamma"].abs(), "n")


@pytest.mark.parametrize("shape,pre", [((1, 1, 2048), True), ((2, 7, 4, 128), False), ((3, 5, 1000), True), ((2, 3, 4104), True),
                                       ((7, 130), True), ((3, 5, 8192), False)], ids=str)
@pytest.mark.parametrize("types", ["bf16", "mixed", "fp32"])
def test_quantized_output(exts, dev, shape, pre, types):
    """Codes and scales stand for the fp32 n within half a code's step: 2^-4 of
    the value, or half the finest step, 2^-10 of the scale."""
    v = _inputs(shape, types, residual=pre, pre=pre)
    h, n, codes, scales = exts["rmsnorm"].block_norm(**v, act="silu", quantize=True)
    r, h64, n64, mag = _reference(v, 1.0, "silu")
    D, R = shape[-1], codes.shape[0]
    Dp = -(-D // 128) * 128
    assert n is None and codes.shape == (R, Dp) and scales.shape == (R, Dp // 128)
    assert codes.dtype == torch.float8_e4m3fn and scales.dtype == torch.float8_e8m0fnu
    what = (n64 if pre else h64).detach().reshape(-1, D)
    s = scales.double().cpu().repeat_interleave(128, 1)
    got = codes.double().cpu() * s
    assert (got[:, D:] == 0).all()
    err = (got[:, :D] - what).abs()
    slack = F32 * (mag.reshape(-1, D) * (r["gamma"].abs() / (h64.pow(2).mean(-1, keepdim=True) + EPS).sqrt().reshape(-1, 1) if pre else 1.0))
    assert (err <= torch.maximum(what.abs() * 2.0 ** -4, s[:, :D] * 2.0 ** -10) + slack).all()
    # the scale is the least power of two that holds the block
    big = torch.nn.functional.pad(what, (0, Dp - D)).reshape(R, -1, 128).abs().amax(-1)
    s = scales.double().cpu()
    assert (big <= 448 * s * (1 + 1e-5)).all() and (big > 224 * s * (1 - 1e-5)).all()


@pytest.mark.parametrize("D", [*range(2, 10), *range(121, 137), *range(1017, 1025)])
def test_every_remainder_of_columns(exts, dev, D):
    """Rows that end at each place of a lane's eight columns, both directions;
    the codes are those of the fp32 n that a call without them writes."""
    f = exts["rmsnorm"].block_norm
    for types in ("bf16", "fp32"):
        v = _inputs((2, 5, D), types, "sequence", seed=D)
        h, n, _, _ = f(**v, act="silu", eps=EPS)
        r, h64, n64, mag = _reference(v, 1.0, "silu")
        _close(h, h64, mag, "h")
        rms = (h64.pow(2).mean(-1, keepdim=True) + EPS).sqrt()
        _close(n, n64, mag / rms * r["gamma"].abs(), "n")
        h2, _, codes, scales = f(**v, act="silu", eps=EPS, quantize=True)
        assert torch.equal(h2, h)
        if types == "fp32":
            rc, rs = _quantize64(n.reshape(-1, D), 1, torch.float8_e4m3fn)
            assert torch.equal(scales.view(torch.uint8).cpu(), rs)
            got = codes.view(torch.uint8).cpu()
            assert ((got == rc) | ((got & 0x7f == 0) & (rc & 0x7f == 0))).all()
        g = torch.Generator().manual_seed(9)
        dh, dn = (torch.randn(h.shape, generator=g).to(h.dtype).to(dev) for _ in range(2))
        _check_grads(_run_backward(exts, v, 1.0, "silu", dh, dn), _grads64(v, 1.0, "silu", dh, dn)[0], 10)


def test_store_h_and_inplace(exts, dev):
    v = _inputs((4, 9, 2048))
    f = exts["rmsnorm"].block_norm
    h, n, _, _ = f(**v, act="tanh")
    h2, n2, _, _ = f(**v, act="tanh", store_h=False)
    assert h2 is None and torch.equal(n, n2)
    keep = dict(v, residual=v["residual"].clone())
    h3, n3, _, _ = f(**keep, act="tanh", inplace=True)
    assert h3.data_ptr() == keep["residual"].data_ptr() and torch.equal(h3, h) and torch.equal(n3, n)


@pytest.mark.parametrize("D", [513, 517, 1001, 2049])
def test_inplace_where_lanes_share_columns(exts, dev, D):
    """The row's last lane reads columns of the lane before it, which here may lie
    in another wave and have h written already."""
    for post in (True, False):
        v = _inputs((700, D), post=post)
        f = exts["rmsnorm"].block_norm
        h, n, _, _ = f(**v, act="silu")
        keep = dict(v, residual=v["residual"].clone())
        h2, n2, _, _ = f(**keep, act="silu", inplace=True)
        assert torch.equal(h2, h) and torch.equal(n2, n)


def test_inplace_overlap(exts, dev):
    """The residual itself as another operand is read before it is written; parts
    of it in other rows' places are refused."""
    f = exts["rmsnorm"].block_norm
    v = _inputs((6, 300))
    h, n, _, _ = f(v["y"], residual=v["y"], gamma=v["gamma"])
    y = v["y"].clone()
    h2, n2, _, _ = f(y, residual=y, gamma=v["gamma"], inplace=True)
    assert h2.data_ptr() == y.data_ptr() and torch.equal(h2, h) and torch.equal(n2, n)
    buf = torch.zeros(7, 300, dtype=torch.bfloat16, device=dev)
    with pytest.raises(RuntimeError, match="memory location"):
        f(buf[:6], residual=buf[1:], inplace=True)
    with pytest.raises(RuntimeError, match="memory location"):
        f(v["y"], residual=buf[:6], gamma=buf[2], inplace=True)
    with pytest.raises(RuntimeError, match="act must be"):
        f(buf[:0], act="gelu")


def test_inplace_strided(exts, dev):
    """Rows of a wider buffer: columns beside the residual's are taken, views that
    share columns with it are refused."""
    f = exts["rmsnorm"].block_norm
    g = torch.Generator().manual_seed(3)
    for D, at in ((256, 0), (600, 8), (1001, 5)):
        wide = torch.randn(9, 3 * D + 24, generator=g).to(torch.bfloat16).to(dev)
        gm, gate = (torch.randn(9, D, generator=g).to(torch.bfloat16).to(dev) for _ in range(2))
        y, r = wide[:, at:at + D], wide[:, at + D:at + 2 * D]
        kw = dict(gamma=wide[4, at + 2 * D:at + 3 * D], gate=gate, act="silu")
        h, n, _, _ = f(y, residual=r, **kw)
        keep = wide.clone()
        h2, n2, _, _ = f(y, residual=r, inplace=True, **kw)
        assert h2.data_ptr() == r.data_ptr() and torch.equal(r, h) and torch.equal(n2, n)
        keep[:, at + D:at + 2 * D] = h
        assert torch.equal(wide, keep)  # the other columns are as they were
        h3 = f(wide[1:, at:at + D], residual=r[:8])[0]  # other rows' columns beside it are apart as well
        assert torch.equal(f(wide[1:, at:at + D], residual=r[:8], inplace=True)[0], h3)
        for t in (wide[:8, at + D - 8:at + 2 * D - 8], wide[1:, at + D:at + 2 * D]):
            with pytest.raises(RuntimeError, match="memory locations of y"):
                f(t, residual=r[:8], inplace=True)
        with pytest.raises(RuntimeError, match="memory locations of gamma"):
            f(y, residual=r, gamma=r[3], inplace=True)
        with pytest.raises(RuntimeError, match="memory locations of gate"):
            f(gate[:8], residual=r[:8], gate=r[1:], inplace=True)


def test_strided_rows(exts, dev):
    """Operands that are column slices of a wider buffer, 16-byte aligned or not."""
    for off, D in ((64, 256), (3, 256), (64, 250)):
        wide = torch.randn(4, 6, 1024, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(dev)
        v = _inputs((4, 6, D))
        v["y"], v["gate"], v["residual"] = wide[..., off:off + D], wide[..., off + 300:off + 300 + D], wide[..., off + 600 - off % 8:off + 600 - off % 8 + D]
        a = exts["rmsnorm"].block_norm(**v, act="silu")
        b = exts["rmsnorm"].block_norm(**{k: t.contiguous() for k, t in v.items()}, act="silu")
        r, h64, n64, mag = _reference(v, 1.0, "silu")
        _close(a[0], h64, mag, "h")
        _close(b[0], h64, mag, "h")
        rms = (h64.pow(2).mean(-1, keepdim=True) + EPS).sqrt()
        _close(a[1], n64, mag / rms * r["gamma"].abs(), "n")


def test_empty_and_zero_rows(exts, dev):
    v = _inputs((0, 3, 256), gate="channel")
    h, n, _, _ = exts["rmsnorm"].block_norm(**v)
    assert h.shape == (0, 3, 256) and n.shape == (0, 3, 256)
    h, n, codes, scales = exts["rmsnorm"].block_norm(torch.zeros(3, 256, dtype=torch.bfloat16, device=dev), gamma=v["gamma"], quantize=True)
    assert (h == 0).all() and (codes.float() == 0).all() and (scales.float() == 1).all()


@pytest.mark.parametrize("size", [1e-15, 1e-18, 1e-19, 3e-20, 1e-20])
@pytest.mark.parametrize("D", [64, 300, 2048])
def test_tiny_rows_without_eps(exts, dev, D, size):
    """Rows whose mean of squares is subnormal: each square is off by half of 2^-149,
    which the norm's other roundings join."""
    y = torch.randn(5, D, generator=torch.Generator().manual_seed(D)).to(dev) * size
    gm = torch.ones(D, device=dev)
    h, n, _, _, ry, rh = exts["rmsnorm"].block_norm(y, post_gamma=gm, gamma=gm, eps=0.0, stats=True)
    _, n2, _, _ = exts["rmsnorm"].block_norm(y, gamma=gm, eps=0.0)
    ms = y.double().pow(2).mean(-1, keepdim=True)
    ref = y.double() / ms.sqrt()
    tol = (F32 + 2.0 ** -150 / ms) * ref.abs()
    for t in (h, n, n2):
        assert ((t.double() - ref).abs() <= tol).all()
    assert ((ry.double() * ms.sqrt()[:, 0] - 1).abs() <= F32 + 2.0 ** -150 / ms[:, 0]).all() and torch.isfinite(rh).all()


def test_not_finite_rows_stay_in_their_row(exts, dev):
    v = _inputs((4, 2048), gate="token")
    clean = exts["rmsnorm"].block_norm(**v, act="silu", quantize=True)
    v["y"][1, 700] = float("nan")
    v["residual"][2, 5] = float("inf")
    h, _, codes, scales = exts["rmsnorm"].block_norm(**v, act="silu", quantize=True)
    for row in (0, 3):
        assert torch.equal(h[row], clean[0][row]) and torch.equal(codes[row].view(torch.uint8), clean[2][row].view(torch.uint8))
        assert torch.equal(scales[row].view(torch.uint8), clean[3][row].view(torch.uint8))
    for row in (1, 2):  # every value of n stands for NaN (or, in the infinite row, for zero)
        got = codes[row].float() * scales[row].float().repeat_interleave(128)
        assert got.isnan().any() and (got.isnan() | (got == 0)).all()


# ---------------------------------------------------------------------------
# Backward
# ---------------------------------------------------------------------------
def _grads64(v, rs, act, dh, dn):
    r, h, n, _ = _reference(v, rs, act)
    loss = 0
    if dh is not None:
        loss = loss + (h * dh.double().cpu()).sum()
    if dn is not None:
        loss = loss + (n * dn.double().cpu()).sum()
    names = [k for k in ("residual", "y", "gate", "post_gamma", "gamma", "scale") if r[k] is not None]
    return dict(zip(names, torch.autograd.grad(loss, [r[k] for k in names], allow_unused=True))), h, n


def _run_backward(exts, v, rs, act, dh, dn):
    out = exts["rmsnorm"].block_norm(**v, residual_scale=rs, act=act, eps=EPS, stats=True)
    g = exts["rmsnorm"].block_norm_backward(dh, dn, **v, residual_scale=rs, act=act, rstd_y=out[4],
                                            rstd_h=out[5] if dn is not None else None)
    return dict(zip(("residual", "y", "gate", "post_gamma", "gamma", "scale"), g))


def _check_grads(got, ref, R):
    """A value of a row is off by its one rounding and some tens of fp32 ones of
    the row's magnitudes: bounded by 1e-5 of the row's largest value.  A sum over
    R rows adds R such errors of random sign at most linearly: 1e-5 of its column
    sums' scale, taken as the largest magnitude over the columns (rows are of
    one distribution)."""
    for k, t in got.items():
        if t is None:
            assert ref.get(k) is None
            continue
        x, r = t.double().cpu(), ref[k]
        r = torch.zeros_like(x) if r is None else r
        assert x.shape == r.shape, k
        eps = torch.finfo(t.dtype).eps / 2
        big = r.abs().amax(-1, keepdim=True)
        far = (x - r).abs() - (eps * r.abs() + 1e-5 * big + 1e-30)
        assert not (far > 0).any(), f"d{k}: {(far > 0).sum().item()} values, the worst {far.max().item():.3g} past its bound"


@pytest.mark.parametrize("types", ["bf16", "bf16_f32", "mixed", "fp32"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_backward(exts, dev, shape, types):
    gate = "token" if len(shape) != 3 else {1: "channel", 2: "sequence", 3: "token", 4: "sequence"}.get(shape[0], "token")
    act = ["none", "sigmoid", "silu", "tanh"][sum(shape) % 4]
    v = _inputs(shape, types, gate, seed=3)
    g = torch.Generator().manual_seed(9)
    dh = torch.randn(shape, generator=g).to(v["residual"].dtype).to(dev)
    dn = torch.randn(shape, generator=g).to(v["y"].dtype).to(dev)
    ref, _, _ = _grads64(v, 0.7, act, dh, dn)
    if shape[-1] == 1:  # gradients through a norm of one value cancel to its eps share: compare the others
        ref = {k: t for k, t in ref.items()}
        got = _run_backward(exts, v, 0.7, act, dh, dn)
        for k in ("gamma",):
            _check_grads({k: got[k]}, ref, 0)
        assert all(torch.isfinite(t.float()).all() for t in got.values())
        return
    _check_grads(_run_backward(exts, v, 0.7, act, dh, dn), ref, v["y"].numel() // shape[-1])


@pytest.mark.parametrize("gate", ["none", "token", "sequence", "channel"])
@pytest.mark.parametrize("absent", ["", "residual", "post_gamma", "gamma", "scale", "dh", "dn"])
def test_backward_without(exts, dev, gate, absent):
    shape = (3, 37, 256)
    v = _inputs(shape, "fp32", gate, seed=4)
    g = torch.Generator().manual_seed(9)
    dh, dn = (torch.randn(shape, generator=g).to(dev) for _ in range(2))
    if absent in v:
        v[absent] = None
    if absent in ("dn", "gamma"):
        dn = None
    if absent == "dh":
        dh = None
    act = "silu" if gate != "none" else "none"
    ref, _, _ = _grads64(v, 1.0, act, dh, dn)
    _check_grads(_run_backward(exts, v, 1.0, act, dh, dn), ref, 111)


@pytest.mark.parametrize("B,T,D", [(2, 300, 136), (5, 41, 700), (17, 3, 64), (31, 2, 130), (32, 9, 96), (33, 9, 96), (70, 2, 40)])
def test_backward_of_shared_gates(exts, dev, B, T, D):
    """Gates a sequence, around the number of them that one launch sums."""
    for types in ("bf16", "fp32"):
        v = _inputs((B, T, D), types, "sequence", seed=B)
        g = torch.Generator().manual_seed(9)
        dh, dn = (torch.randn((B, T, D), generator=g).to(v["y"].dtype).to(dev) for _ in range(2))
        _check_grads(_run_backward(exts, v, 0.7, "tanh", dh, dn), _grads64(v, 0.7, "tanh", dh, dn)[0], B * T)


def test_backward_against_differences(exts, dev):
    """Directional differences of the forward kernel itself, in fp32."""
    shape, act = (2, 5, 384), "silu"
    v = _inputs(shape, "fp32", "sequence", seed=5)
    g = torch.Generator().manual_seed(2)
    dh, dn = (torch.randn(shape, generator=g).to(dev) for _ in range(2))
    got = _run_backward(exts, v, 1.0, act, dh, dn)
    f = exts["rmsnorm"].block_norm

    def loss(w):
        h, n, _, _ = f(**w, act=act)
        return ((h.double() * dh.double()).sum() + (n.double() * dn.double()).sum()).item()

    for k, t in v.items():
        d = torch.randn(t.shape, generator=g).to(dev)
        e = 2.0 ** -8
        diff = (loss(dict(v, **{k: t + e * d})) - loss(dict(v, **{k: t - e * d}))) / (2 * e)
        want = (got[k].double() * d.double()).sum().item()
        # the difference's own error: third order in e = 2^-8 (1.5e-5 of the second
        # derivatives' scale) and the fp32 rounding of some 4e3 outputs over 2 e
        scale = (got[k].double().norm() * d.double().norm()).item()
        assert abs(diff - want) <= 2e-3 * scale, (k, diff, want)


def test_backward_repeats_bit_for_bit(exts, dev):
    v = _inputs((4, 700, 2048), "bf16", "sequence", seed=6)
    g = torch.Generator().manual_seed(9)
    dh, dn = (torch.randn((4, 700, 2048), generator=g).to(torch.bfloat16).to(dev) for _ in range(2))
    a, b = (_run_backward(exts, v, 1.0, "tanh", dh, dn) for _ in range(2))
    assert all(torch.equal(a[k], b[k]) for k in a)


def test_backward_of_no_rows_is_zero(exts, dev):
    v = _inputs((0, 4, 256), gate="channel")
    e = torch.empty(0, dtype=torch.float32, device=dev)
    z = torch.empty(0, 4, 256, dtype=torch.bfloat16, device=dev)
    got = exts["rmsnorm"].block_norm_backward(z, z, **v, rstd_y=e, rstd_h=e)
    assert [tuple(t.shape) for t in got] == [(0, 4, 256), (0, 4, 256), (256,), (256,), (256,), (256,)]
    assert all((t == 0).all() for t in got[2:])


def test_graph_replays_match_eager(exts, dev):
    """Forward and backward captured together, replayed with other work between."""
    v = _inputs((2, 40, 2048), "bf16", "sequence", seed=7)
    g = torch.Generator().manual_seed(9)
    dh, dn = (torch.randn((2, 40, 2048), generator=g).to(torch.bfloat16).to(dev) for _ in range(2))
    eager = _run_backward(exts, v, 1.0, "silu", dh, dn)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _run_backward(exts, v, 1.0, "silu", dh, dn)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _run_backward(exts, v, 1.0, "silu", dh, dn)
    for _ in range(3):
        for t in got.values():
            t.fill_(7.0)
        graph.replay()
        _run_backward(exts, v, 1.0, "silu", dn, dh)
        torch.cuda.synchronize()
        assert all(torch.equal(got[k], eager[k]) for k in eager)
