"""Block norms of more rows than a launch has places for: workgroups walk rows.

The backward pass starts at most some hundreds of workgroups and each keeps the sums
over its rows, so the parameters' and shared gates' gradients come from two or more
rows a place here; the forward pass walks rows of over 4096 columns.  References are
in float64.

Tolerances.  A row's values as in test_block_norm_gpu.py: 64 * 2^-24 of the
magnitudes that enter them, 1e-5 of the row's largest gradient.  A sum over R rows of
one distribution: it is as large as sqrt(R) terms at some of the columns, and so are
the partial sums on its way.  A chain has at most 90 additions (4 rows a place, 16
workgroups a lane, 64 lanes, 3 groups), each off by 2^-24 of its partial sum, 5e-6 in
all; the terms' own errors, up to 4e-6 to either side, grow with sqrt(R) as the sum
does.  1e-5 of the largest column covers both.  A row left out or taken twice changes
a column by 1 / sqrt(R) of that, 7e-3.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

EPS = 1e-6
F32 = 64 * 2.0 ** -24
NAMES = ("residual", "y", "gate", "post_gamma", "gamma", "scale")


def _inputs(B, T, D, dtype, gate, dev, seed):
    g = torch.Generator(device=dev).manual_seed(seed)

    def rnd(shape, std=1.0, mean=0.0):
        return (torch.randn(shape, generator=g, device=dev) * std + mean).to(dtype)

    gs = {"token": (B, T, D), "sequence": (B, D), "channel": (D,)}[gate]
    v = dict(y=rnd((B, T, D), 0.7), residual=rnd((B, T, D), 2.0), gate=rnd(gs), post_gamma=rnd((D,), 0.1, 1.0),
             gamma=rnd((D,), 0.1, 1.0), scale=rnd((D,), 0.1, 1.0))
    return v, rnd((B, T, D)), rnd((B, T, D))


def _forward64(v, rs):
    """(leaves, h, n, magnitude of h's terms) with silu gates, in float64 on the GPU."""
    v = {k: t.double().requires_grad_() for k, t in v.items()}
    z = v["gate"][:, None] if v["gate"].dim() == 2 else v["gate"]
    u = v["y"] * (v["y"].pow(2).mean(-1, keepdim=True) + EPS).rsqrt() * v["post_gamma"] * z * torch.sigmoid(z) * v["scale"]
    h = v["residual"] + rs * u
    n = h * (h.pow(2).mean(-1, keepdim=True) + EPS).rsqrt() * v["gamma"]
    return v, h, n, (v["residual"].abs() + (rs * u).abs()).detach()


def _close(x, ref, tol, what):
    half = torch.finfo(x.dtype).eps / 2
    far = (x.double() - ref).abs() - (half * ref.abs() + (1 + half) * tol + 1e-30)
    assert x.shape == ref.shape and (far <= 0).all(), \
        f"{what}: {(~(far <= 0)).sum().item()} values, the worst {far.max().item():.3g} past its bound"


# sequences x tokens: two rows and more for every place of a workgroup, and a few rows left
@pytest.mark.parametrize("D,places", [(64, 16 * 512), (500, 4 * 512), (1000, 1024), (1001, 512), (2048, 512), (2500, 256), (4104, 256),
                                      (9000, 256)], ids=str)
@pytest.mark.parametrize("gate", ["token", "sequence", "channel"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_backward_of_many_rows(exts, dev, dtype, gate, D, places):
    B = 3
    T = max((2 * places + 5) // B + 1, 1400 if places == 1024 else 0)  # 4096 rows for the 1024 workgroups
    v, dh, dn = _inputs(B, T, D, dtype, gate, dev, D)
    out = exts["rmsnorm"].block_norm(**v, residual_scale=0.7, act="silu", eps=EPS, stats=True)
    got = exts["rmsnorm"].block_norm_backward(dh, dn, **v, residual_scale=0.7, act="silu", rstd_y=out[4], rstd_h=out[5])
    leaves, h, n, _ = _forward64(v, 0.7)
    want = torch.autograd.grad((h * dh.double()).sum() + (n * dn.double()).sum(), [leaves[k] for k in NAMES])
    for k, x, r in zip(NAMES, got, want):
        assert x.dtype == dtype
        _close(x, r, 1e-5 * r.abs().amax(-1, keepdim=True), "d" + k)


@pytest.mark.parametrize("D", [4104, 5001, 8192, 9001, 16384])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_forward_of_many_long_rows(exts, dev, dtype, D):
    """Written apart and over the residual, with codes and without."""
    f = exts["rmsnorm"].block_norm
    v, _, _ = _inputs(3, 207, D, dtype, "sequence", dev, D)
    h, n, _, _, ry, rh = f(**v, act="silu", eps=EPS, stats=True)
    leaves, h64, n64, mag = _forward64(v, 1.0)
    with torch.no_grad():
        rms = (h64.pow(2).mean(-1, keepdim=True) + EPS).sqrt()
        _close(h, h64, F32 * mag, "h")
        _close(n, n64, F32 * mag / rms * leaves["gamma"].abs(), "n")
        ry64 = (leaves["y"].pow(2).mean(-1) + EPS).rsqrt().reshape(-1)
        _close(ry, ry64, F32 * ry64, "rstd_y")
        _close(rh, 1 / rms.reshape(-1), F32 * (mag.pow(2).mean(-1).sqrt() / rms.squeeze(-1) ** 2).reshape(-1), "rstd_h")
    kept = v["residual"].clone()
    h2, n2, _, _ = f(**dict(v, residual=kept), act="silu", eps=EPS, inplace=True)
    assert h2.data_ptr() == kept.data_ptr() and torch.equal(h2, h) and torch.equal(n2, n)
    kept = v["residual"].clone()
    h3, _, codes, scales = f(**dict(v, residual=kept), act="silu", eps=EPS, inplace=True, quantize=True)
    assert torch.equal(h3, h)
    if dtype == torch.float32:  # the codes are those of the fp32 n
        c, s = exts["proj"].fp8_quantize(n.reshape(-1, D))
        assert torch.equal(codes.view(torch.uint8), c.view(torch.uint8)) and torch.equal(scales.view(torch.uint8), s.view(torch.uint8))
