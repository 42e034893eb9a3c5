"""4-bit codes by definition, on the CPU in 64 bits: what the tests of the 4-bit
quantisation, product and linear layer compare with."""

import torch

E2, E4, E5, E8 = torch.float4_e2m1fn_x2, torch.float8_e4m3fn, torch.float8_e5m2, torch.float8_e8m0fnu
VALUES = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], dtype=torch.float64)


def up(n, to):
    return -(-n // to) * to


def nearest(v):
    """The code (0 to 15) nearest to each of v, ties to the even code; |v| <= 6."""
    d = (v.abs()[..., None] - VALUES[:8]).abs()
    best = d.amin(-1, keepdim=True)
    ties = d == best  # one code, or two neighbours of which the even one is wanted
    code = torch.where(ties, torch.arange(8) + torch.arange(8) % 2 * 100, 1000).amin(-1) % 100
    return (code + 8 * torch.signbit(v)).to(torch.uint8)


def quantize64(x, rows):
    """(codes [M, Kp] one an element, scale bytes [M, Kp / 32]) of x [M, K], Kp = K up to a multiple of 256."""
    M, K = x.shape
    p = torch.zeros(up(M, rows), up(K, 256), dtype=torch.float64)
    p[:M, :K] = x.double().cpu()
    t = p.view(p.shape[0] // rows, rows, -1, 32)
    bad = ~torch.isfinite(t).all(3).all(1)
    amax = torch.where(torch.isfinite(t), t.abs(), 0).amax((1, 3))
    m, e = torch.frexp(amax / 6)  # amax / 6 = m 2^e, 1/2 <= m < 1: 2^(e - 1) holds it only at m = 1/2
    e = torch.where(amax > 0, torch.where(m == 0.5, e - 1, e), 0).clamp(min=-127)
    v = t / torch.ldexp(torch.ones_like(amax), e)[:, None, :, None]
    codes = torch.where(bad[:, None, :, None], torch.tensor(0, dtype=torch.uint8), nearest(torch.where(torch.isfinite(v), v, 0).clamp(-6, 6)))
    scales = torch.where(bad, 255, e + 127).to(torch.uint8).repeat_interleave(rows, 0)[:M]
    return codes.view(p.shape)[:M], scales


def unpack(codes):
    """[M, K / 2] of two a byte as [M, K] codes."""
    b = codes.view(torch.uint8).cpu()
    return torch.stack((b & 15, b >> 4), -1).view(b.shape[0], -1)


def pack(codes):
    c = codes.to(torch.uint8)
    return (c[:, 0::2] | c[:, 1::2] << 4).contiguous().view(E2)


def words(s):
    """Scale bytes [M, K / 32] laid out as the product reads them, [M, K / 128, 4]."""
    M, n = s.shape
    buf = torch.full((n // 4, up(M, 16), 4), 255, dtype=torch.uint8, device=s.device)  # what lies behind the last row is not looked at
    buf[:, :M] = s.view(torch.uint8).view(M, -1, 4).transpose(0, 1)
    return buf.view(E8)[:, :M].transpose(0, 1)


def values(codes, scales):
    """What codes [M, Kp] (one an element) with scale bytes [M, Kp / 32] stand for, in 64 bits."""
    s = torch.where(scales == 255, torch.nan, torch.ldexp(torch.ones(scales.shape, dtype=torch.float64), scales.int().cpu() - 127))
    return VALUES[codes.long().cpu()] * s.repeat_interleave(32, 1)
