"""4-bit quantisation, its inverse and the product with 4-bit weights on the GPU
against their definitions.

Quantisation has one answer and so has its inverse: both are compared bit for bit.

The product.  4-bit codes on both sides: an instruction adds 128 products and the
accumulator with an error of at most 2^-21 of the largest of them, none of which is
larger than the sum of the terms' magnitudes; K / 128 instructions and at most eight
partial sums make (K / 128 + 8) 2^-21 of it.  8-bit codes, fp32 results: every
product is exact in fp32 (4 by 2 bits) and so are the powers of two, so the result is
off by the half steps of its K + K / 128 + 8 additions, 2^-24 each.  8-bit codes, bf16
results: the instruction drops 2^-17 of the largest product for each of 128, 2^-10 of
it a block.  A bf16 result adds half its own step, 2^-8.
"""

import pytest
import torch

from gdn_18646_amd import abi
from tests.fp4 import E2, E4, E5, E8, pack, quantize64, unpack, up, values, words

pytestmark = pytest.mark.gpu

SPECIAL = torch.tensor([0.0, -0.0, 6.0, 6.1, 0.25, -0.75, 2.5, 5.0, 1e-38, 1e-40, 3e38, -3e38, 1.0, 2.0 ** -126, 2.0 ** -133])


def _bits(t):
    return t.view(torch.uint8).cpu()


def _compare(codes, scales, x, rows):
    rc, rs = quantize64(x, rows)
    assert codes.dtype == E2 and scales.dtype == E8 and scales.shape == (x.shape[0], up(x.shape[1], 256) // 128, 4)
    assert torch.equal(_bits(scales).reshape(x.shape[0], -1), rs)
    got = unpack(codes)
    assert got.shape == rc.shape
    same = (got == rc) | ((got & 7 == 0) & (rc & 7 == 0))  # the sign of an underflowed zero is free
    assert same.all(), (got[~same][:5], rc[~same][:5])


@pytest.mark.parametrize("block", [1, 32])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("M,K", [(1, 1), (1, 16), (1, 2048), (3, 130), (77, 1000), (128, 128), (129, 384), (300, 513), (260, 8), (33, 31)])
def test_quantize(exts, dev, M, K, dtype, block):
    g = torch.Generator().manual_seed(M * K)
    x = (torch.randn(M, K, generator=g) * torch.exp(3 * torch.randn(M, 1, generator=g))).to(dtype)
    n = min(len(SPECIAL), M * K)
    x.view(-1)[torch.randint(0, M * K, (n,), generator=g)] = SPECIAL[:n].to(dtype)
    if M > 2:
        x[1] = 0
    q = exts["proj"].fp4_quantize(x.to(dev), block_rows=block, rows=True, columns=True)
    _compare(*q[:2], x, block)
    _compare(*q[2:], x.t(), block)
    for kw, pair in ((dict(rows=True), q[:2]), (dict(rows=False, columns=True), q[2:])):  # each alone gives the same
        alone = exts["proj"].fp4_quantize(x.to(dev), block_rows=block, **kw)
        assert len(alone) == 2 and all(torch.equal(_bits(a), _bits(b)) for a, b in zip(alone, pair))
    if block == 32:  # the same values both ways
        rows, columns = (exts["proj"].fp4_dequantize(*p, columns=c, dtype=torch.float32) for p, c in ((q[:2], K), (q[2:], M)))
        assert torch.equal(rows, columns.t())


@pytest.mark.parametrize("K", [*range(2, 10), *range(25, 40), *range(249, 265)])
def test_quantize_every_remainder_of_columns(exts, dev, K):
    for dtype in (torch.bfloat16, torch.float32):
        x = torch.randn(5, K, generator=torch.Generator().manual_seed(K)).to(dtype)
        q = exts["proj"].fp4_quantize(x.to(dev), rows=True, columns=True)
        _compare(*q[:2], x, 1)
        _compare(*q[2:], x.t(), 1)


def test_every_tie_rounds_to_the_even_code(exts, dev):
    x = torch.tensor([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0, 0.0]).repeat(1, 2)
    codes, _ = exts["proj"].fp4_quantize(x.to(dev))
    assert unpack(codes)[0, :16].tolist() == [7, 0, 2, 2, 4, 4, 6, 6, 8, 10, 10, 12, 12, 14, 14, 0]


@pytest.mark.parametrize("block", [1, 32])
def test_quantize_not_finite(exts, dev, block):
    x = torch.randn(200, 300, generator=torch.Generator().manual_seed(1))
    x[5, 7], x[150, 290], x[40, 40] = float("nan"), float("-inf"), float("inf")
    q = exts["proj"].fp4_quantize(x.to(dev), block_rows=block, rows=True, columns=True)
    for pair, t in ((q[:2], x), (q[2:], x.t())):
        _compare(*pair, t, block)
        v = exts["proj"].fp4_dequantize(*pair, columns=t.shape[1], dtype=torch.float32).cpu()
        rc, rs = quantize64(t, block)
        assert torch.equal(v.isnan(), (rs == 255).repeat_interleave(32, 1)[:, :t.shape[1]])


def test_quantize_strided_rows(exts, dev):
    wide = torch.randn(90, 700, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(dev)
    for lo, hi in ((64, 320), (3, 290), (64, 321)):
        a = exts["proj"].fp4_quantize(wide[:, lo:hi], rows=True, columns=True)
        b = exts["proj"].fp4_quantize(wide[:, lo:hi].contiguous(), rows=True, columns=True)
        assert all(torch.equal(_bits(x), _bits(y)) for x, y in zip(a, b))


@pytest.mark.parametrize("block", [1, 32])
@pytest.mark.parametrize("M,K", [(1, 200), (97, 130), (126, 300), (130, 257)])
def test_quantize_leaves_what_lies_behind(dev, M, K, block):
    """Through the C ABI, into buffers that are wider and longer than the results."""
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(M)).to(torch.bfloat16).to(dev)
    Mp, Kp = up(M, 256), up(K, 256)
    ldc, ldt, lds, ldst = Kp // 2 + 32, Mp // 2 + 48, M + 7, K + 5
    codes, scales, codes_t, scales_t = (torch.full(s, 0x55, dtype=torch.uint8, device=dev)
                                        for s in ((M + 2, ldc), (Kp // 128 + 1, lds, 4), (K + 2, ldt), (Mp // 128 + 1, ldst, 4)))
    abi.call("gdn_fp4_quantize_hip", x.data_ptr(), K, 0, M, K, block, codes.data_ptr(), ldc, scales.data_ptr(), lds,
             codes_t.data_ptr(), ldt, scales_t.data_ptr(), ldst, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    for got_c, got_s, t in ((codes, scales, x.cpu()), (codes_t, scales_t, x.t().cpu())):
        rc, rs = quantize64(t, block)
        m, k = rc.shape
        keep_c, keep_s = got_c.cpu(), got_s.cpu()
        assert (keep_c[m:] == 0x55).all() and (keep_c[:, k // 2:] == 0x55).all()
        assert (keep_s[k // 128:] == 0x55).all() and (keep_s[:, m:] == 0x55).all()
        c = unpack(keep_c[:m, :k // 2].contiguous())
        assert ((c == rc) | ((c & 7 == 0) & (rc & 7 == 0))).all()
        assert torch.equal(keep_s[:k // 128, :m].transpose(0, 1).reshape(m, -1), rs)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("M,K", [(1, 1), (1, 2048), (3, 130), (77, 1000), (128, 128), (129, 384), (300, 513), (260, 8), (1030, 1300), (0, 256), (5, 0)])
def test_quantize_to_both_formats(exts, dev, M, K, dtype):
    """4-bit codes along the rows and 8-bit ones along the columns, from one read: what two give."""
    g = torch.Generator().manual_seed(M + 7 * K)
    x = (torch.randn(M, K, generator=g) * torch.exp2(torch.randint(-30, 30, (M, 1), generator=g).float())).to(dev, dtype)
    if M > 100:
        x[3, 5], x[40, 7], x[M - 1, K - 1] = float("nan"), float("inf"), 0.0
        x[:, 6] = 0
    for t in (x, torch.cat([x, x], 1)[:, :K], x[::2]):
        got = exts["proj"].fp4_fp8_quantize(t)
        want = exts["proj"].fp4_quantize(t) + exts["proj"].fp8_quantize(t, rows=False, columns=True)
        for a, b in zip(got, want):
            assert a.shape == b.shape and a.dtype == b.dtype and torch.equal(a.view(torch.uint8), b.view(torch.uint8))
            assert a.stride() == b.stride() or a.numel() == 0


def test_quantize_to_both_formats_leaves_what_lies_behind(dev):
    M, K, ldc, lds, ldt, ldst = 130, 300, 272, 136, 272, 310
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(3)).to(dev)
    full = lambda *n: torch.full(n, 0x5a, dtype=torch.uint8, device=dev)  # noqa: E731
    codes, scales, codes_t, scales_t = full(M + 1, ldc), full(4, lds, 4), full(K + 1, ldt), full(2, ldst)
    abi.call("gdn_fp4_fp8_quantize_hip", x.data_ptr(), K, 1, M, K, codes.data_ptr(), ldc, scales.data_ptr(), lds, codes_t.data_ptr(), ldt,
             scales_t.data_ptr(), ldst, torch.cuda.current_stream().cuda_stream)
    assert (codes[M:] == 0x5a).all() and (codes[:, 256:] == 0x5a).all() and (scales[:, M:] == 0x5a).all()
    assert (codes_t[K:] == 0x5a).all() and (codes_t[:, 256:] == 0x5a).all() and (scales_t[:, K:] == 0x5a).all()
    assert (codes[:M, 150:256] == 0).all() and (codes_t[:K, M:256] == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("M,K", [(1, 256), (3, 256), (16, 512), (70, 2048)])
def test_dequantize(exts, dev, M, K, dtype):
    """Every code with every scale; bf16's and fp32's largest numbers are the same, give or take a rounding."""
    g = torch.Generator().manual_seed(M)
    codes = torch.randint(0, 16, (M, K), generator=g)
    scales = torch.randint(0, 256, (M, K // 32), generator=g).to(torch.uint8)
    want = values(codes, scales).float()
    c, s = pack(codes).to(dev), scales.view(E8).to(dev)
    for n in (K, K - 1, 37, 8, 1, 0):
        for layout in (s, words(s), s.view(M, -1, 4)):
            got = exts["proj"].fp4_dequantize(c, layout, columns=n, dtype=dtype)
            assert got.dtype == dtype and got.shape == (M, n)
            torch.testing.assert_close(got.float().cpu(), want[:, :n], rtol=0, atol=0, equal_nan=True)
    wide = torch.zeros(M, K, dtype=torch.uint8, device=dev)
    wide[:, 20:20 + K // 2] = c.view(torch.uint8)
    assert torch.equal(_bits(exts["proj"].fp4_dequantize(wide.view(E2)[:, 20:20 + K // 2], s, dtype=dtype)), _bits(exts["proj"].fp4_dequantize(c, s, dtype=dtype)))


# ---------------------------------------------------------------------------
# The product
# ---------------------------------------------------------------------------
TOP = {E4: 448.0, E5: 57344.0}


class Side:
    """Codes and scales of an operand, on the CPU and on the GPU, and its values in 64 bits."""

    def __init__(self, rows, K, fmt, g, dev, lo=115, hi=140):
        self.fmt, self.K = fmt, K
        if fmt == E2:
            kp = up(K, 256)
            codes = torch.randint(0, 16, (rows, kp), generator=g)
            codes[:, K:] = 0
            scales = torch.randint(lo, hi, (rows, kp // 32), generator=g).to(torch.uint8)
            self.codes, self.scales = pack(codes).to(dev), words(scales.view(E8).to(dev))
            self.values = values(codes, scales)[:, :K].to(dev)
        else:
            self.codes = (torch.randn(rows, K, generator=g) * (100 if fmt == E4 else 3000)).clamp(-TOP[fmt], TOP[fmt]).to(fmt).to(dev)
            scales = torch.randint(lo, hi, (rows, K // 128), generator=g).to(torch.uint8)
            self.scales = scales.view(E8).to(dev)
            self.values = self.codes.double() * self.scales.double().repeat_interleave(128, 1)

    def top(self):
        return self.values.abs().view(self.values.shape[0], -1, 128).amax(2)


def _operands(M, N, K, fa, dev, seed=0, **kw):
    g = torch.Generator().manual_seed(seed + M + 31 * N + 7 * K)
    return Side(M, K, fa, g, dev, **kw), Side(N, K, E2, g, dev, **kw)


def _check(y, a, b):
    ref, mag, K = a.values @ b.values.t(), a.values.abs() @ b.values.abs().t(), a.K
    if a.fmt == E2:
        tol = (K / 128 + 8) * 2.0 ** -21 * mag
    else:
        tol = (K + K / 128 + 8) * 2.0 ** -24 * mag
        if y.dtype == torch.bfloat16:
            tol = tol + 2.0 ** -10 * a.top() @ b.top().t()
    if y.dtype == torch.bfloat16:
        tol = tol + 2.0 ** -8 * (ref.abs() + tol)
    far = (y.double() - ref).abs() - tol
    assert y.shape == ref.shape and not (far > 0).any() and torch.isfinite(y).all(), f"{(far > 0).sum().item()} values, the worst {far.max().item():.3g} past its bound"


def _product(exts, a, b, out=torch.bfloat16):
    y = exts["proj"].fp4_matmul(a.codes, a.scales, b.codes, b.scales, out_dtype=out)
    assert y.dtype == out
    return y


SIZES = [(1, 1, 256), (1, 2048, 2048), (2, 100, 512), (16, 129, 1280), (17, 40, 256), (33, 65, 256), (77, 300, 1280), (64, 64, 8448),
         (130, 1040, 512), (300, 1030, 512), (513, 2100, 256), (1030, 2050, 512), (2500, 5003, 256), (5, 33, 8448), (3, 5000, 768),
         (16, 4100, 768), (1, 8224, 2048), (48, 2048, 4096), (700, 1500, 768), (1500, 3100, 512), (2100, 450, 768), (2341, 200, 256)]


@pytest.mark.parametrize("fa", [E2, E4, E5], ids=["e2m1", "e4m3", "e5m2"])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_product(exts, dev, M, N, K, fa):
    a, b = _operands(M, N, K, fa, dev)
    for out in (torch.float32, torch.bfloat16):
        print(f"{M} x {N} x {K} {fa} {out}", flush=True)
        _check(_product(exts, a, b, out), a, b)


@pytest.mark.parametrize("fa", [E4, E5], ids=["e4m3", "e5m2"])
@pytest.mark.parametrize("M,N,K", [(1, 40, 128), (2, 300, 384), (3, 33, 128), (16, 129, 640), (70, 300, 1152), (130, 1040, 384), (300, 1030, 896),
                                   (1030, 2050, 384), (2500, 5003, 128), (1500, 3100, 640), (2756, 1500, 128), (2092, 450, 384)])
def test_product_over_half_a_row_of_codes(exts, dev, M, N, K, fa):
    """8-bit codes of an odd number of blocks: the weight's last 128 codes are padding."""
    a, b = _operands(M, N, K, fa, dev)
    b.codes.view(torch.uint8)[:, K // 2:] = 0x77  # whatever it holds: there is nothing to multiply it with
    for out in (torch.float32, torch.bfloat16):
        print(f"{M} x {N} x {K} {fa} {out}", flush=True)
        _check(_product(exts, a, b, out), a, b)


@pytest.mark.parametrize("fa", [E2, E4], ids=["e2m1", "e4m3"])
@pytest.mark.parametrize("M,N,K", [(1, 8192, 256), (2, 9001, 512), (1, 16383, 2560), (2, 16384, 256), (1, 20010, 4352)])
def test_product_of_a_token_by_many_columns(exts, dev, M, N, K, fa):
    a, b = _operands(M, N, K, fa, dev)
    for out in (torch.float32, torch.bfloat16):
        _check(_product(exts, a, b, out), a, b)


@pytest.mark.parametrize("fa", [E4, E5], ids=["e4m3", "e5m2"])
@pytest.mark.parametrize("M,N,K", [(1490, 8210, 1408), (4000, 8100, 1280), (2048, 8192, 2048), (3800, 4111, 1536), (8000, 2000, 4224)])
def test_product_of_large_tiles(exts, dev, M, N, K, fa):
    """8-bit codes by 256 x 256 tiles: rows and columns past the end, odd numbers of blocks, one round and two."""
    a, b = _operands(M, N, K, fa, dev)
    _check(_product(exts, a, b), a, b)


@pytest.mark.parametrize("fa", [E2, E4], ids=["e2m1", "e4m3"])
@pytest.mark.parametrize("M,N", [(2100, 4400), (4200, 4400), (300, 1030), (1300, 1300), (40, 700)])
def test_product_long(exts, dev, M, N, fa):
    a, b = _operands(M, N, 8448, fa, dev)
    for out in (torch.float32, torch.bfloat16):
        _check(_product(exts, a, b, out), a, b)


@pytest.mark.parametrize("fa", [E2, E4], ids=["e2m1", "e4m3"])
@pytest.mark.parametrize("M,N,K,out", [(4096, 4118, 256, torch.bfloat16), (3000, 1297, 512, torch.float32)])
def test_product_in_two_launches(exts, dev, M, N, K, out, fa):
    """A few columns past a multiple of 256 run on tiles of their own."""
    a, b = _operands(M, N, K, fa, dev)
    _check(_product(exts, a, b, out), a, b)


@pytest.mark.parametrize("fa", [E2, E4], ids=["e2m1", "e4m3"])
@pytest.mark.parametrize("M,N,K", [(2499, 4090, 256), (2600, 2040, 768), (2590, 4090, 256), (1594, 4090, 256), (2756, 1500, 256), (2092, 450, 256),
                                   (2341, 200, 256), (2756, 130, 256), (1677, 130, 256)])
def test_product_of_one_round_of_tiles(exts, dev, M, N, K, fa):
    a, b = _operands(M, N, K, fa, dev)
    for out in (torch.float32, torch.bfloat16):
        _check(_product(exts, a, b, out), a, b)


@pytest.mark.parametrize("fa", [E2, E4], ids=["e2m1", "e4m3"])
@pytest.mark.parametrize("M,N,K", [(3, 200, 512), (150, 300, 256)])
def test_product_strides_and_scale_layouts(exts, dev, M, N, K, fa):
    """Codes in wider rows, scales in any layout: the same bits."""
    a, b = _operands(M, N, K, fa, dev)
    f = exts["proj"].fp4_matmul
    want = f(a.codes, a.scales, b.codes, b.scales)
    wide = lambda t, at: torch.nn.functional.pad(t.view(torch.uint8), (at, 48)).view(t.dtype)[:, at:at + t.shape[1]]  # noqa: E731
    assert torch.equal(f(wide(a.codes, 16), a.scales, wide(b.codes, 64), b.scales), want)
    assert torch.equal(f(a.codes, a.scales.contiguous(), b.codes, b.scales.contiguous()), want)
    assert torch.equal(f(a.codes, a.scales, b.codes, b.scales.flatten(1)), want)
    assert torch.equal(f(a.codes, a.scales, b.codes, wide(b.scales.flatten(1), 3)), want)
    if fa == E2:
        assert torch.equal(f(a.codes, a.scales.flatten(1), b.codes, b.scales), want)
    assert torch.equal(f(a.codes[:, :a.codes.shape[1]], a.scales, b.codes[5:], b.scales[5:]), f(a.codes, a.scales, b.codes[5:].clone(), words(b.scales.flatten(1)[5:])))


@pytest.mark.parametrize("fa", [E2, E4], ids=["e2m1", "e4m3"])
@pytest.mark.parametrize("M", [1, 2, 40, 300])
def test_product_of_nan(exts, dev, M, fa):
    """NaN scales (and codes of 8 bits) reach exactly the outputs whose sums meet them."""
    for out in (torch.bfloat16, torch.float32):
        a, b = _operands(M, 300, 512, fa, dev)
        clean = _product(exts, a, b, out)
        want = torch.zeros(M, 300, dtype=torch.bool)
        _bits_on = lambda s: s.view(torch.uint8)  # noqa: E731
        _bits_on(a.scales)[M - 1, 1] = 255
        _bits_on(b.scales)[17, 3, 2] = 255
        want[M - 1], want[:, 17] = True, True
        if fa == E4 and M > 1:
            _bits_on(a.codes)[0, 200] = 0x7f
            want[0] = True
        y = _product(exts, a, b, out)
        assert torch.equal(y.isnan().cpu(), want)
        assert torch.equal(y[~want.to(dev)], clean[~want.to(dev)])


def test_product_of_nothing(exts, dev):
    a, b = _operands(4, 32, 256, E2, dev)
    f = exts["proj"].fp4_matmul
    assert f(a.codes[:0], a.scales[:0], b.codes, b.scales).shape == (0, 32)
    assert f(a.codes, a.scales, b.codes[:0], b.scales[:0]).shape == (4, 0)
    q = exts["proj"].fp4_quantize(torch.zeros(0, 300, dtype=torch.bfloat16, device=dev), rows=True, columns=True)
    assert [tuple(t.shape) for t in q] == [(0, 256), (0, 4, 4), (300, 0), (300, 0, 4)]
    assert exts["proj"].fp4_dequantize(q[0], q[1], columns=300).shape == (0, 300)


@pytest.mark.parametrize("fa", [E2, E4], ids=["e2m1", "e4m3"])
def test_rows_do_not_depend_on_their_neighbours(exts, dev, fa):
    a, b = _operands(200, 300, 512, fa, dev)
    for out in (torch.bfloat16, torch.float32):
        want = _product(exts, a, b, out)
        s = a.scales.clone()
        s.view(torch.uint8)[100:] = 255
        assert torch.equal(exts["proj"].fp4_matmul(a.codes, s, b.codes, b.scales, out_dtype=out)[:100], want[:100])
        assert torch.equal(_product(exts, a, b, out), want)


@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("fa", [E2, E4, E5], ids=["e2m1", "e4m3", "e5m2"])
@pytest.mark.parametrize("M,N,K", [(1, 300, 2048), (2, 70, 2048), (16, 129, 2048), (40, 100, 2048), (70, 2048, 2048), (300, 1030, 2048),
                                   (700, 2100, 2048), (1594, 4090, 512), (4100, 4090, 512)])
def test_product_of_far_scales(exts, dev, M, N, K, fa, out):
    """Scales far from 1 that one operand's and the other's bring back together."""
    a, b = _operands(M, N, K, fa, dev)
    g = torch.Generator().manual_seed(K)
    mid = torch.linspace(6, 248, K // 128).round().int()
    near = lambda rows, n, at: (at[None, :, None] + torch.randint(-4, 5, (rows, K // 128, n), generator=g)).clamp(0, 250).to(torch.uint8)  # noqa: E731
    sa, sb = near(M, 4 if fa == E2 else 1, mid), near(N, 4, 254 - mid)
    of = lambda s: torch.ldexp(torch.ones(s.shape, dtype=torch.float64), s.int() - 127).flatten(1)  # noqa: E731
    old_a = a.scales.double().flatten(1)
    a.values = a.values / old_a.repeat_interleave(K // old_a.shape[1], 1) * of(sa).to(dev).repeat_interleave(K // (sa[0].numel()), 1)
    b.values = b.values / b.scales.double().flatten(1).repeat_interleave(32, 1)[:, :K] * of(sb).to(dev).repeat_interleave(32, 1)
    a.scales = words(sa.flatten(1).view(E8).to(dev)) if fa == E2 else sa[:, :, 0].contiguous().view(E8).to(dev)
    b.scales = words(sb.flatten(1).view(E8).to(dev))
    _check(_product(exts, a, b, out), a, b)


@pytest.mark.parametrize("M,N,K", [(1, 300, 512), (16, 129, 1152), (70, 2048, 512), (300, 1030, 512), (520, 4090, 384), (2600, 2040, 384)])
def test_product_of_large_terms_that_cancel(exts, dev, M, N, K):
    """In every block two products of 448 and 6 take each other away and the rest is small
    beside them: bf16 results are within the bound of what the instruction drops, fp32
    results have all of it."""
    g = torch.Generator().manual_seed(M)
    small = torch.tensor([-0.0625, -0.03125, 0.03125, 0.0625])
    a, b = _operands(M, N, K, E4, dev)
    va = small[torch.randint(0, 4, (M, K), generator=g)]
    cb = torch.randint(0, 2, (N, b.codes.shape[1] * 2), generator=g)
    for k in range(0, K, 128):
        at = torch.randperm(32, generator=g)[:2] + k
        va[:, at] = 448.0
        cb[:, at[0]], cb[:, at[1]] = 7, 15
    cb[:, K:] = 0
    a.codes, b.codes = va.to(E4).to(dev), pack(cb).to(dev)
    sb = b.scales.flatten(1).contiguous()
    a.values = a.codes.double() * a.scales.double().repeat_interleave(128, 1)
    b.values = values(cb, _bits(sb))[:, :K].to(dev)
    for out in (torch.bfloat16, torch.float32):
        _check(_product(exts, a, b, out), a, b)


@pytest.mark.parametrize("kind", ["cancel", "one sign"])
@pytest.mark.parametrize("M,N,K", [(1, 300, 512), (2, 70, 2048), (16, 129, 1280), (48, 2048, 4096), (70, 2048, 512), (300, 1030, 512), (520, 4090, 512),
                                   (2600, 2040, 512), (4096, 4118, 256)])
def test_product_of_4_bit_codes_loses_little_beside_the_largest(exts, dev, M, N, K, kind):
    """One instruction (128 products and the accumulator) is off by at most 2^-21 of the
    largest of: its products, their four sums of 32, the accumulator, the result.  No
    accumulator or result is larger than the sum of the instructions' magnitudes, nor any
    of at most eight partial sums that are added in fp32 (2^-24 each).  Scales lie up to
    2^78 apart; in every block of 128 products of 36 and -36 times the scales cancel, or
    none do."""
    g = torch.Generator().manual_seed(M + K)
    a, b = _operands(M, N, K, E2, dev, lo=107, hi=147)
    ca, cb = (torch.randint(0, 16, (n, K), generator=g) for n in (M, N))
    if kind == "one sign":
        ca, cb = ca & 7, cb & 7
    else:
        for k in range(0, K, 128):
            at = k + 32 * torch.randint(0, 4, (1,), generator=g) + torch.randperm(32, generator=g)[:2]
            ca[:, at], cb[:, at[0]], cb[:, at[1]] = 7, 7, 15
    sa, sb = (_bits(t.scales.flatten(1).contiguous()) for t in (a, b))
    a.codes, b.codes = pack(ca).to(dev), pack(cb).to(dev)
    a.values, b.values = values(ca, sa).to(dev), values(cb, sb).to(dev)
    ref, sums, largest = (torch.zeros(M, N, dtype=torch.float64, device=dev) for _ in range(3))
    for k in range(0, K, 128):
        parts = [a.values[:, i:i + 32] @ b.values[:, i:i + 32].t() for i in range(k, k + 128, 32)]
        # of 32 products the largest is no larger than the product of the largest two
        tops = [a.values[:, i:i + 32].abs().amax(1)[:, None] * b.values[:, i:i + 32].abs().amax(1) for i in range(k, k + 128, 32)]
        ref, sums = ref + sum(parts), sums + sum(parts).abs()
        largest = largest + torch.stack([p.abs() for p in parts] + tops).amax(0)
    tol = 2.0 ** -21 * (largest + (K / 128 + 1) * sums * (1 + 2.0 ** -10))
    for out in (torch.float32, torch.bfloat16):
        y = _product(exts, a, b, out).double()
        far = (y - ref).abs() - tol - (2.0 ** -8 * (ref.abs() + tol) if out == torch.bfloat16 else 0)
        assert not (far > 0).any() and torch.isfinite(y).all(), f"{(far > 0).sum().item()} values of {out}, the worst {far.max().item():.3g} past its bound"


def test_quantised_operands_go_straight_in(exts, dev):
    """The codes of block_norm, fp8_quantize and fp4_quantize as they come, K no multiple of 256."""
    g = torch.Generator().manual_seed(8)
    x, w = (torch.randn(n, 1100, generator=g).to(torch.bfloat16).to(dev) for n in (70, 330))
    wc, ws = exts["proj"].fp4_quantize(w)
    wv = exts["proj"].fp4_dequantize(wc, ws, columns=1100, dtype=torch.float32).double()
    q8, q4 = exts["proj"].fp8_quantize(x), exts["proj"].fp4_quantize(x)
    _, _, nc, ns = exts["rmsnorm"].block_norm(x, gamma=torch.ones(1100, dtype=torch.bfloat16, device=dev), quantize=True)
    for codes, scales in (q8, q4, (nc, ns)):
        if codes.dtype == E2:
            v = exts["proj"].fp4_dequantize(codes, scales, columns=1100, dtype=torch.float32).double()
        else:
            v = (codes.double() * scales.double().repeat_interleave(128, 1))[:, :1100]
        y = exts["proj"].fp4_matmul(codes, scales, wc, ws, out_dtype=torch.float32)
        tol = (1280 + 18) * 2.0 ** -23 * (v.abs() @ wv.abs().t())  # either bound above, at K = 1280
        assert ((y.double() - v @ wv.t()).abs() <= tol).all()


def test_offsets_past_32_bits(exts, dev):
    """A weight of more than 2^32 bytes of codes and results of more than 2^32 bytes."""
    N, K, M = 600_000, 16384, 40
    codes = torch.zeros(N, K // 2, dtype=torch.uint8, device=dev)
    scales = torch.full((K // 128, up(N, 16), 4), 127, dtype=torch.uint8, device=dev)
    rows = torch.tensor([0, 5, 262143, 262144, 524288, 524289, N - 1], device=dev)
    g = torch.Generator().manual_seed(5)
    some = torch.randint(0, 256, (len(rows), K // 2), generator=g).to(torch.uint8).to(dev)
    codes[rows] = some
    s = scales.view(E8)[:, :N].transpose(0, 1)
    for M in (2, 40):
        x = torch.randn(M, K, generator=g).to(torch.bfloat16).to(dev)
        xc, xs = exts["proj"].fp4_quantize(x)
        y = exts["proj"].fp4_matmul(xc, xs, codes.view(E2), s)
        part = exts["proj"].fp4_matmul(xc, xs, some.view(E2), words(torch.full((len(rows), K // 32), 127, dtype=torch.uint8, device=dev).view(E8)),
                                       out_dtype=torch.float32)
        assert ((y[:, rows].float() - part).abs() <= 2.0 ** -7 * part.abs() + 2.0 ** -10).all()
        rest = torch.ones(N, dtype=torch.bool, device=dev)
        rest[rows] = False
        assert (y[:, rest] == 0).all()
    v = exts["proj"].fp4_dequantize(codes.view(E2)[-70000:], s[-70000:])  # 2.3 GB of results
    want = exts["proj"].fp4_dequantize(some[-1:].view(E2), s[:1])
    assert torch.equal(v[-1:], want)


def test_on_another_stream_and_replayed(exts, dev):
    x = torch.randn(130, 512, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).to(dev)
    w = torch.randn(300, 512, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).to(dev)
    wq, ws = exts["proj"].fp4_quantize(w, block_rows=32)

    def f():
        return exts["proj"].fp4_matmul(*exts["proj"].fp8_quantize(x), wq, ws), exts["proj"].fp4_matmul(*exts["proj"].fp4_quantize(x), wq, ws)

    eager = f()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = f()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(there, eager))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = f()
    for _ in range(3):
        for t in y:
            t.fill_(7.0)
        graph.replay()
        exts["proj"].fp4_matmul(*exts["proj"].fp8_quantize(w), wq, ws)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(y, eager))


# Kernels of the product by size: a token or two, rings of small tiles, the stream's tiles (inside the
# result and past it, with columns in a launch of their own), the phased ones.
SPREAD = [(1, 300, 512, E2), (2, 9001, 384, E4), (5, 33, 512, E2), (33, 65, 256, E5), (300, 1030, 512, E2), (513, 2100, 256, E4), (1030, 2050, 512, E2),
          (2600, 2040, 768, E4), (4096, 4118, 256, E2), (1490, 8210, 1408, E4)]


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("M,N,K,fa", SPREAD, ids=str)
def test_product_into_wider_rows_at_odd_addresses(exts, dev, M, N, K, fa, out):
    """Through the C ABI: results at any address of their type, in rows further apart than they
    are long, have the same bits; what lies around them is left as it is."""
    a, b = _operands(M, N, K, fa, dev)
    want = _product(exts, a, b, out)
    sa = a.scales
    if fa != E2:  # as fp8_quantize lays them out
        sa = torch.full((K // 128, up(M, 16)), 255, dtype=torch.uint8, device=dev)
        sa[:, :M] = a.scales.view(torch.uint8).t()
    for ldo, at in ((N + 3, 1), (N + 8, 5), (N, 3)):
        buf = torch.full((at + M * ldo + 7,), 7.0, dtype=out, device=dev)
        print(f"{M} x {N} x {K} {fa} {out} rows of {ldo} from {at}", flush=True)
        abi.call("gdn_fp4_matmul_hip", a.codes.data_ptr(), a.codes.shape[1], {E4: 0, E5: 1, E2: 2}[fa], sa.data_ptr(), up(M, 16), b.codes.data_ptr(),
                 b.codes.shape[1], b.scales.data_ptr(), up(N, 16), buf[at:].data_ptr(), ldo, 1 if out == torch.float32 else 0, M, N, K,
                 torch.cuda.current_stream().cuda_stream)
        rows = buf[at:at + M * ldo].view(M, ldo)
        assert torch.equal(rows[:, :N], want)
        assert (rows[:, N:] == 7).all() and (buf[:at] == 7).all() and (buf[at + M * ldo:] == 7).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("M,K", [(1, 1), (1, 37), (3, 256), (70, 1001), (33, 2048)])
def test_dequantize_into_wider_rows_at_odd_addresses(exts, dev, M, K, dtype):
    """The same of the way back."""
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(M)).to(dev)
    codes, scales = exts["proj"].fp4_quantize(x)
    want = exts["proj"].fp4_dequantize(codes, scales, columns=K, dtype=dtype)
    for ldo, at in ((K + 3, 1), (K + 9, 5), (K, 3)):
        buf = torch.full((at + M * ldo + 7,), 77.0, dtype=dtype, device=dev)
        abi.call("gdn_fp4_dequantize_hip", codes.data_ptr(), codes.shape[1], scales.data_ptr(), up(M, 16), buf[at:].data_ptr(), ldo,
                 1 if dtype == torch.float32 else 0, M, K, torch.cuda.current_stream().cuda_stream)
        rows = buf[at:at + M * ldo].view(M, ldo)
        assert torch.equal(rows[:, :K], want)
        assert (rows[:, K:] == 77).all() and (buf[:at] == 77).all() and (buf[at + M * ldo:] == 77).all()


@pytest.mark.parametrize("M,N,K,fa,out", [(16500, 131101, 256, E2, torch.bfloat16), (16500, 131101, 1280, E4, torch.bfloat16), (16500, 65601, 256, E4, torch.float32),
                                          (16500, 65601, 256, E2, torch.float32), (40, 54_000_011, 256, E2, torch.bfloat16)],
                         ids=["stream", "phased", "ring", "stream fp32", "few rows"])
def test_results_past_32_bits(exts, dev, M, N, K, fa, out):
    """Results of more than 2^32 bytes, of codes whose sums (quarters below 2^14 in magnitude) are
    exact in fp32: rows from all over them have the bits that they have alone, in columns from
    all over them."""
    g = torch.Generator(device=dev).manual_seed(M)
    codes_b = torch.randint(0, 256, (N, K // 2), generator=g, device=dev, dtype=torch.uint8)
    sb = torch.full((K // 128, up(N, 16), 4), 127, dtype=torch.uint8, device=dev).view(E8)[:, :N].transpose(0, 1)
    if fa == E2:
        codes_a = torch.randint(0, 256, (M, K // 2), generator=g, device=dev, dtype=torch.uint8).view(E2)
        sa = torch.full((K // 128, up(M, 16), 4), 127, dtype=torch.uint8, device=dev).view(E8)[:, :M].transpose(0, 1)
    else:  # 0, 1/2 .. 2 in magnitude
        codes_a = (torch.randint(-4, 5, (M, K), generator=g, device=dev).float() / 2).to(fa)
        sa = torch.full((K // 128, up(M, 16)), 127, dtype=torch.uint8, device=dev).view(E8)[:, :M].t()
    y = exts["proj"].fp4_matmul(codes_a, sa, codes_b.view(E2), sb, out_dtype=out)
    size = 4 if out == torch.float32 else 2
    border = 2 ** 32 // size // N  # the row that 2^32 bytes end in
    assert border < M
    row = torch.tensor(sorted({0, 1, M // 3, M // 2, border, M - 2, M - 1}), device=dev)
    col = torch.unique(torch.cat([torch.arange(0, N, max(1, N // 500), device=dev), torch.arange(max(0, N - 300), N, device=dev)]))
    four = lambda bytes_: exts["proj"].fp4_dequantize(bytes_.view(E2), torch.full((len(bytes_), K // 32), 127, dtype=torch.uint8, device=dev).view(E8), dtype=torch.float32)  # noqa: E731
    va, vb = four(codes_a.view(torch.uint8)[row]) if fa == E2 else codes_a.float()[row], four(codes_b[col])
    want = (va.double() @ vb.double().t()).float().to(out)
    assert torch.equal(y[row][:, col], want)


def test_dequantized_values_past_32_bits(exts, dev):
    """2.3 billion values, 4.6 GB of bf16."""
    M, K = 140_000, 16384
    codes, scales = torch.zeros(M, K // 2, dtype=torch.uint8, device=dev), torch.full((K // 128, up(M, 16), 4), 127, dtype=torch.uint8, device=dev)
    rows = torch.tensor([0, 65535, 131071, 131072, M - 1], device=dev)
    some = torch.randint(0, 256, (len(rows), K // 2), generator=torch.Generator().manual_seed(5)).to(torch.uint8).to(dev)
    codes[rows] = some
    s = scales.view(E8)[:, :M].transpose(0, 1)
    v = exts["proj"].fp4_dequantize(codes.view(E2), s)
    assert v.numel() * 2 > 2 ** 32 and torch.equal(v[rows], exts["proj"].fp4_dequantize(some.view(E2), s[:len(rows)]))
    assert torch.count_nonzero(v).item() == torch.count_nonzero(v[rows]).item()


@pytest.mark.parametrize("block", [1, 32])
def test_quantized_values_past_32_bits(exts, dev, block):
    """2.2 billion values, 4.3 GB of bf16: rows and columns from all over them have the codes that they have alone."""
    M, K = 262_200, 8320
    x = torch.randn(1024, K, generator=torch.Generator().manual_seed(6)).to(torch.bfloat16).to(dev).repeat(257, 1)[:M]
    x[-1, -1] = 40.0  # no period in the last row's or column's block
    assert x.numel() * 2 > 2 ** 32
    c, s, ct, st = exts["proj"].fp4_quantize(x, block_rows=block, rows=True, columns=True)
    for lo, hi in ((0, 64), (131072, 131136), (261_952, M)):  # of whole blocks
        part = exts["proj"].fp4_quantize(x[lo:hi].clone(), block_rows=block, rows=True, columns=True)
        assert torch.equal(_bits(c[lo:hi]), _bits(part[0])) and torch.equal(_bits(s[lo:hi]), _bits(part[1]))
        n = (hi - lo + 1) // 2
        assert torch.equal(_bits(ct.view(torch.uint8)[:, lo // 2:lo // 2 + n]), _bits(part[2])[:, :n])
        blocks_t = st.view(torch.uint8).flatten(1)[:, lo // 32:-(-hi // 32)]
        assert torch.equal(blocks_t.cpu(), _bits(part[3]).flatten(1)[:, :blocks_t.shape[1]])
