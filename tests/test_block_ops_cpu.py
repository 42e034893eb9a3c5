"""Refusals of the block norms, the fp8 quantisation and the fp8 product: every
bad call is turned down on the host, before any HIP call (none runs here)."""

import pytest
import torch

from gdn_18646_amd import abi, compile_kernels
from gdn_18646_amd.abi import GdnError

FAKE = 4096  # non-null, aligned; never dereferenced
BF, F32, E8 = 0, 1, 2


def _norm(**k):
    a = dict(y=FAKE, ldy=256, residual=FAKE, ldr=256, gate=FAKE, ldg=256, rpg=1, post=FAKE, gamma=FAKE, scale=FAKE, rs=1.0,
             act=2, eps=1e-6, h=FAKE, ldh=256, n=FAKE, ldn=256, codes=None, ldc=0, scales=None, lds=0, ry=None, rh=None,
             R=4, D=256, ty=BF, tr=BF, tp=BF, stream=None)
    assert set(k) <= set(a)
    a.update(k)
    abi.call("gdn_block_norm_hip", *a.values())


@pytest.mark.parametrize("bad,match", [
    (dict(R=-1), "INVALID_ARGUMENT"), (dict(D=0), "INVALID_ARGUMENT"), (dict(D=16385), "UNSUPPORTED.*16384"),
    (dict(R=1 << 31), "UNSUPPORTED"), (dict(R=(1 << 31) - 1), "too many"), (dict(ty=F32), "UNSUPPORTED.*types"), (dict(tp=3), "UNSUPPORTED.*types"),
    (dict(tr=F32), "UNSUPPORTED.*types"), (dict(act=4), "act=4"), (dict(y=None), "null"), (dict(h=None, n=None), "null"),
    (dict(gamma=None), "need gamma"), (dict(gamma=None, n=None, rh=FAKE), "need gamma"), (dict(post=None, ry=FAKE), "needs post_gamma"),
    (dict(rpg=0), "rows_per_gate"), (dict(codes=FAKE), "codes"), (dict(codes=FAKE, scales=FAKE, ldc=128, lds=4), "codes"),
    (dict(codes=FAKE, scales=FAKE, ldc=256, lds=3), "codes"), (dict(codes=FAKE + 8, scales=FAKE, ldc=256, lds=4), "codes"),
    (dict(y=FAKE + 1), "aligned"), (dict(gamma=FAKE + 1), "aligned")])
def test_block_norm_refusals(bad, match):
    with pytest.raises(GdnError, match=match):
        _norm(**bad)


@pytest.mark.parametrize("over,name", [
    (dict(y=FAKE + 1024), "y"),                          # rows of one buffer, a row on (rows 1024 bytes apart)
    (dict(y=FAKE - 1024), "y"),
    (dict(y=FAKE + 256), "y"),                           # columns of the same rows, half a row on
    (dict(y=FAKE + 768), "y"),                           # past the row's end into the next one
    (dict(y=FAKE + 512, ldy=320), "y"),                  # steps that have 128 bytes in common
    (dict(y=FAKE, ldy=256), "y"),                        # the same place, another step
    (dict(residual=FAKE + 1024), "residual"),
    (dict(gate=FAKE + 2048), "gate"),
    (dict(gate=FAKE, rpg=2), "gate"),                    # rows 0 and 1 are read by others
    (dict(gate=FAKE, rpg=4), "gate"),
    (dict(post=FAKE), "post_gamma"), (dict(gamma=FAKE + 2048), "gamma"), (dict(scale=FAKE + 1500), "scale")])
def test_block_norm_refuses_h_over_what_others_read(over, name):
    """h in every second 512 bytes of a buffer, at FAKE; the other operands elsewhere."""
    far = dict(y=1 << 20, residual=FAKE, ldr=512, ldy=512, ldg=512, gate=2 << 20, post=3 << 20, gamma=3 << 20, scale=3 << 20, h=FAKE, ldh=512,
               n=4 << 20)
    with pytest.raises(GdnError, match=f"INVALID_ARGUMENT.*memory locations of {name} "):
        _norm(**{**far, **over})


@pytest.mark.parametrize("bad", [dict(ldh=255), dict(ldh=0), dict(ldh=-256), dict(ldn=255), dict(ldn=0)])
def test_block_norm_refuses_results_whose_rows_overlap(bad):
    apart = dict(residual=1 << 20, gate=1 << 21, y=1 << 22, post=1 << 23, gamma=1 << 23, scale=1 << 23)
    with pytest.raises(GdnError, match="INVALID_ARGUMENT.*overlap"):
        _norm(**apart, **bad)


def test_no_rows_is_no_call():
    _norm(R=0, residual=None)
    _norm(R=0, y=None)


def _bwd(**k):
    a = dict(dh=FAKE, lddh=256, dn=FAKE, lddn=256, y=FAKE, ldy=256, residual=FAKE, ldr=256, gate=FAKE, ldg=256, rpg=1, post=FAKE,
             gamma=FAKE, scale=FAKE, rs=1.0, act=2, ry=FAKE, rh=FAKE, dres=FAKE, dy=FAKE, dgate=FAKE, dpost=FAKE, dgamma=FAKE,
             dscale=FAKE, R=4, D=256, ty=BF, tr=BF, tp=BF, ws=FAKE, bytes=1 << 30, stream=None)
    assert set(k) <= set(a)
    a.update(k)
    abi.call("gdn_block_norm_bwd_hip", *a.values())


@pytest.mark.parametrize("bad,match", [
    (dict(R=-1), "INVALID_ARGUMENT"), (dict(D=20000), "UNSUPPORTED"), (dict(tr=F32), "types"), (dict(act=-1), "act"),
    (dict(rpg=0), "rows_per_gate"), (dict(rh=None), "go together"), (dict(gamma=None, dgamma=None), "go together"),
    (dict(dn=None), "go together"), (dict(ry=None), "go together"), (dict(gate=None), "absent input"),
    (dict(residual=None), "absent input"), (dict(scale=None), "absent input"), (dict(dy=None), "null"), (dict(y=None), "null"),
    (dict(dh=None, dn=None, gamma=None, rh=None, dgamma=None), "null"), (dict(dy=FAKE + 1), "aligned"),
    (dict(bytes=64), "WORKSPACE"), (dict(ws=None), "WORKSPACE"), (dict(R=200000, rpg=2), "gate rows")])
def test_block_norm_backward_refusals(bad, match):
    with pytest.raises(GdnError, match=match):
        _bwd(**bad)


def test_backward_workspace_covers_the_launch():
    """Two fp32 sums a column for each workgroup, at most 512 of them and one a
    row group; one set more a gate row where rows share over 32 gate rows."""
    f = abi.load().gdn_block_norm_bwd_workspace_bytes
    assert f(0, 256, 1) == 0
    assert f(16384, 2048, 1) == 512 * 2 * 2048 * 4
    assert f(3, 2048, 1) == 3 * 2 * 2048 * 4
    assert f(16384, 2048, 4096) == 512 * 2 * 2048 * 4
    assert f(16384, 2048, 256) == (512 + 64) * 2 * 2048 * 4
    assert f(100, 128, 100) == 7 * 2 * 128 * 4


def _quant(**k):
    a = dict(x=FAKE, ldx=300, type=BF, M=200, K=300, block=1, fmt=0, codes=FAKE, ldc=384, scales=FAKE, lds=208, codes_t=FAKE,
             ldt=256, scales_t=FAKE, ldst=304, stream=None)
    assert set(k) <= set(a)
    a.update(k)
    abi.call("gdn_fp8_quantize_hip", *a.values())


@pytest.mark.parametrize("bad,match", [
    (dict(M=-1), "INVALID_ARGUMENT"), (dict(block=64), "UNSUPPORTED.*64 x 128"), (dict(type=2), "type 2"), (dict(fmt=2), "format 2"),
    (dict(M=1 << 31), "too large"), (dict(codes=None, codes_t=None), "no output"), (dict(x=None), "null"), (dict(ldx=299), "ldx"),
    (dict(x=FAKE + 1), "unaligned"), (dict(ldc=368), "codes"), (dict(ldc=392), "codes"), (dict(lds=200), "codes"),
    (dict(scales=None), "codes"), (dict(codes=FAKE + 8), "codes"), (dict(ldt=240), "codes_t"), (dict(ldst=299), "codes_t"),
    (dict(block=128, lds=2), "codes"), (dict(block=128, ldst=1, lds=3), "codes_t")])
def test_quantize_refusals(bad, match):
    with pytest.raises(GdnError, match=match):
        _quant(**bad)


def test_quantize_nothing():
    _quant(M=0)
    _quant(K=0)


def _mm(**k):
    a = dict(a=FAKE, lda=256, fa=0, sa=FAKE, ldas=48, b=FAKE, ldb=256, fb=0, sb=FAKE, ldbs=2, brows=128, tsb=E8, out=FAKE, ldo=100,
             to=BF, M=40, N=100, K=256, stream=None)
    assert set(k) <= set(a)
    a.update(k)
    abi.call("gdn_fp8_matmul_hip", *a.values())


@pytest.mark.parametrize("bad,match", [
    (dict(M=-1), "INVALID_ARGUMENT"), (dict(K=0), "INVALID_ARGUMENT"), (dict(K=200), "multiple of 128"), (dict(fa=2), "formats"),
    (dict(fb=-1), "formats"), (dict(brows=64), "UNSUPPORTED.*64 x 128"), (dict(tsb=BF), "type 0 of b"), (dict(to=E8), "type 2 of out"),
    (dict(lda=1 << 23), "too large"), (dict(M=1 << 31), "too large"), (dict(a=None), "null"), (dict(sb=None), "null"),
    (dict(out=None), "null"), (dict(a=FAKE + 8), "16-byte"), (dict(ldb=240), "16-byte"), (dict(ldb=264), "16-byte"),
    (dict(ldas=32), "a's scales"), (dict(ldas=40), "a's scales"), (dict(sa=FAKE + 4), "a's scales"), (dict(ldbs=1), "b's scales"),
    (dict(brows=1, ldbs=96), "b's scales"), (dict(brows=1, ldbs=104), "b's scales"), (dict(tsb=F32, sb=FAKE + 2), "b's scales"),
    (dict(ldo=99), "ldo"), (dict(M=1, N=1 << 30, ldo=1 << 30), "N=.*too large for a launch"), (dict(out=FAKE + 1), "unaligned")])
def test_product_refusals(bad, match):
    with pytest.raises(GdnError, match=match):
        _mm(**bad)


def test_product_refuses_scales_past_32_bit_offsets():
    N = (1 << 30) + 16
    wide = dict(brows=1, tsb=F32, M=3, N=N, ldbs=N, ldo=N)
    with pytest.raises(GdnError, match="UNSUPPORTED.*2.30 columns"):
        _mm(**wide)
    for other in (dict(N=1 << 30), dict(tsb=E8), dict(brows=128, ldbs=2)):  # these are told of another fault
        with pytest.raises(GdnError, match="null"):
            _mm(**{**wide, **other, "a": None})


def test_product_of_nothing():
    _mm(M=0)
    _mm(N=0)


def test_binding_refusals_on_the_host():
    e = compile_kernels()
    y = torch.zeros(4, 256, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        e["rmsnorm"].block_norm(y)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        e["rmsnorm"].block_norm_backward(y, None, y)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        e["proj"].fp8_quantize(y)
    with pytest.raises(RuntimeError, match="GPU tensors"):
        e["proj"].fp8_matmul(y, y, y, y)


def test_inplace_over_a_residual_that_requires_grad_is_refused():
    f = compile_kernels()["rmsnorm"].block_norm
    y = torch.zeros(4, 256, dtype=torch.bfloat16)
    leaf = torch.zeros(4, 256, dtype=torch.bfloat16, requires_grad=True)
    for r in (leaf, leaf * 2, leaf[:]):
        with pytest.raises(RuntimeError, match="requires grad"):
            f(y, residual=r, inplace=True)
        with torch.no_grad(), pytest.raises(RuntimeError, match="GPU tensor"):  # past that check
            f(y, residual=r, inplace=True)
