"""Refusals of the 4-bit quantisation, product and the gradients' norm: every bad call
is turned down on the host, before any HIP call (none runs here).  And what the 4-bit
kernels' counted waits rest on, in their assembly."""

import ctypes
import re

import pytest
import torch
from torch.autograd import forward_ad

from gdn_18646_amd import abi, blocks, compile_kernels, native_extension
from gdn_18646_amd.abi import GdnError, GradTensor
from tests.fp4 import nearest, pack, quantize64, unpack, values
from tests.test_isa_cpu import _assembly, _function

FAKE = 4096  # non-null, aligned; never dereferenced
BF, F32, E8 = 0, 1, 2
E4M3, E2M1 = 0, 2


def _quant(**k):
    a = dict(x=FAKE, ldx=300, type=BF, M=200, K=300, block=1, codes=FAKE, ldc=256, scales=FAKE, lds=200, codes_t=FAKE, ldt=128, scales_t=FAKE, ldst=300,
             stream=None)
    assert set(k) <= set(a)
    a.update(k)
    abi.call("gdn_fp4_quantize_hip", *a.values())


@pytest.mark.parametrize("bad,match", [
    (dict(M=-1), "INVALID_ARGUMENT"), (dict(block=128), "UNSUPPORTED.*128 x 32"), (dict(type=2), "type 2"), (dict(M=1 << 31), "too large"),
    (dict(K=1 << 31), "too large"), (dict(codes=None, codes_t=None), "no output"), (dict(x=None), "null"), (dict(ldx=299), "ldx"), (dict(x=FAKE + 1), "unaligned"),
    (dict(ldc=240), "codes"), (dict(ldc=264), "codes"), (dict(lds=199), "codes"), (dict(scales=None), "codes"), (dict(codes=FAKE + 8), "codes"),
    (dict(scales=FAKE + 2), "codes"), (dict(ldt=112), "codes_t"), (dict(ldst=299), "codes_t"), (dict(scales_t=None), "codes_t")])
def test_quantize_refusals(bad, match):
    with pytest.raises(GdnError, match=match):
        _quant(**bad)


def _quant48(**k):
    a = dict(x=FAKE, ldx=300, type=BF, M=200, K=300, codes=FAKE, ldc=256, scales=FAKE, lds=200, codes_t=FAKE, ldt=256, scales_t=FAKE, ldst=300, stream=None)
    assert set(k) <= set(a)
    a.update(k)
    abi.call("gdn_fp4_fp8_quantize_hip", *a.values())


@pytest.mark.parametrize("bad,match", [
    (dict(M=-1), "INVALID_ARGUMENT"), (dict(type=2), "type 2"), (dict(M=1 << 31), "too large"), (dict(K=1 << 31), "too large"), (dict(x=None), "null"),
    (dict(ldx=299), "ldx"), (dict(x=FAKE + 1), "unaligned"), (dict(codes=None), "codes "), (dict(ldc=240), "codes "), (dict(lds=199), "codes "),
    (dict(scales=FAKE + 2), "codes "), (dict(codes_t=None), "codes_t"), (dict(codes_t=FAKE + 8), "codes_t"), (dict(ldt=240), "codes_t"),
    (dict(ldt=264), "codes_t"), (dict(ldst=299), "codes_t"), (dict(scales_t=None), "codes_t")])
def test_quantize_to_both_formats_refusals(bad, match):
    with pytest.raises(GdnError, match=match):
        _quant48(**bad)
    _quant48(M=0)
    _quant48(K=0)


def _dequant(**k):
    a = dict(codes=FAKE, ldc=152, scales=FAKE, lds=200, out=FAKE, ldo=300, to=BF, M=200, K=300, stream=None)
    assert set(k) <= set(a)
    a.update(k)
    abi.call("gdn_fp4_dequantize_hip", *a.values())


@pytest.mark.parametrize("bad,match", [
    (dict(M=-1), "INVALID_ARGUMENT"), (dict(to=E8), "type 2"), (dict(M=1 << 31), "too large"), (dict(codes=None), "codes"), (dict(codes=FAKE + 2), "codes"),
    (dict(ldc=148), "codes"), (dict(ldc=154), "codes"), (dict(scales=None), "scales"), (dict(lds=199), "scales"), (dict(out=None), "out"),
    (dict(out=FAKE + 1), "out"), (dict(ldo=299), "out")])
def test_dequantize_refusals(bad, match):
    with pytest.raises(GdnError, match=match):
        _dequant(**bad)


def _mm(**k):
    a = dict(a=FAKE, lda=256, fa=E2M1, sa=FAKE, ldas=48, b=FAKE, ldb=256, sb=FAKE, ldbs=112, out=FAKE, ldo=100, to=BF, M=40, N=100, K=512, stream=None)
    assert set(k) <= set(a)
    a.update(k)
    abi.call("gdn_fp4_matmul_hip", *a.values())


@pytest.mark.parametrize("bad,match", [
    (dict(M=-1), "INVALID_ARGUMENT"), (dict(K=0), "INVALID_ARGUMENT"), (dict(K=384), "multiple of 256"), (dict(fa=E4M3, K=200), "multiple of 128"),
    (dict(fa=3), "format 3"), (dict(to=E8), "type 2 of out"), (dict(lda=1 << 23), "too large"), (dict(M=1 << 29), "too large"), (dict(N=1 << 29), "too large"),
    (dict(ldbs=1 << 30), "too large"), (dict(M=1, N=1 << 28, ldbs=1 << 28, ldo=1 << 28), "too large for a launch"), (dict(a=None), "null"), (dict(sb=None), "null"), (dict(out=None), "null"), (dict(a=FAKE + 8), "16-byte"),
    (dict(ldb=240), "16-byte"), (dict(ldb=264), "16-byte"), (dict(fa=E4M3), "16-byte"), (dict(ldas=36), "a's scales"), (dict(ldas=42), "a's scales"),
    (dict(sa=FAKE + 4), "a's scales"), (dict(fa=E4M3, lda=512, ldas=40), "a's scales"), (dict(ldbs=96), "b's scales"), (dict(ldbs=102), "b's scales"),
    (dict(sb=FAKE + 8), "b's scales"), (dict(ldo=99), "ldo"), (dict(out=FAKE + 1), "unaligned"), (dict(fa=E4M3, K=384, lda=384, ldb=128), "16-byte")])
def test_product_refusals(bad, match):
    with pytest.raises(GdnError, match=match):
        _mm(**bad)


def test_nothing_to_do_is_no_call():
    _quant(M=0)
    _quant(K=0)
    _dequant(M=0)
    _dequant(K=0)
    _mm(M=0)
    _mm(N=0)


def _grads(entry, tensors, most=1.0, norm=FAKE, ws=FAKE, size=1 << 24, count=None):
    a = (GradTensor * max(len(tensors), 1))(*[GradTensor(*t) for t in tensors])
    clip = [most] if "clip" in entry else []
    abi.call(entry, ctypes.addressof(a), len(tensors) if count is None else count, *clip, norm, ws, size, None)


A, B = 1 << 20, 1 << 24


@pytest.mark.parametrize("tensors,kw,match", [
    ([(A, A, 10, F32, F32)], dict(count=-1), "INVALID_ARGUMENT.*-1 tensors"), ([(A, A, 10, F32, F32)], dict(norm=None), "null"),
    ([(A, A, 10, F32, F32)], dict(ws=None), "WORKSPACE"), ([(A, A, 10, F32, F32)], dict(size=16), "WORKSPACE"), ([(A, A, 10, F32, F32)], dict(ws=FAKE + 4), "WORKSPACE"),
    ([(A, A, 10, 2, F32)], {}, "UNSUPPORTED.*type"), ([(A, A, -1, F32, F32)], {}, "elements"), ([(A, A, 1 << 60, F32, F32)], {}, "elements"),
    ([(None, A, 10, F32, F32)], {}, "null or unaligned"), ([(A + 2, A, 10, F32, F32)], {}, "null or unaligned"), ([(A + 1, A, 10, BF, F32)], {}, "null or unaligned")])
@pytest.mark.parametrize("entry", ["gdn_grad_norm_hip", "gdn_clip_grad_norm_hip"])
def test_grad_refusals(entry, tensors, kw, match):
    with pytest.raises(GdnError, match=match):
        _grads(entry, tensors, **kw)


@pytest.mark.parametrize("tensors,kw,match", [
    ([(A, A, 10, F32, F32)], dict(most=-1.0), "max_norm"), ([(A, A, 10, F32, F32)], dict(most=float("nan")), "max_norm"),
    ([(A, A, 10, F32, 2)], {}, "UNSUPPORTED.*type"), ([(A, None, 10, F32, F32)], {}, "null or unaligned"),
    ([(A, A, 10, F32, BF)], {}, "lies over"),                                            # in place, of another type
    ([(A, A + 4, 10, F32, F32)], {}, "lies over"), ([(A + 4, A, 10, F32, F32)], {}, "lies over"),  # an element on
    ([(A, A, 10, F32, F32), (A, A, 10, F32, F32)], {}, "share memory"), ([(A, A, 10, F32, F32), (A + 36, A + 36, 10, F32, F32)], {}, "share memory"),
    ([(A, A, 1000, F32, F32), (A + 400, B, 10, F32, F32)], {}, "lies over"), ([(A, B, 10, F32, F32), (B + 39 - 3, A - 4000, 10, F32, F32)], {}, "lies over"),
    ([(A, B + 10000, 10, F32, F32), (A, B, 10, BF, F32), (B + 4, B - 10000, 10, BF, BF)], {}, "lies over")])
def test_clip_refuses_results_over_what_others_read(tensors, kw, match):
    with pytest.raises(GdnError, match=match):
        _grads("gdn_clip_grad_norm_hip", tensors, **kw)


def test_workspace_of_the_norm():
    f = abi.load().gdn_grad_norm_workspace_bytes
    assert f(0) == 8 and f(1) == f(128) == 2049 * 8 and f(129) == 4097 * 8 and f(-1) == 0


def test_binding_refusals_on_the_host():
    p, t = compile_kernels()["proj"], torch.zeros(4, 256, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        p.fp4_quantize(t)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        p.fp4_dequantize(t, t)
    with pytest.raises(RuntimeError, match="GPU tensors"):
        p.fp4_matmul(t, t, t, t)
    grads = native_extension().grads
    for call in (lambda: grads.norm([t]), lambda: grads.clip([t], 1.0)):
        with pytest.raises(RuntimeError, match="GPU tensor"):
            call()
    with pytest.raises(RuntimeError, match="no tensors"):
        grads.norm([])


def test_layers_check_their_arguments():
    x, w = torch.zeros(4, 256, dtype=torch.bfloat16), torch.zeros(8, 256, dtype=torch.bfloat16)
    for args, match in (((x, w[:, :128]), "weight"), ((x, w[0]), "weight"), ((x[0, 0], w), "weight"), ((x, w, torch.bfloat16), "activations")):
        with pytest.raises(ValueError, match=match):
            blocks.fp4_linear(*args)
    with pytest.raises(ValueError, match="weight"):
        blocks.Fp4Weight(w[0])
    assert blocks.grad_norm([]).item() == 0 and blocks.clip_grad_norm([None], 1.0).item() == 0


def test_tangents_of_gradients_are_not_dropped():
    t, plain = torch.ones(4, 5), torch.ones(4, 5)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(torch.ones(4, 5), t)
        for call in (lambda: blocks.grad_norm([dual]), lambda: blocks.grad_norm([dual, plain]), lambda: blocks.clip_grad_norm([dual], 0.5),
                     lambda: blocks.clip_grad_norm([dual, plain], 0.5)):
            for mode in (torch.enable_grad, torch.no_grad):
                with mode(), pytest.raises(RuntimeError, match="forward-mode tangent"):
                    call()
        assert torch.equal(forward_ad.unpack_dual(dual).primal, plain)


def test_the_definition_that_the_kernels_are_held_to():
    """Every value between two codes goes to the nearer one, ties to the even code."""
    v = torch.arange(-96, 97, dtype=torch.float64) / 16
    c = nearest(v)
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
    got = torch.where(c > 7, -1.0, 1.0) * table[(c & 7).long()]
    step = torch.where(v.abs() >= 4, 2.0, torch.where(v.abs() >= 2, 1.0, 0.5))
    assert torch.equal(got, torch.round(v / step) * step)
    x = torch.randn(3, 70, generator=torch.Generator().manual_seed(1), dtype=torch.float64)
    codes, scales = quantize64(x, 1)
    assert torch.equal(unpack(pack(codes)), codes)
    big = x[:, :64].view(3, 2, 32).abs().amax(2)
    s = torch.ldexp(torch.ones(3, 8, dtype=torch.float64), scales.int() - 127)
    assert (big <= 6 * s[:, :2]).all() and (big > 3 * s[:, :2]).all() and (scales[:, 3:] == 127).all()
    assert ((values(codes, scales)[:, :70] - x).abs() <= s.repeat_interleave(32, 1)[:, :70]).all()


# ---------------------------------------------------------------------------
# Assembly
# ---------------------------------------------------------------------------
# staged rows of a token, waves along columns, tokens, MFMA tiles of a wave along each, stages, workgroups on a CU
STREAM = {"e2m1 256x256": (0, 2, 4, 8, 4, 2, 1), "e2m1 128x128": (0, 2, 2, 4, 4, 2, 2), "e4m3 256x128": (1, 4, 2, 4, 4, 2, 1), "e4m3 128x64": (1, 2, 2, 4, 2, 2, 2)}


@pytest.fixture(scope="module")
def asm(tmp_path_factory):
    return {f: _assembly(f"fp4_mm_{f}.hip", tmp_path_factory) for f in ("e2m1", "e4m3")}


def _kernels(text, kind, tile=""):
    return re.findall(rf"^(_Z\w*gdn_fp4_{kind}_kernel\w*Fp4TileILb{tile}\w*):", text, re.M)


def test_no_tile_spills(asm):
    """And every copy into LDS has its base in scalar registers."""
    for text, stream, ring in ((asm["e2m1"], 2 * 2, 2 * 6), (asm["e4m3"], 2, 5 + 6)):
        kernels = _kernels(text, "stream"), _kernels(text, "ring")
        assert [len(k) for k in kernels] == [stream, ring]
        for name in sum(kernels, []):
            lines = _function(text, name)
            assert not any("scratch_" in ln for ln in lines), name
            assert not any("global_load_lds" in ln and "s[" not in ln for ln in lines), name


@pytest.mark.parametrize("tile", STREAM)
def test_stream_tiles_keep_their_counted_waits(asm, tile):
    """A stage's wait counts what has been issued since the copies that it waits for: the next
    W with its scales, and the stores of the tile before.  It holds if there are no fewer of
    them: all of a tile's products before its stores, at least as many stores as are counted,
    and no vector memory access of the compiler's own."""
    x8, cw, tw, wmt, wnt, ns, per = STREAM[tile]
    w, x = 2 * wmt // tw, 2 * wnt * (1 + x8) // cw  # 1 KiB copies of a wave: 16 wmt cw rows over 8 cw tw, and so on
    text = asm[tile.split()[0]]
    names = _kernels(text, "stream", "".join(("%dE" % x8, *(f"Li{v}E" for v in (cw, tw, wmt, wnt, ns, per)))))
    assert len(names) == (1 if x8 else 2), names  # bf16 and fp32 results
    for name in names:
        lines = _function(text, name)
        assert sum("v_mfma_scale" in ln for ln in lines) == 2 * wmt * wnt
        waits = {int(n) for ln in lines for n in re.findall(r"vmcnt\((\d+)\)", ln)}
        assert waits == {0, w + 2, 4 * wnt + w + 2, w + 2 + x}, waits
        last = max(i for i, ln in enumerate(lines) if "v_mfma" in ln)
        whole = [ln for ln in lines if re.search(r"global_store_dwordx[24]", ln)]
        assert len(whole) >= 2 * 4 * wnt  # inside the result, and at its edges
        assert not any(re.search(r"\bglobal_load_(?!lds)|\bflat_|\bbuffer_", ln) for ln in lines[:last])


def _stream_functions(asm, tile):
    x8, cw, tw, wmt, wnt, ns, per = STREAM[tile]
    text = asm[tile.split()[0]]
    names = _kernels(text, "stream", "".join(("%dE" % x8, *(f"Li{v}E" for v in (cw, tw, wmt, wnt, ns, per)))))
    assert len(names) == (1 if x8 else 2), names  # bf16 and fp32 results
    return [_function(text, name) for name in names]


@pytest.mark.parametrize("tile", STREAM)
def test_a_tile_inside_the_result_has_the_stores_that_are_counted(asm, tile):
    """The wait for a stage's copies lets the stores of a tile inside the result, 4 a token tile
    at least, be under way; those past the caches are that tile's (the edges' are ordinary)."""
    wnt = STREAM[tile][4]
    for lines in _stream_functions(asm, tile):
        stores = [ln for ln in lines if re.search(r"\bglobal_store_", ln)]
        inside = [i for i, ln in enumerate(lines) if re.search(r"\bglobal_store_\w+ .*\bnt\b", ln)]
        assert 4 * wnt <= len(inside) < len(stores)
        # all of them in one piece without branches: a tile issues them all or none
        assert not any(re.search(r"\bs_c?branch|^\.L", ln.strip()) for ln in lines[inside[0]:inside[-1]])


@pytest.mark.parametrize("tile", STREAM)
def test_stream_tiles_keep_their_counted_lds_wait(asm, tile):
    """The barrier after which W's buffer is copied over waits for all LDS reads but the last
    ones, which have to be of x: they lie behind products of the half slice, before which
    all of W and its scales were read, and no branch lies between."""
    x8, cw, tw, wmt, wnt, ns, per = STREAM[tile]
    first = wnt // 4  # the token tile behind whose reads the barrier stands
    for lines in _stream_functions(asm, tile):
        ops = [ln.split(";")[0].strip() for ln in lines]
        counted = [i for i, ln in enumerate(ops) if ln == "s_barrier" and (m := re.fullmatch(r"s_waitcnt lgkmcnt\((\d+)\)", ops[i - 1])) and m.group(1) != "0"]
        assert len(counted) == 1, counted
        at = counted[0] - 1
        n = int(re.search(r"\((\d+)\)", ops[at]).group(1))
        assert n == (first + 1) * (1 + x8)
        start = max(i for i in range(at) if re.search(r"^s_c?branch|^\.L\w+:", ops[i]))
        window = ops[start + 1:at]
        products = [i for i, ln in enumerate(window) if ln.startswith("v_mfma")]
        reads = [i for i, ln in enumerate(window) if ln.startswith("ds_")]
        assert len(products) == (first + 1) * wmt and all(window[i].startswith("ds_read") for i in reads)
        behind = [window[i] for i in reads if i > products[0]]
        before = [window[i] for i in reads if i < products[0]]
        assert len(behind) == n and all(ln.startswith("ds_read_b128") for ln in behind)
        assert sum(ln.startswith("ds_read_b128") for ln in before) == wmt  # W's codes
        assert len(before) > wmt                                          # and scales


def test_the_phased_tile(asm):
    """No spills, scalar bases, the counted waits of its phases, and none of the compiler's own before its stores."""
    (name,) = re.findall(r"^(_Z\w*gdn_fp4_phased_kernel\w*):", asm["e4m3"], re.M)
    lines = _function(asm["e4m3"], name)
    assert not any("scratch_" in ln for ln in lines) and not any("global_load_lds" in ln and "s[" not in ln for ln in lines)
    w, x, stages = 1, 2, 3  # copies of a region by a wave: 64 columns, 128 tokens a wave's part
    all_ = 2 * (w + x) + 2
    steady = {x + (stages - 1) * all_, x + 2 + (stages - 1) * all_, w + (stages - 1) * all_}
    last = {x + t * all_ for t in range(stages)} | {t * all_ for t in range(stages)} | {w + x + (t - 1) * all_ for t in range(1, stages)}
    assert {int(n) for ln in lines for n in re.findall(r"vmcnt\((\d+)\)", ln)} == steady | last | {0}
    assert sum("v_mfma_scale" in ln for ln in lines) == 4 * 8 * (1 + stages)
    assert not any(re.search(r"\bglobal_load_(?!lds)|\bflat_|\bbuffer_", ln) for ln in lines)
