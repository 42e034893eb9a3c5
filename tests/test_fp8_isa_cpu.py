"""ISA checks of the tiled fp8 product, on the CPU (hipcc cross-compiles gfx950).

Its phased tiles refill a stage's LDS buffer region by region and wait, before
the barrier that opens a phase, for the region that the next phase reads, by
counting the copies issued after it (vector memory operations retire in issue
order).  The counts hold only for these copies in this order: none moved over a
wait, merged or dropped.
"""

import re

import pytest

from tests.test_isa_cpu import _assembly, _events, _function

# columns: waves along columns, tokens, MFMA tiles of a wave along each, stages
PHASED = {"256x256": (4, 2, 4, 8, 2), "256x192": (4, 2, 4, 6, 2), "256x160": (4, 2, 4, 5, 2), "256x128": (4, 2, 4, 4, 3),
          "128x192": (2, 4, 4, 3, 3)}
ROW_SCALES = 1


@pytest.fixture(scope="module")
def asm(tmp_path_factory):
    return _assembly("fp8_mm_e4m3_e4m3.hip", tmp_path_factory)


def _kernels(asm, tile="", scales=r"\d"):
    return re.findall(rf"^(_Z\w*gdn_fp8_matmul_kernel\w*Fp8TileI{tile}\w*?ELi0ELi0ELi{scales}ELb[01]E\w+):", asm, re.M)


def test_no_tile_spills(asm):
    names = _kernels(asm)
    assert len(names) == 4 * (12 + 7), names  # layouts of b's scales x tiles of bf16 and of fp32 results
    for name in names:
        assert not any("scratch_" in ln for ln in _function(asm, name)), name


@pytest.mark.parametrize("tile", PHASED)
def test_phased_tiles_keep_their_counted_waits(asm, tile):
    cw, tw, wmt, wnt, ns = PHASED[tile]
    m0, x0 = wmt // 2, (wnt + 1) // 2
    groups = [2 * tw * x0, 2 * cw * m0, 2 * cw * (wmt - m0), 2 * tw * (wnt - x0)]  # X0, W0, W1, X1: 8-row copies, split over 8 waves
    n = [g // 8 + g % 8 // 4 for g in groups]
    n[0] += 2  # the scales of both operands
    every = sum(n)
    names = _kernels(asm, "".join(f"Li{v}E" for v in (cw, tw, wmt, wnt, ns)), ROW_SCALES)
    assert len(names) == 1, names
    events = _events(_function(asm, names[0]))

    def found(want):
        return any(events[i:i + len(want)] == want for i in range(len(events)))

    # a stage of the loop, from any of its phases on
    stage = (["c"] * n[3] + [n[3] + (ns - 1) * every, "b", "b"] + ["c"] * n[0] + [n[0] + (ns - 1) * every, "b", "b"]
             + ["c"] * n[1] + ["b", "b"] + ["c"] * n[2] + [n[2] + (ns - 1) * every, "b", "b"])
    assert any(found(stage[i:] + stage[:i]) for i in range(len(stage)))
    # the stages after the last issued one, t of them left
    for t in range(ns):
        tail = [n[3] + t * every, "b", "b", t * every, "b", "b", "b", "b"]
        tail += [n[2] + n[3] + (t - 1) * every, "b"] if t else []
        assert found((["c"] * n[3] if t == ns - 1 else []) + tail), t
    # the ring is filled (all but X1 of its last stage) before a tile's first stage waits for X0, the scales and W0
    assert n[2] + (ns - 1) * every in events[events.index("c"):]
