"""What gdn_18646_amd.blocks does around the kernels, on the CPU with stand-ins for
them."""

import pytest
import torch
from torch.autograd import forward_ad

from gdn_18646_amd import blocks


class _Norm:
    """A stand-in for the block norm's kernels: n = y gamma, h = y, gradients of ones."""

    def __init__(self):
        self.stats = []

    def block_norm(self, y, residual=None, gamma=None, stats=False, **kw):
        self.stats.append(stats)
        out = [y.detach().clone(), y.detach() * gamma.detach(), None, None]
        return out + [None, torch.ones(y.shape[:-1])] if stats else out


@pytest.fixture
def norm(monkeypatch):
    n = _Norm()
    monkeypatch.setattr(blocks, "compile_kernels", lambda: {"rmsnorm": n})
    return n


def test_forward_mode_tangents_raise(norm):
    """A tangent that the kernel cannot carry is not dropped."""
    y, gm = torch.randn(4, 8), torch.randn(8)
    t = torch.randn(4, 8)
    with forward_ad.dual_level():
        for args in (dict(y=forward_ad.make_dual(y, t), gamma=gm), dict(y=y, gamma=forward_ad.make_dual(gm, t[0])),
                     dict(y=y, residual=forward_ad.make_dual(y, t), gamma=gm)):
            for mode in (torch.enable_grad, torch.no_grad):
                with mode(), pytest.raises((RuntimeError, NotImplementedError), match="jvp|forward"):
                    blocks.block_norm(**args)
        assert forward_ad.unpack_dual(blocks.block_norm(y, gamma=gm)[1]).tangent is None


def test_block_norm_keeps_statistics_for_recorded_calls_alone(norm):
    y, gm = torch.randn(4, 8), torch.randn(8)
    blocks.block_norm(y, gamma=gm)
    blocks.block_norm(y.requires_grad_(), gamma=gm)
    with torch.no_grad():
        blocks.block_norm(y, gamma=gm)
    assert norm.stats == [False, True, False]
