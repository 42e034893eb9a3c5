"""What gdn_18646_amd.blocks does around the kernels, on the CPU with stand-ins for
them."""

import pytest
import torch
from torch.autograd import forward_ad

from gdn_18646_amd import blocks, native_extension


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


class _Look(torch.autograd.Function):
    """Notes what the native extension says of the backward pass that it is in."""

    @staticmethod
    def forward(ctx, x, w, seen):
        ctx.seen = seen
        return x * 1.0, w * 1.0

    @staticmethod
    def backward(ctx, dx, dw):
        ctx.seen.append(sorted(name.split("::")[-1] for name, _ in native_extension()._backward_nodes()))
        assert not any(out for _, out in native_extension()._backward_nodes())  # no streams here
        return dx, dw, None


def test_a_backward_pass_names_the_nodes_that_it_reaches():
    """The check of a captured backward pass sees leaves behind views and casts,
    and no nodes that the pass does not run (its root has run)."""
    x, w = torch.randn(4, 8, requires_grad=True), torch.randn(8, dtype=torch.float64, requires_grad=True)
    for asked, nodes in ((None, ["AccumulateGrad"] * 2 + ["SumBackward0", "SumBackward0", "ToCopyBackward0", "ViewBackward0", "_LookBackward"]),
                         ((x,), ["AccumulateGrad", "SumBackward0", "SumBackward0", "ViewBackward0", "_LookBackward"])):
        seen = []
        a, b = _Look.apply(x.view(8, 4), w.float(), seen)
        loss = a.sum() + b.sum()
        loss.backward() if asked is None else torch.autograd.grad(loss, asked)
        assert seen == [nodes]
    assert native_extension()._backward_nodes() == []
