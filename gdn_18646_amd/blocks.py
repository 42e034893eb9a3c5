"""What stands between and beside layers: differentiable block norms and 8-bit
linear layers on the kernels ``rmsnorm.block_norm`` and ``proj.fp8_quantize`` /
``proj.fp8_matmul``.

* ``block_norm``: the norms before and after a block fused with its gate and
  residual scale,

      u = RMSNorm(y) post_gamma;  h = residual + residual_scale scale act(gate) u;
      n = RMSNorm(h) gamma

  with gradients of every operand (one kernel and a sum over rows);
* ``fp8_linear``: ``x W^T`` on 8-bit codes with a power-of-two scale for each
  block of 128 (1 x 128 of activations and gradients, 128 x 128 of weights),
  forward in e4m3, gradients in e5m2;
* ``Fp8Weight``: a weight quantised once, for serving.

The kernels' own entry points (``compile_kernels()['rmsnorm'].block_norm`` and so
on) take the same operands without recording gradients.
"""

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import compile_kernels, native_extension

__all__ = ["block_norm", "fp8_linear", "Fp8Weight"]

BLOCK = 128


def _check_capture():
    """Refuses a backward pass that is being captured into a graph and has yet to
    reach nodes of eager work, such as the gradient accumulators of leaves that an
    eager graph keeps alive: they belong to the eager work's stream, which autograd
    would draw into the capture, and that ends the process."""
    if not torch.cuda.is_current_stream_capturing():
        return
    outside = sorted({name for name, out in native_extension()._backward_nodes() if out})
    if outside:
        raise RuntimeError("a backward pass is captured while an eager autograd graph of the same leaves is alive: "
                           f"drop (or detach) the eager results before the capture ({', '.join(outside)})")


class _BlockNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, residual, gate, post_gamma, gamma, scale, residual_scale, act, eps):
        h, n, _, _, rstd_y, rstd_h = compile_kernels()["rmsnorm"].block_norm(
            y, residual=residual, gate=gate, post_gamma=post_gamma, gamma=gamma, scale=scale,
            residual_scale=residual_scale, act=act, eps=eps, stats=True)
        ctx.save_for_backward(y, residual, gate, post_gamma, gamma, scale, rstd_y, rstd_h)
        ctx.residual_scale, ctx.act = residual_scale, act
        ctx.set_materialize_grads(False)
        return h, n

    @staticmethod
    @once_differentiable
    def backward(ctx, dh, dn):
        _check_capture()
        y, residual, gate, post_gamma, gamma, scale, rstd_y, rstd_h = ctx.saved_tensors
        if dh is None and dn is None:
            return (None,) * 9
        dh, dn = (None if t is None else t.contiguous() for t in (dh, dn))
        dresidual, dy, dgate, dpost, dgamma, dscale = compile_kernels()["rmsnorm"].block_norm_backward(
            dh, dn, y, residual=residual, gate=gate, post_gamma=post_gamma, gamma=gamma, scale=scale,
            residual_scale=ctx.residual_scale, act=ctx.act, rstd_y=rstd_y, rstd_h=rstd_h)
        grads = (dy, dresidual, dgate, dpost, dgamma, dscale)
        return tuple(g if need else None for g, need in zip(grads, ctx.needs_input_grad)) + (None, None, None)


def block_norm(y, residual=None, gate=None, post_gamma=None, gamma=None, scale=None, residual_scale=1.0, act="none",
               eps=1e-6):
    """(h, n) of a block's output y [..., D]; n is None without ``gamma``.

    residual: y's shape.  gate: y's shape, [B, D] (a gate a sequence of
    y [B, ..., D]; the backward pass takes at most 65535 of them) or [D]; act: none,
    sigmoid, silu or tanh.  post_gamma, gamma,
    scale: [D].  What is None is left out.  Differentiable in every tensor, in
    reverse mode; an operand with a forward-mode tangent raises.
    """
    tensors = (y, residual, gate, post_gamma, gamma, scale)
    there = [t for t in tensors if t is not None]
    recorded = torch.is_grad_enabled() and any(t.requires_grad for t in there)
    if not recorded and all(forward_ad.unpack_dual(t).tangent is None for t in there):
        h, n, _, _ = compile_kernels()["rmsnorm"].block_norm(
            y, residual=residual, gate=gate, post_gamma=post_gamma, gamma=gamma, scale=scale,
            residual_scale=residual_scale, act=act, eps=eps)
        return h, n
    return _BlockNorm.apply(*tensors, float(residual_scale), act, float(eps))


def _adjacent(x):
    """x [M, K] with a row's elements adjacent, as the quantisation reads them;
    expanded and transposed ones are copied."""
    return x if x.stride(1) == 1 and x.stride(0) >= x.shape[1] else x.contiguous()


class Fp8Weight:
    """A weight [N, K] (bf16 or fp32) as e4m3 codes with a scale for each 128 x 128
    block: ``codes`` / ``scales`` for x W^T and, with ``transposed``, ``codes_t`` /
    ``scales_t`` for the gradient of x."""

    def __init__(self, weight, transposed=False):
        if weight.dim() != 2:
            raise ValueError(f"weight must be [N, K], got {tuple(weight.shape)}")
        self.shape = tuple(weight.shape)
        out = compile_kernels()["proj"].fp8_quantize(_adjacent(weight.detach()), block_rows=BLOCK, rows=True, columns=transposed)
        self.codes, self.scales = out[:2]
        self.codes_t, self.scales_t = out[2:] if transposed else (None, None)


class _Fp8Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, record):
        proj = compile_kernels()["proj"]
        need_x, need_w = (record and need for need in ctx.needs_input_grad[:2])
        x2 = _adjacent(x.reshape(-1, x.shape[-1]))
        q = proj.fp8_quantize(x2, rows=True, columns=need_w)
        w = weight if isinstance(weight, Fp8Weight) else Fp8Weight(weight, transposed=need_x)
        if need_x and w.codes_t is None:
            raise ValueError("fp8_linear: the gradient of x needs an Fp8Weight with transposed=True")
        ctx.save_for_backward(*(q[2:] if need_w else (None, None)), *((w.codes_t, w.scales_t) if need_x else (None, None)))
        ctx.shape, ctx.dtypes = x.shape, (x.dtype, getattr(weight, "dtype", None))
        ctx.sizes = w.shape
        return proj.fp8_matmul(q[0], q[1], w.codes, w.scales, out_dtype=x.dtype).reshape(*x.shape[:-1], w.shape[0])

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        _check_capture()
        proj = compile_kernels()["proj"]
        xt, xts, wt, wts = ctx.saved_tensors
        N, K = ctx.sizes
        need_x, need_w = ctx.needs_input_grad[:2]
        if dy.numel() == 0:  # no tokens, or no columns
            return (torch.zeros(ctx.shape, dtype=ctx.dtypes[0], device=dy.device) if need_x else None,
                    torch.zeros(N, K, dtype=ctx.dtypes[1], device=dy.device) if need_w else None, None)
        d = proj.fp8_quantize(_adjacent(dy.reshape(-1, N)), dtype=torch.float8_e5m2, rows=need_x, columns=need_w)
        dx = dw = None
        if need_x:
            dx = proj.fp8_matmul(d[0], d[1], wt, wts, out_dtype=ctx.dtypes[0]).reshape(ctx.shape)
        if need_w:
            dt, dts = d[-2:]
            dw = proj.fp8_matmul(dt, dts, xt, xts, out_dtype=ctx.dtypes[1])
        return dx, dw, None


def fp8_linear(x, weight):
    """x [..., K] times weight^T on 8-bit codes: [..., N] of x's type.

    weight: a tensor [N, K], quantised in the call and differentiable, or an
    ``Fp8Weight``.  x and a weight tensor are bf16 or fp32; fp32 ones get fp32
    results.  In the backward pass the incoming gradient is quantised to e5m2 in
    blocks of 1 x 128 along each product's own sum, x along its tokens.
    """
    if len(weight.shape) != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"fp8_linear: x [..., {x.shape[-1]}] and weight {tuple(weight.shape)}")
    return _Fp8Linear.apply(x, weight, torch.is_grad_enabled())
