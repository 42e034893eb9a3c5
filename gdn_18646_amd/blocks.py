"""What stands between and beside layers: differentiable block norms, linear layers
on 8-bit and 4-bit codes and the clipping of gradients, on the kernels
``rmsnorm.block_norm``, ``proj.fp8_quantize`` / ``proj.fp8_matmul``,
``proj.fp4_quantize`` / ``proj.fp4_matmul`` and ``grads``.

* ``block_norm``: the norms before and after a block fused with its gate and
  residual scale,

      u = RMSNorm(y) post_gamma;  h = residual + residual_scale scale act(gate) u;
      n = RMSNorm(h) gamma

  with gradients of every operand (one kernel and a sum over rows);
* ``fp8_linear``: ``x W^T`` on 8-bit codes with a power-of-two scale for each
  block of 128 (1 x 128 of activations and gradients, 128 x 128 of weights),
  forward in e4m3, gradients in e5m2;
* ``fp4_linear``: the same with the weight in 4-bit codes and a scale for each 32
  x 32 of them, activations in 8-bit or 4-bit codes, gradients in e5m2;
* ``Fp8Weight``, ``Fp4Weight``: a weight quantised once, for serving;
* ``grad_norm``, ``clip_grad_norm``: the 2-norm of many gradients together, and
  their clipping to it, in place or into other tensors.

The kernels' own entry points (``compile_kernels()['rmsnorm'].block_norm`` and so
on) take the same operands without recording gradients.
"""

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import compile_kernels, native_extension

__all__ = ["block_norm", "fp8_linear", "Fp8Weight", "fp4_linear", "Fp4Weight", "grad_norm", "clip_grad_norm"]

BLOCK = 128
E2M1X2, E4M3 = torch.float4_e2m1fn_x2, torch.float8_e4m3fn


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


def _plain(weight):
    """weight [N, K] as it is quantised once: without its graph; a forward-mode tangent,
    which the codes do not carry, raises."""
    if weight.dim() != 2:
        raise ValueError(f"weight must be [N, K], got {tuple(weight.shape)}")
    if forward_ad.unpack_dual(weight).tangent is not None:
        raise RuntimeError("a weight that is quantised once has a forward-mode tangent")
    return _adjacent(weight.detach())


class Fp8Weight:
    """A weight [N, K] (bf16 or fp32) as e4m3 codes with a scale for each 128 x 128
    block: ``codes`` / ``scales`` for x W^T and, with ``transposed``, ``codes_t`` /
    ``scales_t`` for the gradient of x."""

    def __init__(self, weight, transposed=False):
        w = _plain(weight)
        self.shape = tuple(weight.shape)
        out = compile_kernels()["proj"].fp8_quantize(w, block_rows=BLOCK, rows=True, columns=transposed)
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


class Fp4Weight:
    """A weight [N, K] (bf16 or fp32) as e2m1 codes with a scale for each block_rows (32
    or 1) x 32 block: ``codes`` / ``scales`` for x W^T and, with ``transposed``,
    ``codes_t`` / ``scales_t`` for the gradient of x.  With block_rows=32 both stand for
    the same weight, as ``fp4_linear`` quantises a tensor; blocks of 1 x 32 are finer,
    along each product's own sum."""

    def __init__(self, weight, transposed=False, block_rows=32):
        w = _plain(weight)
        self.shape = tuple(weight.shape)
        out = compile_kernels()["proj"].fp4_quantize(w, block_rows=block_rows, rows=True, columns=transposed)
        self.codes, self.scales = out[:2]
        self.codes_t, self.scales_t = out[2:] if transposed else (None, None)

    def dequantize(self, dtype=torch.bfloat16):
        """The weight that the codes stand for, [N, K]."""
        return compile_kernels()["proj"].fp4_dequantize(self.codes, self.scales, columns=self.shape[1], dtype=dtype)


def fp4_linear(x, weight, activations=E4M3):
    """x [..., K] times weight^T, the weight in 4-bit codes: [..., N] of x's type.

    weight: a tensor [N, K], quantised in the call in blocks of 32 x 32 and
    differentiable (the quantisation passes gradients through), or an ``Fp4Weight``.
    activations: torch.float8_e4m3fn (blocks of 1 x 128) or torch.float4_e2m1fn_x2
    (blocks of 1 x 32, twice the speed for many tokens).  x and a weight tensor are bf16
    or fp32; fp32 ones get fp32 results.  In the backward pass the incoming gradient is
    quantised to e5m2 in blocks of 1 x 128 along each product's own sum, and multiplied
    with the 4-bit weight for the gradient of x and with x in e4m3 along its tokens for
    the weight's.  bf16 results of 8-bit codes (dx is always one of those) leave out what
    lies below 2^-17 of the largest of 128 products, a bf16 result's own rounding being
    2^-8; fp32 ones have all of it.  4-bit weights halve what is read of them, which sets
    the time of a few tokens by a large one; for many tokens 8-bit activations set the
    speed, and ``fp8_linear`` takes as long.
    """
    if len(weight.shape) != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"fp4_linear: x [..., {x.shape[-1] if x.dim() else ''}] and weight {tuple(weight.shape)}")
    if activations not in (E4M3, E2M1X2):
        raise ValueError(f"fp4_linear: activations in torch.float8_e4m3fn or torch.float4_e2m1fn_x2, got {activations}")
    f, fp4 = compile_kernels()["proj"].fp4_linear, activations == E2M1X2
    if not isinstance(weight, Fp4Weight):
        return f(x, weight, None, None, None, None, weight.shape[0], fp4)
    if weight.codes_t is None and x.requires_grad and torch.is_grad_enabled():
        raise ValueError("fp4_linear: the gradient of x needs an Fp4Weight with transposed=True")
    return f(x, None, weight.codes, weight.scales, weight.codes_t, weight.scales_t, weight.shape[0], fp4)


def grad_norm(grads):
    """The 2-norm of all the gradients' elements together, a float32 tensor of no axes.

    grads: a list of bf16 and fp32 tensors on one GPU, such as ``[p.grad for p in
    parameters if p.grad is not None]``; None among them is left out, and without any
    the norm is 0.  No gradients of the norm are recorded; a forward-mode tangent raises.
    """
    grads = [g for g in grads if g is not None]
    return native_extension().grads.norm(grads) if grads else torch.zeros(())


def clip_grad_norm(grads, max_norm, out=None):
    """Multiplies the gradients by min(1, max_norm / (norm + 1e-6)), where norm is
    ``grad_norm(grads)``, in place or into ``out`` (tensors of the same shapes, bf16 or
    fp32, for an optimiser that keeps its own, one for each of the gradients); returns
    the norm before.  None among the gradients is left out.

    Nothing is read back to the host, so the call can be captured into a graph.  A norm
    that is NaN makes every result NaN; an infinite gradient makes the others 0, or, where
    max_norm is infinite too, NaN.  No gradients are recorded; a forward-mode tangent
    raises.
    """
    if out is not None:
        if len(out) != len(grads):
            raise ValueError(f"clip_grad_norm: {len(grads)} gradients and {len(out)} results")
        out = [o for g, o in zip(grads, out) if g is not None]
    grads = [g for g in grads if g is not None]
    return native_extension().grads.clip(grads, float(max_norm), out) if grads else torch.zeros(())
