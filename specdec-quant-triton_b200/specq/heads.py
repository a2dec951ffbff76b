"""Query and key heads before the cache: their norm and rotary turn in one pass, with the gradients.

    qk_norm_rope(q, k, q_weight, k_weight, pos, table, eps=1e-6, layout="half")  -> (q', k')

For models that normalise every query and key head by its own root mean square before the rotation.  The
append of the block-scaled cache then takes k' without a table (it is turned already), attention q'.  There is
no reference counterpart.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib

# The argument checks and the calls are in csrc/py_blocks.cpp, in the order of these signatures.
_native = _lib.native()


def qk_norm_rope(q, k, q_weight, k_weight, pos, table, eps=1e-6, layout="half", q_out=None, k_out=None, plan=None):
    """Every head x of q [T, H, D] and k [T, H_KV, D] becomes turn(x / sqrt(mean(x^2) + eps) * weight), its
    first rot = table.shape[1] elements turned to positions pos [T] int32 as `rope` turns them.

    q and k: float16, bfloat16 or float32, any row and head strides (views of a projection's rows), D up to
    2048.  q_weight, k_weight: [D] of the same type, or both float32; None: ones.  fp32 inside, rounded once.
    `q_out` may be q, `k_out` k.  Where q, k or a weight requires grad the outputs record it (without q_out and k_out; once
    differentiable; the table has none): the weights' gradients are sums over all tokens and heads in a fixed order.
    With `plan`, only rows < plan[0]: the others of new outputs and gradients are 0, those of q_out and k_out keep
    what they hold."""
    y = _native.qk_norm_rope(q, k, q_weight, k_weight, pos, table, eps, layout, q_out, k_out, plan)
    return y if y is not NotImplemented else _QkNormRope.apply(q, k, q_weight, k_weight, pos, table, eps, layout, plan)


class _QkNormRope(torch.autograd.Function):
    """Both outputs with the gradients of q, k and the weights (the binding leaves tensors that require grad to it)."""

    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, pos, table, eps, layout, plan):
        ctx.save_for_backward(q, k, q_weight, k_weight, pos, table, plan)
        ctx.eps, ctx.layout = eps, layout
        return _native.qk_norm_rope(q, k, q_weight, k_weight, pos, table, eps, layout, None, None, plan)

    @staticmethod
    @once_differentiable
    def backward(ctx, gq, gk):
        q, k, q_weight, k_weight, pos, table, plan = ctx.saved_tensors
        gq, gk = (g if g.stride(-1) == 1 else g.contiguous() for g in (gq, gk))
        want = sum(1 << i for i in range(4) if ctx.needs_input_grad[i])
        d = _native.qk_norm_rope_grad(gq, gk, q, k, q_weight, k_weight, pos, table, ctx.eps, ctx.layout, plan, want)
        return *d, None, None, None, None, None
