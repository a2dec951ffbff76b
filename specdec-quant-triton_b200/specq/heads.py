"""Query and key heads before the cache: their norm and rotary turn in one pass, with the gradients.

    qk_norm_rope(q, k, q_weight, k_weight, pos, table, eps=1e-6, layout="half")  -> (q', k')

For models that normalise every query and key head by its own root mean square before the rotation.  The
append of the block-scaled cache then takes k' without a table (it is turned already), attention q'.  There is
no reference counterpart.
"""
from __future__ import annotations

from . import _lib

# The argument checks, the calls and the gradient's record are in csrc/py_blocks.cpp, in the order of this signature.
_native = _lib.native()


def qk_norm_rope(q, k, q_weight, k_weight, pos, table, eps=1e-6, layout="half", q_out=None, k_out=None, plan=None):
    """Every head x of q [T, H, D] and k [T, H_KV, D] becomes turn(x / sqrt(mean(x^2) + eps) * weight), its
    first rot = table.shape[1] elements turned to positions pos [T] int32 as `rope` turns them.

    q and k: float16, bfloat16 or float32, any row and head strides (views of a projection's rows), D up to
    2048.  q_weight, k_weight: [D] of the same type, or both float32; None: ones.  fp32 inside, rounded once.
    `q_out` may be q, `k_out` k; else they share no memory with q and k.  Where q, k or a weight requires grad the
    outputs record it (without q_out and k_out; once differentiable; the table has none; no forward mode): the
    weights' gradients are sums over all tokens and heads in a fixed order.
    With `plan`, only rows < plan[0]: the others of new outputs and gradients are 0, those of q_out and k_out keep
    what they hold."""
    return _native.qk_norm_rope(q, k, q_weight, k_weight, pos, table, eps, layout, q_out, k_out, plan)
