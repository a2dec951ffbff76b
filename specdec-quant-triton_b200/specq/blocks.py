"""The block-scaled KV cache: 8 bits a number, one fp32 scale for each page and KV head.

    rope_table(n_pos, rot, base=10000.0, scaling=None)        cosines | sines, fp32 [n_pos, rot]
    rope(x, pos, table, layout="half", inverse=False)         rotary positions of packed rows
    kv_append_blocks(k, v, kc, vc, ks, vs, block_tbl, ctx_len, q_len, q=..., table=...)
    paged_attention_blocks(q, kc, vc, ks, vs, block_tbl, ctx_len, tree=...)
    kv_compact_blocks(kc, vc, ks, vs, block_tbl, ctx_len, q_len, accept, n_accept)
    pages_release / pages_reserve / pages_fork                the pool of pages

kc, vc [P, page, H_KV, D] int8 or float8_e4m3fn, ks, vs float32 [P, H_KV]; value = number *
scale.  Compaction and fork also take a cache of several layers, [L, P, page, H_KV, D] with
scales [L, P, H_KV].  Every function launches on the current stream, synchronises nothing and may
be captured in a CUDA graph; what the device finds wrong in the tensors' contents (a page number
outside the cache, a context past its table) is skipped or clamped and recorded in the status
word that `get_status` reads.  There is no reference counterpart: the reference's cache has a
scale for each token and head (kernels.py:265-286), and no rotary positions, pool or trees.
"""
from __future__ import annotations

import math

import torch

from . import _lib

# The argument checks and the calls are in csrc/py_blocks.cpp, in the order of these signatures.
_native = _lib.native()


# ----------------------------------------------------------------------------------------------
# rotary positions
# ----------------------------------------------------------------------------------------------
def rope_table(n_pos, rot, base=10000.0, scaling=None, device="cuda"):
    """Cosines and sines of positions 0 .. n_pos - 1 for `rot` rotated elements, float32 [n_pos, rot].

    Pair i turns by pos * base^(-2i / rot), computed in 64 bits.  `scaling` (a dict) stretches the
    angles for contexts longer than the model was trained on:
      {"type": "linear", "factor": f}         every angle divided by f
      {"type": "ntk", "factor": f}            base * f^(rot / (rot - 2))
      {"type": "llama3", "factor": f, "original": n, "low": 1.0, "high": 4.0}
          pairs that turn fewer than `low` times in n positions are divided by f, those that turn
          more than `high` times are kept, those between are blended
      {"type": "yarn", "factor": f, "original": n, "slow": 1.0, "fast": 32.0, "attention": None}
          the same with a ramp over the pair index (its ends rounded outwards, the upper one no further
          than rot - 1: past the last pair the ramp is cut short), and cosines and sines times `attention`
          (default 0.1 ln f + 1, and 1 where f <= 1)"""
    if rot < 2 or rot % 2 or n_pos < 1:
        raise ValueError(f"rope_table: n_pos={n_pos} rot={rot} (rot even, both positive)")
    i = torch.arange(0, rot, 2, dtype=torch.float64)
    gain = 1.0
    kind = None if scaling is None else scaling.get("type")
    f = 1.0 if scaling is None else float(scaling["factor"])
    if f <= 0:
        raise ValueError(f"rope_table: factor {f}")
    if kind == "ntk":
        if rot <= 2:
            raise ValueError("rope_table: ntk scaling needs rot > 2")
        base = base * f ** (rot / (rot - 2))
    inv = base ** (-i / rot)
    if kind == "linear":
        inv = inv / f
    elif kind == "llama3":
        n, low, high = float(scaling["original"]), float(scaling.get("low", 1.0)), float(scaling.get("high", 4.0))
        if high <= low:
            raise ValueError("rope_table: llama3 scaling needs high > low")
        turns = n * inv / (2 * math.pi)
        keep = ((turns - low) / (high - low)).clamp(0, 1)
        inv = inv * keep + inv / f * (1 - keep)
    elif kind == "yarn":
        n, slow, fast = float(scaling["original"]), float(scaling.get("slow", 1.0)), float(scaling.get("fast", 32.0))

        def pair_of(turns):   # the pair that turns so many times in n positions
            return rot * math.log(n / (turns * 2 * math.pi)) / (2 * math.log(base))
        lo, hi = max(math.floor(pair_of(fast)), 0), min(math.ceil(pair_of(slow)), rot - 1)
        ramp = ((torch.arange(rot // 2, dtype=torch.float64) - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        inv = inv * (1 - ramp) + inv / f * ramp
        gain = scaling.get("attention")
        gain = 0.1 * math.log(max(f, 1.0)) + 1.0 if gain is None else float(gain)
    elif kind not in (None, "ntk"):
        raise ValueError(f"rope_table: scaling type {kind!r}")
    ang = torch.arange(n_pos, dtype=torch.float64, device=device)[:, None] * inv.to(device)
    return torch.cat([ang.cos() * gain, ang.sin() * gain], 1).float()


def rope(x, pos, table, layout="half", inverse=False, out=None, plan=None):
    """Turn the first rot = table.shape[1] elements of every head of x [T, H, D] (float16, bfloat16 or
    float32; any row and head strides) to positions pos [T] int32; `out` may be x.  inverse=True
    turns back, which is the gradient of the rotation: an x that requires grad gets it (without `out`; the
    table has none).  With `plan`, only rows < plan[0]: the others of a new output are 0, those of `out`
    keep what they hold."""
    y = _native.rope(x, pos, table, layout, inverse, out, plan)
    return y if y is not NotImplemented else _Rope.apply(x, pos, table, layout, inverse, plan)


class _Rope(torch.autograd.Function):
    """The rotation with its gradient, the inverse rotation of the output's (the binding leaves an x that
    requires grad to it)."""

    @staticmethod
    def forward(ctx, x, pos, table, layout, inverse, plan):
        ctx.save_for_backward(pos, table, *(() if plan is None else (plan,)))
        ctx.layout, ctx.inverse = layout, bool(inverse)
        return _native.rope(x, pos, table, layout, inverse, None, plan)

    @staticmethod
    def backward(ctx, g):
        pos, table, *plan = ctx.saved_tensors
        if g.stride(-1) != 1:
            g = g.contiguous()
        return rope(g, pos, table, ctx.layout, not ctx.inverse, plan=plan[0] if plan else None), None, None, None, None, None


# ----------------------------------------------------------------------------------------------
# append, attention, compaction
# ----------------------------------------------------------------------------------------------
def kv_append_blocks(k, v, kc, vc, ks, vs, block_tbl, ctx_len, q_len, q=None, q_out=None, table=None, pos=None,
                     layout="half", plan=None, n_seqs=None, ql_max=None):
    """Write the K and V [T, H_KV, D] of the q_len newest tokens of each sequence (row b * q_len + t,
    position ctx_len[b] - q_len + t) into the cache, K turned by `table` when one is given, and return
    the same tokens' queries q [T, H, D] turned (q_out, which may be q; a new tensor by default, 0 in rows
    that the call does not reach).

    A page's scale grows when a new token needs it, and the page's older tokens are requantised.
    `pos` [T] int32: rotary positions other than the tokens' places (a draft tree's depths).  With
    `plan`, plan[0] sequences of plan[1] tokens are active and q_len is ignored for ql_max."""
    return _native.kv_append_blocks(k, v, kc, vc, ks, vs, block_tbl, ctx_len, q_len, q, q_out, table, pos, layout, plan,
                                    n_seqs, ql_max)


def paged_attention_blocks(q, kc, vc, ks, vs, block_tbl, ctx_len, q_len=None, tree=None, sm_scale=None, out=None,
                           plan=None, n_seqs=None, ql_max=None):
    """Attention of the q_len newest tokens of each sequence over the block-scaled cache -> out like q.

    q: [B, q_len, H, D], or packed rows [T, H, D] (sequence b's token t at row b * q_len + t; give
    q_len), float16 or bfloat16.  Row qi sees tokens t <= ctx_len[b] - q_len + qi, or, with `tree`
    (int64 [B, q_len] bit sets, q_len <= 64), every token before the drafts and draft j where bit j of
    tree[b, qi] is set.  A row that sees nothing is 0, and so is one of a new output that the call does
    not reach.  With `plan`, plan[0] sequences of plan[1] tokens are active, ql_max is the most tokens
    and packed rows follow the active q_len."""
    return _native.paged_attention_blocks(q, kc, vc, ks, vs, block_tbl, ctx_len, q_len, tree, sm_scale, out, plan, n_seqs,
                                          ql_max)


def kv_compact_blocks(kc, vc, ks, vs, block_tbl, ctx_len, q_len, accept, n_accept, ctx_out=None):
    """Move the accepted drafts of each sequence together and return the new context lengths.

    accept [B, A] int32: for each sequence the accepted drafts' indices among its q_len newest tokens,
    strictly growing; n_accept [B] int32: how many count.  kc, vc, ks, vs: one layer, or all layers of
    a cache [L, P, page, H_KV, D] / [L, P, H_KV].  ctx_out (not ctx_len itself): int32 [B]."""
    return _native.kv_compact_blocks(kc, vc, ks, vs, block_tbl, ctx_len, q_len, accept, n_accept, ctx_out)


# ----------------------------------------------------------------------------------------------
# the page pool
# ----------------------------------------------------------------------------------------------
def pages_release(ref, tbl, held, drop):
    """Rows r with drop[r] (bool [S]) give up their pages: ref int32 [P] counts the rows that hold a page,
    tbl int32 [S, C] has the rows' pages (-1: none), held int32 [S] their number."""
    return _native.pages_release(ref, tbl, held, drop)


def pages_reserve(ref, tbl, held, want_len, page, short=None):
    """Extend row r to the pages of want_len[r] tokens, lowest free pages first, every row or none.
    Returns `short`, int32 [1]: the pages that were missing (0: done)."""
    return _native.pages_reserve(ref, tbl, held, want_len, page, short)


def pages_fork(kc, vc, ks, vs, ref, tbl, held, parent, length, short=None):
    """Row r with parent[r] = p (0 <= p != r; any other value keeps the row) becomes a copy of row p's first
    length[p] tokens: full pages are shared, a part-filled last page is copied in every layer to the
    lowest free page, and what r held is released; every row or none, all at once.  kc, vc, ks, vs: one
    layer or all layers.  Returns `short` as pages_reserve does."""
    return _native.pages_fork(kc, vc, ks, vs, ref, tbl, held, parent, length, short)
