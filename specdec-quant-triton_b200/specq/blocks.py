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

import ctypes as C
import math

import torch

from . import _lib
from .ops import _plan_ptr, _ptr, _require_cuda, _stream

_ROW_DTYPES = {torch.float16: _lib.SPECQ_DTYPE_F16, torch.float32: _lib.SPECQ_DTYPE_F32,
               torch.bfloat16: _lib.SPECQ_DTYPE_BF16}
_CACHE_DTYPES = {torch.int8: _lib.SPECQ_CACHE_INT8, torch.float8_e4m3fn: _lib.SPECQ_CACHE_E4M3}
_LAYOUTS = {"half": _lib.SPECQ_ROPE_HALF, "interleaved": _lib.SPECQ_ROPE_INTERLEAVED}


# ----------------------------------------------------------------------------------------------
# checks
# ----------------------------------------------------------------------------------------------
def _layout(name, layout):
    if layout not in _LAYOUTS:
        raise ValueError(f"{name}: layout must be 'half' or 'interleaved', got {layout!r}")
    return _LAYOUTS[layout]


def _rows3(name, what, t, dtypes=_ROW_DTYPES):
    if t.dtype not in dtypes:
        raise TypeError(f"{name}: {what} must be one of {[str(d) for d in dtypes]}, got {t.dtype}")
    if t.dim() != 3 or (t.stride(2) != 1 and t.shape[2] > 1):
        raise ValueError(f"{name}: {what} must be [rows, heads, dim] with unit inner stride, got {tuple(t.shape)} "
                         f"strides {t.stride()}")


def _int32(name, what, t, *shape):
    """int32, and at least `shape` long in each dimension (None: any), unit inner stride."""
    if t.dtype != torch.int32:
        raise TypeError(f"{name}: {what} must be int32, got {t.dtype}")
    if t.dim() != len(shape) or any(n is not None and d < n for d, n in zip(t.shape, shape)):
        raise ValueError(f"{name}: {what} must be at least {shape}, got {tuple(t.shape)}")
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name}: {what} needs unit inner stride")


def _cache(name, kc, vc, ks, vs, dims):
    """Checks a cache of `dims` dimensions (4, or 5 with layers)."""
    if kc.dtype not in _CACHE_DTYPES or vc.dtype != kc.dtype:
        raise TypeError(f"{name}: kc and vc must both be int8 or both float8_e4m3fn")
    if ks.dtype != torch.float32 or vs.dtype != torch.float32:
        raise TypeError(f"{name}: ks and vs must be float32")
    if kc.dim() != dims or vc.shape != kc.shape or vc.stride() != kc.stride():
        raise ValueError(f"{name}: kc and vc must be alike with {dims} dimensions, got {tuple(kc.shape)} and "
                         f"{tuple(vc.shape)}")
    if kc.stride(-1) != 1:
        raise ValueError(f"{name}: the cache needs unit stride along D")
    want = tuple(kc.shape[: dims - 3]) + (kc.shape[-2],)
    if tuple(ks.shape) != want or vs.shape != ks.shape or vs.stride() != ks.stride():
        raise ValueError(f"{name}: ks and vs must be alike, {want}, got {tuple(ks.shape)} and {tuple(vs.shape)}")


def _same_device(name, first, *ts):
    _require_cuda(first, *ts)
    for t in ts:
        if t is not None and t.device != first.device:
            raise ValueError(f"{name}: tensors on {first.device} and {t.device}")


def _table(name, table, dim):
    if table.dtype != torch.float32 or table.dim() != 2 or not table.is_contiguous():
        raise TypeError(f"{name}: table must be a contiguous float32 [n_pos, rot]")
    if table.shape[0] < 1 or table.shape[1] < 2 or table.shape[1] % 2 or table.shape[1] > dim:
        raise ValueError(f"{name}: table {tuple(table.shape)} needs positions and an even rot <= {dim}")


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
          the same with a ramp over the pair index, and cosines and sines times `attention`
          (default 0.1 ln f + 1)"""
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
        lo, hi = max(math.floor(pair_of(fast)), 0), min(math.ceil(pair_of(slow)), rot // 2 - 1)
        ramp = ((torch.arange(rot // 2, dtype=torch.float64) - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        inv = inv * (1 - ramp) + inv / f * ramp
        gain = scaling.get("attention")
        gain = 0.1 * math.log(f) + 1.0 if gain is None else float(gain)
    elif kind not in (None, "ntk"):
        raise ValueError(f"rope_table: scaling type {kind!r}")
    ang = torch.arange(n_pos, dtype=torch.float64, device=device)[:, None] * inv.to(device)
    return torch.cat([ang.cos() * gain, ang.sin() * gain], 1).float()


def rope(x, pos, table, layout="half", inverse=False, out=None, plan=None):
    """Turn the first rot = table.shape[1] elements of every head of x [T, H, D] (float16, bfloat16 or
    float32; any row and head strides) to positions pos [T] int32; `out` may be x.  inverse=True
    turns back, which is the gradient of the rotation.  With `plan`, only rows < plan[0]."""
    lay = _layout("rope", layout)
    _rows3("rope", "x", x)
    _table("rope", table, x.shape[2])
    _int32("rope", "pos", pos, x.shape[0])
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    else:
        _rows3("rope", "out", out)
        if out.dtype != x.dtype or out.shape != x.shape:
            raise ValueError(f"rope: out must be {x.dtype} {tuple(x.shape)}, got {out.dtype} {tuple(out.shape)}")
    _same_device("rope", x, pos, table, out)
    T, H, D = x.shape
    _lib.check(_lib.load().specq_rope(
        x.data_ptr(), x.stride(0), x.stride(1), out.data_ptr(), out.stride(0), out.stride(1), _ROW_DTYPES[x.dtype],
        pos.data_ptr(), table.data_ptr(), table.shape[0], T, H, D, table.shape[1], lay, 1 if inverse else 0,
        _plan_ptr(plan), _stream()))
    return out


# ----------------------------------------------------------------------------------------------
# append, attention, compaction
# ----------------------------------------------------------------------------------------------
def kv_append_blocks(k, v, kc, vc, ks, vs, block_tbl, ctx_len, q_len, q=None, q_out=None, table=None, pos=None,
                     layout="half", plan=None, n_seqs=None, ql_max=None):
    """Write the K and V [T, H_KV, D] of the q_len newest tokens of each sequence (row b * q_len + t,
    position ctx_len[b] - q_len + t) into the cache, K turned by `table` when one is given, and return
    the same tokens' queries q [T, H, D] turned (q_out, which may be q; a new tensor by default).

    A page's scale grows when a new token needs it, and the page's older tokens are requantised.
    `pos` [T] int32: rotary positions other than the tokens' places (a draft tree's depths).  With
    `plan`, plan[0] sequences of plan[1] tokens are active and q_len is ignored for ql_max."""
    name = "kv_append_blocks"
    lay = _layout(name, layout)
    _cache(name, kc, vc, ks, vs, 4)
    rows = (torch.float16, torch.bfloat16)
    _rows3(name, "k", k, rows)
    _rows3(name, "v", v, rows)
    P, page, H_KV, D = kc.shape
    B = block_tbl.shape[0] if block_tbl.dim() == 2 else -1
    _int32(name, "block_tbl", block_tbl, None, None)
    _int32(name, "ctx_len", ctx_len, B)
    n_seqs = B if n_seqs is None else n_seqs
    ql_max = q_len if ql_max is None else ql_max
    if not 0 <= n_seqs <= B or not 0 <= q_len <= ql_max:
        raise ValueError(f"{name}: n_seqs={n_seqs} of {B}, q_len={q_len} of {ql_max}")
    need = B * ql_max if plan is not None else n_seqs * q_len
    for t, what in ((k, "k"), (v, "v")):
        if t.dtype != k.dtype or tuple(t.shape[1:]) != (H_KV, D) or t.shape[0] < need:
            raise ValueError(f"{name}: {what} must be {k.dtype} [>= {need}, {H_KV}, {D}], got {t.dtype} {tuple(t.shape)}")
    H = 0
    if table is not None:
        _table(name, table, D)
    elif q is not None or pos is not None:
        raise ValueError(f"{name}: q and pos need a rotary table")
    if pos is not None:
        _int32(name, "pos", pos, need)
    if q is not None:
        _rows3(name, "q", q, rows)
        if q.dtype != k.dtype or q.shape[2] != D or q.shape[0] < need:
            raise ValueError(f"{name}: q must be {k.dtype} [>= {need}, H, {D}], got {q.dtype} {tuple(q.shape)}")
        H = q.shape[1]
        if q_out is None:
            q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        else:
            _rows3(name, "q_out", q_out, rows)
            if q_out.dtype != q.dtype or q_out.shape != q.shape:
                raise ValueError(f"{name}: q_out must be {q.dtype} {tuple(q.shape)}")
    elif q_out is not None:
        raise ValueError(f"{name}: q_out without q")
    _same_device(name, kc, vc, ks, vs, k, v, q, q_out, table, pos, block_tbl, ctx_len, plan)
    _lib.check(_lib.load().specq_block_append(
        k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), _ptr(q),
        q.stride(0) if H else 0, q.stride(1) if H else 0, _ptr(q_out), q_out.stride(0) if H else 0,
        q_out.stride(1) if H else 0, _ROW_DTYPES[k.dtype], _ptr(table), table.shape[0] if table is not None else 0,
        table.shape[1] if table is not None else 0, lay, _ptr(pos), kc.data_ptr(), vc.data_ptr(), kc.stride(0),
        kc.stride(1), kc.stride(2), _CACHE_DTYPES[kc.dtype], P, ks.data_ptr(), vs.data_ptr(), ks.stride(0),
        ks.stride(1), block_tbl.data_ptr(), block_tbl.stride(0), block_tbl.shape[1], ctx_len.data_ptr(),
        _plan_ptr(plan), B, n_seqs, q_len, ql_max, H, H_KV, D, page, _stream()))
    return q_out


def paged_attention_blocks(q, kc, vc, ks, vs, block_tbl, ctx_len, q_len=None, tree=None, sm_scale=None, out=None,
                           plan=None, n_seqs=None, ql_max=None):
    """Attention of the q_len newest tokens of each sequence over the block-scaled cache -> out like q.

    q: [B, q_len, H, D], or packed rows [T, H, D] (sequence b's token t at row b * q_len + t; give
    q_len), float16 or bfloat16.  Row qi sees tokens t <= ctx_len[b] - q_len + qi, or, with `tree`
    (int64 [B, q_len] bit sets, q_len <= 64), every token before the drafts and draft j where bit j of
    tree[b, qi] is set.  A row that sees nothing is 0.  With `plan`, plan[0] sequences of plan[1]
    tokens are active, ql_max is the most tokens and packed rows follow the active q_len."""
    name = "paged_attention_blocks"
    _cache(name, kc, vc, ks, vs, 4)
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"{name}: q must be float16 or bfloat16, got {q.dtype}")
    P, page, H_KV, D = kc.shape
    _int32(name, "block_tbl", block_tbl, None, None)
    B = block_tbl.shape[0]
    _int32(name, "ctx_len", ctx_len, B)
    packed = q.dim() == 3
    if packed:
        if q_len is None:
            raise ValueError(f"{name}: packed queries need q_len")
    elif q.dim() == 4:
        q_len = q.shape[1] if q_len is None else q_len
        if q.shape[0] < B or q.shape[1] < q_len:
            raise ValueError(f"{name}: q is {tuple(q.shape)} for {B} sequences of {q_len} tokens")
    else:
        raise ValueError(f"{name}: q must have 3 or 4 dimensions, got {tuple(q.shape)}")
    n_seqs = B if n_seqs is None else n_seqs
    ql_max = (q_len if packed else max(q_len, q.shape[1] if plan is not None else 0)) if ql_max is None else ql_max
    if not 0 <= n_seqs <= B or not 0 <= q_len <= ql_max or (not packed and plan is not None and q.shape[1] < ql_max):
        raise ValueError(f"{name}: n_seqs={n_seqs} of {B}, q_len={q_len} of {ql_max}, q {tuple(q.shape)}")
    if packed and q.shape[0] < (B * ql_max if plan is not None else n_seqs * q_len):
        raise ValueError(f"{name}: {q.shape[0]} packed rows for {B} sequences of {ql_max} tokens")
    H = q.shape[-2]
    if q.shape[-1] != D or H % H_KV:
        raise ValueError(f"{name}: q heads {tuple(q.shape[-2:])} do not fit the cache's {(H_KV, D)}")
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device) if plan is None and n_seqs == B else torch.zeros_like(
            q, memory_format=torch.contiguous_format)
    elif out.dtype != q.dtype or out.shape != q.shape:
        raise ValueError(f"{name}: out must be {q.dtype} {tuple(q.shape)}, got {out.dtype} {tuple(out.shape)}")
    if q.stride(-1) != 1 or out.stride(-1) != 1:
        raise ValueError(f"{name}: q and out need unit stride along D")
    if sm_scale is not None and not sm_scale > 0:
        raise ValueError(f"{name}: sm_scale={sm_scale} must be positive")
    if tree is not None:
        if tree.dtype != torch.int64 or tree.dim() != 2 or tree.shape[0] < B or tree.shape[1] < ql_max:
            raise ValueError(f"{name}: tree must be int64 [>= {B}, >= {ql_max}], got {tree.dtype} {tuple(tree.shape)}")
    _same_device(name, kc, vc, ks, vs, q, out, block_tbl, ctx_len, tree, plan)
    lib = _lib.load()
    cols = block_tbl.shape[1]
    size = C.c_int64(0)
    _lib.check(lib.specq_block_attention_workspace(B, n_seqs, q_len, ql_max, H, H_KV, D, page, cols,
                                                   0 if plan is None else 1, C.byref(size)))
    # from torch's allocator on the current stream: nothing outlives the call but what its launches need
    ws = torch.empty(size.value, dtype=torch.uint8, device=q.device) if size.value else None
    qs, os_ = ((0,) + q.stride() if packed else q.stride()), ((0,) + out.stride() if packed else out.stride())
    _lib.check(lib.specq_block_attention(
        q.data_ptr(), qs[0], qs[1], qs[2], _ROW_DTYPES[q.dtype], kc.data_ptr(), vc.data_ptr(), kc.stride(0), kc.stride(1),
        kc.stride(2), _CACHE_DTYPES[kc.dtype], P, ks.data_ptr(), vs.data_ptr(), ks.stride(0), ks.stride(1),
        block_tbl.data_ptr(), block_tbl.stride(0), cols, ctx_len.data_ptr(), _ptr(tree),
        tree.stride(0) if tree is not None else 0, tree.stride(1) if tree is not None else 0,
        D ** -0.5 if sm_scale is None else float(sm_scale), out.data_ptr(), os_[0], os_[1], os_[2], _plan_ptr(plan), B,
        n_seqs, q_len, ql_max, H, H_KV, D, page, _ptr(ws), size.value, _stream()))
    return out


def _layered(t, dims):
    return t if t.dim() == dims else t.unsqueeze(0)


def kv_compact_blocks(kc, vc, ks, vs, block_tbl, ctx_len, q_len, accept, n_accept, ctx_out=None):
    """Move the accepted drafts of each sequence together and return the new context lengths.

    accept [B, A] int32: for each sequence the accepted drafts' indices among its q_len newest tokens,
    strictly growing; n_accept [B] int32: how many count.  kc, vc, ks, vs: one layer, or all layers of
    a cache [L, P, page, H_KV, D] / [L, P, H_KV].  ctx_out (not ctx_len itself): int32 [B]."""
    name = "kv_compact_blocks"
    dims = 5 if kc.dim() == 5 else 4
    _cache(name, kc, vc, ks, vs, dims)
    _int32(name, "block_tbl", block_tbl, None, None)
    B = block_tbl.shape[0]
    _int32(name, "ctx_len", ctx_len, B)
    _int32(name, "accept", accept, B, None)
    _int32(name, "n_accept", n_accept, B)
    if q_len < 0:
        raise ValueError(f"{name}: q_len={q_len}")
    if ctx_out is None:
        ctx_out = torch.empty((B,), dtype=torch.int32, device=ctx_len.device)
    _int32(name, "ctx_out", ctx_out, B)
    _same_device(name, kc, vc, ks, vs, block_tbl, ctx_len, accept, n_accept, ctx_out)
    kc, vc, ks, vs = _layered(kc, 5), _layered(vc, 5), _layered(ks, 3), _layered(vs, 3)
    L, P, page, H_KV, D = kc.shape
    if L == 0:
        raise ValueError(f"{name}: a cache without layers")
    _lib.check(_lib.load().specq_block_compact(
        kc.data_ptr(), vc.data_ptr(), kc.stride(0), kc.stride(1), kc.stride(2), kc.stride(3), _CACHE_DTYPES[kc.dtype], L,
        P, ks.data_ptr(), vs.data_ptr(), ks.stride(0), ks.stride(1), ks.stride(2), block_tbl.data_ptr(),
        block_tbl.stride(0), block_tbl.shape[1], ctx_len.data_ptr(), accept.data_ptr(), accept.stride(0),
        accept.shape[1], n_accept.data_ptr(), ctx_out.data_ptr(), B, q_len, H_KV, D, page, _stream()))
    return ctx_out


# ----------------------------------------------------------------------------------------------
# the page pool
# ----------------------------------------------------------------------------------------------
def _pool(name, ref, tbl, held):
    _int32(name, "ref", ref, None)
    _int32(name, "tbl", tbl, None, None)
    _int32(name, "held", held, tbl.shape[0])
    if ref.shape[0] > 1 and ref.stride(0) != 1:
        raise ValueError(f"{name}: ref must be contiguous")
    return (ref.data_ptr(), ref.shape[0], tbl.data_ptr(), tbl.stride(0) if tbl.shape[0] > 1 else max(tbl.shape[1], 1),
            held.data_ptr(), tbl.shape[0], tbl.shape[1])


def pages_release(ref, tbl, held, drop):
    """Rows r with drop[r] (bool [S]) give up their pages: ref int32 [P] counts the rows that hold a page,
    tbl int32 [S, C] has the rows' pages (-1: none), held int32 [S] their number."""
    pool = _pool("pages_release", ref, tbl, held)
    if drop.dtype not in (torch.bool, torch.uint8) or drop.dim() != 1 or drop.shape[0] < tbl.shape[0] or (
            drop.shape[0] > 1 and drop.stride(0) != 1):
        raise ValueError(f"pages_release: drop must be a contiguous bool [{tbl.shape[0]}], got {drop.dtype} {tuple(drop.shape)}")
    _same_device("pages_release", ref, tbl, held, drop)
    _lib.check(_lib.load().specq_pages_release(*pool, drop.data_ptr(), _stream()))


def pages_reserve(ref, tbl, held, want_len, page, short=None):
    """Extend row r to the pages of want_len[r] tokens, lowest free pages first, every row or none.
    Returns `short`, int32 [1]: the pages that were missing (0: done)."""
    pool = _pool("pages_reserve", ref, tbl, held)
    _int32("pages_reserve", "want_len", want_len, tbl.shape[0])
    if page < 1:
        raise ValueError(f"pages_reserve: page={page}")
    if short is None:
        short = torch.empty((1,), dtype=torch.int32, device=ref.device)
    _int32("pages_reserve", "short", short, 1)
    _same_device("pages_reserve", ref, tbl, held, want_len, short)
    _lib.check(_lib.load().specq_pages_reserve(*pool, want_len.data_ptr(), page, short.data_ptr(), _stream()))
    return short


def pages_fork(kc, vc, ks, vs, ref, tbl, held, parent, length, short=None):
    """Row r with parent[r] = p (0 <= p != r; any other value keeps the row) becomes a copy of row p's first
    length[p] tokens: full pages are shared, a part-filled last page is copied in every layer to the
    lowest free page, and what r held is released; every row or none, all at once.  kc, vc, ks, vs: one
    layer or all layers.  Returns `short` as pages_reserve does."""
    name = "pages_fork"
    _cache(name, kc, vc, ks, vs, 5 if kc.dim() == 5 else 4)
    pool = _pool(name, ref, tbl, held)
    S, cols = tbl.shape
    _int32(name, "parent", parent, S)
    _int32(name, "length", length, S)
    kc, vc, ks, vs = _layered(kc, 5), _layered(vc, 5), _layered(ks, 3), _layered(vs, 3)
    L, P, page, H_KV, D = kc.shape
    if P < ref.shape[0]:
        raise ValueError(f"{name}: a pool of {ref.shape[0]} pages over a cache of {P}")
    if short is None:
        short = torch.empty((1,), dtype=torch.int32, device=ref.device)
    _int32(name, "short", short, 1)
    _same_device(name, ref, kc, vc, ks, vs, tbl, held, parent, length, short)
    scratch = torch.empty((S * (cols + 1),), dtype=torch.int32, device=ref.device)
    _lib.check(_lib.load().specq_pages_fork(
        kc.data_ptr(), vc.data_ptr(), kc.stride(0), kc.stride(1), kc.stride(2), kc.stride(3), L, ks.data_ptr(),
        vs.data_ptr(), ks.stride(0), ks.stride(1), ks.stride(2), *pool, parent.data_ptr(), length.data_ptr(),
        scratch.data_ptr(), short.data_ptr(), H_KV, D, page, _stream()))
    return short
