"""Cases of the block-scaled KV-cache operators: what one pass of each reads and returns.

The cache holds K and V in 8 bits (int8 or e4m3) in pages of `page` tokens, with ONE fp32 scale
for each page and KV head (value = stored number * scale).  The operators around it:

  rope     rotary positions of the heads of packed token rows, or their inverse (the gradient)
  append   the K/V of the newest tokens rotated, quantised and written into their pages (a page's
           scale grows when a new token needs it, and what the page held is requantised), and the
           same tokens' queries rotated
  attend   attention over the cache: causal or tree-masked verification of the newest tokens
  pages    one tick of the page pool: rows dropped, pages reserved, rows forked from other rows
  compact  the accepted tokens of a verified draft tree moved together

`own` False: plain torch operations in 32 bits.  `own` True: this package's operators.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
FLOATS = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
CACHES = {"int8": (torch.int8, 127.0), "e4m3": (torch.float8_e4m3fn, 448.0)}
FLOOR = 1e-8          # the least maximum that a scale is made from
H8B, KV8B, D8B = 32, 8, 128   # the head layout of this repository's stack and benchmark


def listed():
    return [
        # one new token of one request: 32 query and 8 key heads of a packed projection row
        dict(name="rope one token", op="rope", rows=1, heads=40, dim=128, rot=128, layout="half", dtype="fp16",
             inverse=False, n_pos=4096, gap=1024),
        # a prompt batch, interleaved pairs over the first half of each head
        dict(name="rope prompt partial", op="rope", rows=8190, heads=40, dim=128, rot=64, layout="interleaved",
             dtype="bf16", inverse=False, n_pos=32768, gap=0),
        # a verification step: 8 sequences, 9 new tokens each, contexts about 4096
        dict(name="append verify", op="append", batch=8, q_len=9, kv=8, group=4, dim=128, page=16, rot=128,
             layout="half", dtype="fp16", ctx_max=4096),
        # prompts: 4 sequences of 2047 tokens into empty and part-filled caches
        dict(name="append prompt", op="append", batch=4, q_len=2047, kv=8, group=4, dim=128, page=64, rot=128,
             layout="interleaved", dtype="bf16", ctx_max=3000),
        # one token of one short request: latency
        dict(name="attend one short", op="attend", batch=1, q_len=1, kv=8, group=4, dim=128, page=16, cache="int8",
             dtype="fp16", ctx_min=37, ctx_max=37, tree=False),
        # the repository's attention benchmark shape: B=8, k=8, context 4096, page 16
        dict(name="attend verify", op="attend", batch=8, q_len=9, kv=8, group=4, dim=128, page=16, cache="int8",
             dtype="fp16", ctx_min=4096, ctx_max=4096, tree=False),
        # decoding 32 requests of ragged lengths
        dict(name="attend ragged decode", op="attend", batch=32, q_len=1, kv=8, group=4, dim=128, page=64,
             cache="e4m3", dtype="bf16", ctx_min=1, ctx_max=8192, tree=False),
        # draft trees of 21 nodes over long contexts, wide groups, 64-wide heads
        dict(name="attend tree long", op="attend", batch=5, q_len=21, kv=2, group=8, dim=64, page=32, cache="e4m3",
             dtype="fp16", ctx_min=21, ctx_max=16421, tree=True),
        # a scheduler tick of a small server, one layer's cache
        dict(name="pages small", op="pages", rows=8, page=16, kv=8, dim=128, layers=1, len_max=500, beams=4),
        # a tick of a large one: 192 rows in beams of 4, 16 layers
        dict(name="pages large", op="pages", rows=192, page=16, kv=8, dim=128, layers=16, len_max=1200, beams=4),
        # 8 verified chains of 9 drafts, one layer
        dict(name="compact verify", op="compact", batch=8, q_len=9, kv=8, dim=128, page=16, layers=1, ctx_max=4096),
        # 48 draft trees of 33 nodes, 32 layers
        dict(name="compact trees", op="compact", batch=48, q_len=33, kv=8, dim=128, page=32, layers=32,
             ctx_max=1500),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("rope", "append", "attend", "attend", "pages", "compact"))
    dim = rng.choice((64, 128, 128))
    kv = rng.choice((1, 2, 4, 8))
    page = rng.choice((8, 16, 32, 64, 128))
    dtype = rng.choice(("fp16", "bf16"))
    layout = rng.choice(("half", "interleaved"))
    if op == "rope":
        heads, dtype = rng.randint(1, 40), rng.choice(("fp16", "bf16", "fp32"))
        return dict(op=op, rows=_log(rng, 1, 4095 if dtype == "fp32" else 8190), heads=heads, dim=dim,
                    rot=rng.choice((dim, dim, dim // 2)), layout=layout, dtype=dtype, inverse=rng.random() < 0.4,
                    n_pos=_log(rng, 1024, 65536), gap=rng.choice((0, 256, 1024)))
    if op == "append":
        batch, q_len = _log(rng, 1, 32), _log(rng, 1, 2047)
        q_len = max(1, min(q_len, 8188 // batch))
        return dict(op=op, batch=batch, q_len=q_len, kv=kv, group=rng.choice((1, 2, 4)), dim=dim, page=page,
                    rot=rng.choice((dim, dim, dim // 2)), layout=layout, dtype=dtype,
                    ctx_max=q_len + _log(rng, 1, 4096))
    if op == "attend":
        batch, q_len, group = _log(rng, 1, 48), _log(rng, 1, 33), rng.choice((1, 2, 4, 8))
        most = 32 * 8192 * 8 * 128 // (batch * kv * dim)
        most = min(most, 8 * 4096 * 9 * 4 * 8 * 128 // (batch * kv * dim * q_len * group))
        hi = _log(rng, q_len + 1, max(q_len + 2, min(32768, most)))
        return dict(op=op, batch=batch, q_len=q_len, kv=kv, group=group, dim=dim, page=page,
                    cache=rng.choice(("int8", "e4m3")), dtype=dtype, ctx_min=rng.choice((1, q_len, hi)), ctx_max=hi,
                    tree=rng.random() < 0.4)
    if op == "pages":
        rows = _log(rng, 2, 192)
        return dict(op=op, rows=rows, page=rng.choice((8, 16, 32, 64)), kv=kv, dim=dim, layers=_log(rng, 1, 16),
                    len_max=_log(rng, 8, 1200), beams=rng.choice((1, 2, 4)))
    batch, q_len = _log(rng, 1, 48), _log(rng, 2, 33)
    return dict(op=op, batch=batch, q_len=q_len, kv=kv, dim=dim, page=page, layers=_log(rng, 1, 32),
                ctx_max=q_len + _log(rng, 1, 1500))


# ---- inputs ------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _randint(g, lo, hi, shape, dtype=torch.int32):
    return torch.randint(lo, hi, shape, generator=g, device=DEV, dtype=dtype)


def _table(n_pos, rot, base=500000.0):
    """cos | sin of every position, [n_pos, rot] fp32: a model's table, made once in 64 bits."""
    inv = base ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=DEV) / rot)
    ang = torch.arange(n_pos, dtype=torch.float64, device=DEV)[:, None] * inv
    return torch.cat([ang.cos(), ang.sin()], 1).float()


def _stored(g, shape, cache):
    """Numbers as a quantised cache holds them: about normal, the largest near the type's end."""
    dt, top = CACHES[cache]
    n = 1 << 22
    base = (torch.randn(n, generator=g, device=DEV) * (top / 4)).clamp(-top, top)
    base = base.round().to(dt) if dt == torch.int8 else base.to(dt)
    total = math.prod(shape)
    if total <= n:
        return base[:total].reshape(shape)
    return base.view(torch.uint8).repeat(-(-total // n))[:total].view(dt).reshape(shape)


def _scales(g, shape, cache, lo=1.0, hi=3.0):
    top = CACHES[cache][1]
    return (torch.rand(shape, generator=g, device=DEV) * (hi - lo) + lo) / top


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    if op == "rope":
        T, H, D = case["rows"], case["heads"], case["dim"]
        dt = FLOATS[case["dtype"]]
        rows = torch.randn(T, H * D + case["gap"], generator=g, device=DEV).to(dt)   # the row of a projection
        return dict(case=case, x=rows[:, : H * D].view(T, H, D), pos=_randint(g, 0, case["n_pos"], (T,)),
                    table=_table(case["n_pos"], case["rot"]))
    page, kv, D = case["page"], case["kv"], case["dim"]
    if op == "append":
        B, Q, H = case["batch"], case["q_len"], case["kv"] * case["group"]
        T = B * Q
        dt = FLOATS[case["dtype"]]
        qkv = torch.randn(T, (H + 2 * kv) * D, generator=g, device=DEV).to(dt)
        ctx = _randint(g, Q, case["ctx_max"] + 1, (B,))
        C = -(-case["ctx_max"] // page) + 2
        P = B * C
        table = torch.randperm(P, generator=g, device=DEV, dtype=torch.int64).to(torch.int32).view(B, C)
        return dict(case=case, q=qkv[:, : H * D].view(T, H, D), k=qkv[:, H * D: (H + kv) * D].view(T, kv, D),
                    v=qkv[:, (H + kv) * D:].view(T, kv, D), ctx=ctx, tbl=table,
                    kc=_stored(g, (P, page, kv, D), "e4m3"), vc=_stored(g, (P, page, kv, D), "e4m3"),
                    ks=_scales(g, (P, kv), "e4m3", 0.5, 5.0), vs=_scales(g, (P, kv), "e4m3", 0.5, 5.0),
                    table=_table(case["ctx_max"] + 1, case["rot"]))
    if op == "attend":
        B, Q, H = case["batch"], case["q_len"], case["kv"] * case["group"]
        dt = FLOATS[case["dtype"]]
        ctx = _randint(g, case["ctx_min"], case["ctx_max"] + 1, (B,))
        ctx[0] = case["ctx_max"]
        C = -(-case["ctx_max"] // page)
        P = B * C + 3
        table = torch.randperm(P, generator=g, device=DEV, dtype=torch.int64)[: B * C].to(torch.int32).view(B, C)
        tree = None
        if case["tree"]:
            # node j's parent is an earlier node or the last verified token; a node sees its ancestors
            par = [-1] + [int(v) for v in
                          torch.randint(0, 1 << 30, (Q,), generator=torch.Generator().manual_seed(int(seed)))]
            masks = []
            for j in range(Q):
                p = par[j + 1] % (j + 1) - 1
                masks.append((masks[p] if p >= 0 else 0) | (1 << j))
            tree = torch.tensor([m - (1 << 64) if m >> 63 else m for m in masks], dtype=torch.int64, device=DEV)
            tree = tree[None].expand(B, Q).contiguous()
        return dict(case=case, q=torch.randn(B, Q, H, D, generator=g, device=DEV).to(dt),
                    kc=_stored(g, (P, page, kv, D), case["cache"]), vc=_stored(g, (P, page, kv, D), case["cache"]),
                    ks=_scales(g, (P, kv), case["cache"]), vs=_scales(g, (P, kv), case["cache"]), tbl=table, ctx=ctx,
                    tree=tree)
    if op == "pages":
        S, L, n = case["rows"], case["layers"], case["beams"]
        C = -(-case["len_max"] // page) + 2
        row = torch.arange(S, device=DEV)
        # beams of one request share the pages of its prompt: the first third of the leader's tokens
        lead = (row // n) * n
        want = _randint(g, 1, case["len_max"] + 1, (S,))
        want = want[lead].contiguous()
        full = -(-want // page)
        held = (full - _randint(g, 0, 2, (S,))).clamp(min=0)      # some rows need another page
        share = torch.minimum(held, held[lead]) // 3
        P = S * (C + 2)
        perm = torch.randperm(P, generator=g, device=DEV, dtype=torch.int64).to(torch.int32)[: S * C].view(S, C)
        col = torch.arange(C, device=DEV)
        tbl = torch.where(col < share[:, None], perm[lead], perm)
        tbl = torch.where(col < held[:, None], tbl, torch.full_like(tbl, -1))
        ref = torch.zeros(P + 1, dtype=torch.int32, device=DEV)
        ref.scatter_add_(0, torch.where(tbl < 0, P, tbl).long().flatten(),
                         (tbl >= 0).to(torch.int32).flatten())
        # a request that ended makes room for another; beams are reordered within their request
        drop = _randint(g, 0, 8, (S,))[lead] == 0
        parent = lead + (_randint(g, 0, n, (S,)) % (S - lead).clamp(max=n))
        parent = torch.where(_randint(g, 0, 4, (S,)) == 0, torch.full_like(parent, -1), parent)
        return dict(case=case, ref=ref[:P].contiguous(), tbl=tbl.contiguous(), held=held.to(torch.int32), drop=drop,
                    want=want.to(torch.int32), parent=parent.to(torch.int32),
                    kc=_stored(g, (L, P, page, kv, D), "e4m3"), vc=_stored(g, (L, P, page, kv, D), "e4m3"),
                    ks=_scales(g, (L, P, kv), "e4m3"), vs=_scales(g, (L, P, kv), "e4m3"))
    # compact
    B, Q, L = case["batch"], case["q_len"], case["layers"]
    ctx = _randint(g, Q, case["ctx_max"] + 1, (B,))
    C = -(-case["ctx_max"] // page) + 2
    NP = (Q - 1) // page + 2
    P = B * NP
    # the pool of this case has the pages that the drafts lie in; a table's earlier columns are not read
    first = (ctx - Q) // page
    perm = torch.randperm(P, generator=g, device=DEV, dtype=torch.int64).to(torch.int32).view(B, NP)
    tbl = torch.full((B, C + NP), -1, dtype=torch.int32, device=DEV)
    tbl.scatter_(1, first[:, None].long() + torch.arange(NP, device=DEV), perm)
    keep = torch.rand(B, Q, generator=g, device=DEV) < 0.4
    n_acc = keep.sum(1).to(torch.int32)
    accept = torch.where(keep, torch.arange(Q, device=DEV), Q).sort(1).values
    accept = accept.clamp(max=Q - 1).to(torch.int32)
    return dict(case=case, ctx=ctx, tbl=tbl, accept=accept.contiguous(), n_acc=n_acc,
                kc=_stored(g, (L, P, page, kv, D), "e4m3"), vc=_stored(g, (L, P, page, kv, D), "e4m3"),
                ks=_scales(g, (L, P, kv), "e4m3"), vs=_scales(g, (L, P, kv), "e4m3"))


# ---- one pass ----------------------------------------------------------------------------------
_package = None


def _specq():
    global _package
    if _package is None:
        at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "specdec-quant-triton_b200")
        if at not in sys.path:
            sys.path.insert(0, at)
        import specq
        _package = specq
    return _package


def run(s):
    op = s["case"]["op"]
    return (_OWN if own else _PLAIN)[op](s)


def _own_rope(s):
    return _specq().rope(s["x"], s["pos"], s["table"], layout=s["case"]["layout"], inverse=s["case"]["inverse"])


def _own_append(s):
    q = _specq().kv_append_blocks(s["k"], s["v"], s["kc"], s["vc"], s["ks"], s["vs"], s["tbl"], s["ctx"],
                                  s["case"]["q_len"], q=s["q"], table=s["table"], layout=s["case"]["layout"])
    return dict(q=q, kc=s["kc"], vc=s["vc"], ks=s["ks"], vs=s["vs"])


def _own_attend(s):
    return _specq().paged_attention_blocks(s["q"], s["kc"], s["vc"], s["ks"], s["vs"], s["tbl"], s["ctx"],
                                           tree=s["tree"])


def _own_pages(s):
    specq, page = _specq(), s["case"]["page"]
    specq.pages_release(s["ref"], s["tbl"], s["held"], s["drop"])
    short = specq.pages_reserve(s["ref"], s["tbl"], s["held"], s["want"], page)
    short2 = specq.pages_fork(s["kc"], s["vc"], s["ks"], s["vs"], s["ref"], s["tbl"], s["held"], s["parent"],
                              s["want"])
    return dict(ref=s["ref"], tbl=s["tbl"], held=s["held"], short=short, short2=short2, kc=s["kc"], vc=s["vc"],
                ks=s["ks"], vs=s["vs"])


def _own_compact(s):
    ctx = _specq().kv_compact_blocks(s["kc"], s["vc"], s["ks"], s["vs"], s["tbl"], s["ctx"], s["case"]["q_len"],
                                     s["accept"], s["n_acc"])
    return dict(ctx=ctx, kc=s["kc"], vc=s["vc"], ks=s["ks"], vs=s["vs"])


# ---- the plain forms ---------------------------------------------------------------------------
def _rotate(x, pos, table, layout, inverse=False):
    """x [T, H, D] in 32 or 64 bits: the first `rot` elements of each head turned by the position's angles."""
    rot = table.shape[1]
    h = rot // 2
    t = table[pos.long()].to(x.dtype)[:, None]
    c, n = t[..., :h], -t[..., h:] if inverse else t[..., h:]
    if layout == "half":
        a, b = x[..., :h], x[..., h:rot]
        return torch.cat([a * c - b * n, b * c + a * n, x[..., rot:]], -1)
    a, b = x[..., 0:rot:2], x[..., 1:rot:2]
    return torch.cat([torch.stack([a * c - b * n, b * c + a * n], -1).flatten(-2), x[..., rot:]], -1)


def _plain_rope(s):
    c = s["case"]
    return _rotate(s["x"].float(), s["pos"], s["table"], c["layout"], c["inverse"]).to(s["x"].dtype)


def _bytes_at(cache, idx):
    return cache.view(torch.uint8)[idx].view(cache.dtype)


def _append_one(x, cache, scale, pid, off, slot_new, slot_old, fresh, touched):
    """x [B, Q, kv, D] fp32 into the window of pages pid [B, N]; off [B, Q]: a token's slot in the window."""
    B, Q, kv, D = x.shape
    N, page = pid.shape[1], cache.shape[1]
    inv = torch.tensor(1.0 / 448.0, dtype=torch.float32, device=x.device)
    amax = torch.zeros(B, N, kv, dtype=torch.float32, device=x.device)
    amax = amax.scatter_reduce(1, (off // page)[..., None].expand(B, Q, kv), x.abs().amax(-1), "amax")
    old = scale[pid]
    need = amax.clamp(min=FLOOR) * inv
    new = torch.where(touched[..., None], torch.where(fresh[..., None], need, torch.maximum(old, need)), old)
    raw = _bytes_at(cache, pid)
    was = raw.float() * (old / new)[:, :, None, :, None]
    mine = torch.zeros(B, N * page, kv, D, dtype=torch.float32, device=x.device)
    mine.scatter_(1, off[..., None, None].expand(B, Q, kv, D), x)
    mine = mine.view(B, N, page, kv, D) * (1.0 / new)[:, :, None, :, None]
    to = torch.where(slot_new[..., None, None], mine, was).to(cache.dtype)
    keep = (slot_new | slot_old)[..., None, None]
    cache.view(torch.uint8)[pid] = torch.where(keep, to.view(torch.uint8), raw.view(torch.uint8))
    scale[pid] = new


def _window(ctx, Q, page, N, tbl):
    """The pages that the Q newest tokens of each sequence lie in, and which slots are whose."""
    base = ctx.long() - Q
    first = base // page
    col = first[:, None] + torch.arange(N, device=ctx.device)
    pid = tbl.gather(1, col).long()
    off = (base - first * page)[:, None] + torch.arange(Q, device=ctx.device)
    slot = (col[..., None] * page + torch.arange(page, device=ctx.device))
    slot_new = (slot >= base[:, None, None]) & (slot < ctx[:, None, None])
    touched = slot_new.any(-1)
    fresh = touched & slot_new[..., 0]
    slot_old = touched[..., None] & (slot < base[:, None, None])
    return pid, off, slot_new, slot_old, fresh, touched


def _plain_append(s):
    c = s["case"]
    B, Q, page, kv, D = c["batch"], c["q_len"], c["page"], c["kv"], c["dim"]
    pos = (s["ctx"][:, None] - Q + torch.arange(Q, device=s["ctx"].device)).flatten()
    q = _rotate(s["q"].float(), pos, s["table"], c["layout"]).to(s["q"].dtype)
    k = _rotate(s["k"].float(), pos, s["table"], c["layout"])
    # a window past the last page that is written falls on pages of the table that nothing uses
    w = _window(s["ctx"], Q, page, (Q - 1) // page + 2, s["tbl"])
    _append_one(k.view(B, Q, kv, D), s["kc"], s["ks"], *w)
    _append_one(s["v"].float().view(B, Q, kv, D), s["vc"], s["vs"], *w)
    return dict(q=q, kc=s["kc"], vc=s["vc"], ks=s["ks"], vs=s["vs"])


def _allowed(s, L):
    """[B, Q, L] True where a new token sees a cached one."""
    c, ctx = s["case"], s["ctx"].long()[:, None, None]
    Q = c["q_len"]
    t = torch.arange(L, device=ctx.device)
    qi = torch.arange(Q, device=ctx.device)[:, None]
    j = t - (ctx - Q)
    if s["tree"] is None:
        return j <= qi
    bit = (s["tree"][:, :, None] >> j.clamp(0, 63)) & 1
    return (j < 0) | ((j < Q) & (bit == 1))


def _plain_attend(s):
    c, q = s["case"], s["q"]
    B, Q, H, D = q.shape
    kv = c["kv"]
    idx = s["tbl"].long()
    k = (_bytes_at(s["kc"], idx).float() * s["ks"][idx][:, :, None, :, None]).view(B, -1, kv, D)
    v = (_bytes_at(s["vc"], idx).float() * s["vs"][idx][:, :, None, :, None]).view(B, -1, kv, D)
    x = torch.einsum("bqkgd,btkd->bkgqt", q.float().view(B, Q, kv, H // kv, D), k) * D ** -0.5
    x = x.masked_fill(~_allowed(s, k.shape[1])[:, None, None], -torch.inf)
    top = x.amax(-1, keepdim=True)
    p = (x - torch.where(torch.isfinite(top), top, torch.zeros_like(top))).exp()
    total = p.sum(-1)
    out = torch.einsum("bkgqt,btkd->bqkgd", p, v)
    total = total.permute(0, 3, 1, 2)[..., None]
    out = torch.where(total > 0, out / total.clamp(min=1e-30), torch.zeros_like(out))
    return out.reshape(B, Q, H, D).to(q.dtype)


def _plain_pages(s):
    c, ref, tbl, held = s["case"], s["ref"], s["tbl"], s["held"]
    page = c["page"]
    S, C = tbl.shape
    P = ref.shape[0]
    col = torch.arange(C, device=ref.device)
    one = torch.ones((), dtype=torch.int32, device=ref.device)
    more = torch.zeros(1, dtype=torch.int32, device=ref.device)

    def count(pages, here, sign):
        """ref +- 1 for each of `pages` where `here`; what is not here counts in one more slot."""
        wide = torch.cat([ref, more])
        at = torch.where(here, pages, torch.full_like(pages, P)).long().flatten()
        wide.scatter_add_(0, at, (sign * one).expand(at.shape))
        ref.copy_(wide[:P])

    # drop
    gone = s["drop"][:, None] & (col < held[:, None])
    count(tbl, gone, -1)
    tbl.copy_(torch.where(s["drop"][:, None], torch.full_like(tbl, -1), tbl))
    held.copy_(torch.where(s["drop"], torch.zeros_like(held), held))
    # reserve: the lowest free pages, row by row
    need = ((s["want"] + page - 1) // page - held).clamp(min=0)
    start = need.cumsum(0) - need
    free = ref == 0
    order = torch.sort((~free).to(torch.int32), stable=True).indices.to(torch.int32)
    short = (need.sum() - free.sum()).clamp(min=0).to(torch.int32).view(1)
    k = col - held[:, None]
    new = (k >= 0) & (k < need[:, None]) & (short == 0)
    got = order[(start[:, None] + k).clamp(0, P - 1).long()]
    tbl.copy_(torch.where(new, got, tbl))
    count(tbl, new, 1)
    held.add_(torch.where(short == 0, need, torch.zeros_like(need)).to(torch.int32))
    # fork: full pages shared, a part-filled last page copied to the lowest free one
    row = torch.arange(S, device=ref.device)
    forks = (s["parent"] >= 0) & (s["parent"] != row)
    par = torch.where(forks, s["parent"].long(), row)
    size = s["want"][par]
    n_full, rest = size // page, size % page
    part = forks & (rest > 0)
    free = ref == 0
    order = torch.sort((~free).to(torch.int32), stable=True).indices.to(torch.int32)
    short2 = (part.sum() - free.sum()).clamp(min=0).to(torch.int32).view(1)
    ok = short2 == 0
    forks, part = forks & ok, part & ok
    fresh = order[(part.cumsum(0) - 1).clamp(0, P - 1).long()]
    old = tbl.clone()
    from_parent = old[par]
    src = from_parent.gather(1, n_full.clamp(max=C - 1).long()[:, None])[:, 0]
    row_new = torch.where(col < n_full[:, None], from_parent, torch.full_like(old, -1))
    row_new = torch.where((col == n_full[:, None]) & part[:, None], fresh[:, None], row_new)
    # a row that copies nothing copies a page in use onto itself
    still = torch.argmax((ref > 0).to(torch.int32)).to(torch.int32)
    dst = torch.where(part, fresh, still).long()
    src = torch.where(part, src, still).long()
    slot = torch.arange(page, device=ref.device)
    src_slot = torch.where(slot < rest[:, None], src[:, None], dst[:, None])
    for_all = slice(None)
    _copy(s["kc"], for_all, dst, src_slot, slot)
    _copy(s["vc"], for_all, dst, src_slot, slot)
    s["ks"][:, dst] = s["ks"][:, src]
    s["vs"][:, dst] = s["vs"][:, src]
    count(row_new, forks[:, None] & (row_new >= 0), 1)
    count(old, forks[:, None] & (col < held[:, None]), -1)
    tbl.copy_(torch.where(forks[:, None], row_new, old))
    held.copy_(torch.where(forks, (n_full + part.to(torch.int32)).to(torch.int32), held))
    return dict(ref=ref, tbl=tbl, held=held, short=short, short2=short2, kc=s["kc"], vc=s["vc"], ks=s["ks"],
                vs=s["vs"])


def _copy(cache, layers, dst, src_slot, slot):
    raw = cache.view(torch.uint8)
    raw[layers, dst] = raw[layers, src_slot, slot]


def _compact_one(cache, scale, pid, at, to, valid, slot0, old_slots):
    """cache [L, P, page, kv, D]; pid [B, N] the window; at / to [B, Q] slots of the window."""
    L, _, page, kv, D = cache.shape
    B, N = pid.shape
    Q = at.shape[1]
    inv = torch.tensor(1.0 / 448.0, dtype=torch.float32, device=cache.device)
    raw = cache.view(torch.uint8)[:, pid]
    num = raw.view(cache.dtype).float().view(L, B, N * page, kv, D)
    old = scale[:, pid]                                                       # [L, B, N, kv]
    pick = at[None, :, :, None, None].expand(L, B, Q, kv, D)
    moved = num.gather(2, pick)
    src_scale = old.gather(2, (at // page)[None, :, :, None].expand(L, B, Q, kv))
    need = moved.abs().amax(-1) * inv * src_scale
    need = torch.where(valid[None, :, :, None], need, torch.zeros_like(need))
    page_to = (to // page)[None, :, :, None].expand(L, B, Q, kv)
    new = old.scatter_reduce(2, page_to, need, "amax")
    was = (num.view(L, B, N, page, kv, D) * (old / new)[:, :, :, None, :, None]).to(cache.dtype)
    out = torch.where(old_slots[None, :, :, :, None, None], was.view(torch.uint8), raw)
    moved = (moved * (src_scale / new.gather(2, page_to))[..., None]).to(cache.dtype).view(torch.uint8)
    wide = torch.cat([out.view(L, B, N * page, kv, D), torch.zeros_like(raw.view(L, B, -1, kv, D)[:, :, :1])], 2)
    put = torch.where(valid, to, N * page)[None, :, :, None, None].expand(L, B, Q, kv, D)
    wide.scatter_(2, put, moved)
    cache.view(torch.uint8)[:, pid] = wide[:, :, : N * page].reshape(L, B, N, page, kv, D)
    scale[:, pid] = new


def _compact_plan(s):
    c = s["case"]
    Q, page = c["q_len"], c["page"]
    N = (Q - 1) // page + 2
    base = s["ctx"].long() - Q
    first = base // page
    pid = s["tbl"].gather(1, first[:, None] + torch.arange(N, device=base.device)).long()
    slot0 = base - first * page
    j = torch.arange(Q, device=base.device)
    valid = j < s["n_acc"][:, None]
    at = slot0[:, None] + s["accept"].long()
    to = slot0[:, None] + j
    old_slots = torch.arange(N * page, device=base.device).view(1, N, page) < slot0[:, None, None]
    return pid, at, to, valid, slot0, old_slots


def _plain_compact(s):
    plan = _compact_plan(s)
    _compact_one(s["kc"], s["ks"], *plan)
    _compact_one(s["vc"], s["vs"], *plan)
    return dict(ctx=s["ctx"] - s["case"]["q_len"] + s["n_acc"], kc=s["kc"], vc=s["vc"], ks=s["ks"], vs=s["vs"])


_PLAIN = dict(rope=_plain_rope, append=_plain_append, attend=_plain_attend, pages=_plain_pages,
              compact=_plain_compact)
_OWN = dict(rope=_own_rope, append=_own_append, attend=_own_attend, pages=_own_pages, compact=_own_compact)


# ---- what a pass cannot do without ---------------------------------------------------------------
def work(case):
    c = case
    op, D = c["op"], c["dim"]
    if op == "rope":
        el = 4 if c["dtype"] == "fp32" else 2
        n = c["rows"] * c["heads"]
        return dict(bytes=n * D * el * 2 + c["rows"] * (4 + c["rot"] * 4), flops=n * c["rot"] * 3)
    kv, page = c["kv"], c["page"]
    if op == "append":
        T, H = c["batch"] * c["q_len"], kv * c["group"]
        reads = T * (H + 2 * kv) * D * 2 + T * c["rot"] * 4
        return dict(bytes=reads + T * H * D * 2 + T * 2 * kv * D + T / page * kv * 8,
                    flops=T * ((H + kv) * c["rot"] * 3 + 2 * kv * D * 3))
    if op == "attend":
        H = kv * c["group"]
        tokens = c["ctx_max"] + (c["batch"] - 1) * (c["ctx_min"] + c["ctx_max"]) / 2
        rows = c["batch"] * c["q_len"] * H
        return dict(bytes=tokens * kv * (2 * D + 8 / page) + tokens / page * 4 + rows * D * 4,
                    flops=4 * tokens * c["q_len"] * H * D)
    if op == "pages":
        S = c["rows"]
        cells = S * (c["len_max"] / 2 / page)
        copied = S * 0.75 * (1 - 1 / c["beams"]) * page / 2 * kv * D * 2 * c["layers"] + S
        return dict(bytes=2 * copied + cells * 4 * 3 + S * 8 * c["len_max"] / page, flops=0)
    moved = c["batch"] * c["q_len"] * 0.4 * kv * D * 2 * c["layers"] + c["batch"]
    return dict(bytes=2 * moved, flops=moved)


# ---- the definition in 64 bits ---------------------------------------------------------------------
def exact(case, seed):
    """Written apart from the plain form; an 8-bit number is given as the value before its rounding."""

    def turn(x, pos, table, layout, inverse):
        """Pairs as complex numbers times e^(+-i angle)."""
        x = x.double().clone()
        rot = table.shape[1]
        t = table.double()[pos.long()]
        turn = torch.complex(t[:, : rot // 2], -t[:, rot // 2:] if inverse else t[:, rot // 2:])[:, None]
        if layout == "half":
            z = torch.complex(x[..., : rot // 2], x[..., rot // 2: rot]) * turn
            x[..., : rot // 2], x[..., rot // 2: rot] = z.real, z.imag
        else:
            z = torch.complex(x[..., 0:rot:2], x[..., 1:rot:2]) * turn
            x[..., 0:rot:2], x[..., 1:rot:2] = z.real, z.imag
        return x

    def append(s):
        """Page by page; what an 8-bit number stands for is given before its rounding."""
        c = s["case"]
        B, Q, page = c["batch"], c["q_len"], c["page"]
        if B * (Q / page + 2) > 20000:
            return None
        ctx, tbl = s["ctx"].tolist(), s["tbl"].tolist()
        pos = torch.cat([torch.arange(n - Q, n, device=DEV) for n in ctx])
        q = turn(s["q"], pos, s["table"], c["layout"], False)
        k = turn(s["k"], pos, s["table"], c["layout"], False)
        got = dict(q=q)
        for name, x in (("k", k), ("v", s["v"].double())):
            cache, scale = s[name + "c"].double(), s[name + "s"].double()
            for b in range(B):
                base = ctx[b] - Q
                for col in range(base // page, (ctx[b] - 1) // page + 1):
                    p = tbl[b][col]
                    lo, hi = max(base, col * page), min(ctx[b], (col + 1) * page)
                    rows = x[b * Q + lo - base: b * Q + hi - base]
                    need = rows.abs().amax((0, 2)).clamp(min=FLOOR) / 448
                    new = need if lo == col * page else torch.maximum(need, scale[p])
                    cache[p, : lo - col * page] *= (scale[p] / new)[None, :, None]
                    cache[p, lo - col * page: hi - col * page] = rows / new[None, :, None]
                    scale[p] = new
            got[name + "c"], got[name + "s"] = cache, scale
        return got

    def attend(s):
        c, q = s["case"], s["q"].double()
        B, Q, H, D = q.shape
        G, page = c["group"], c["page"]
        out = torch.zeros_like(q)
        for b, n in enumerate(s["ctx"].tolist()):
            if n == 0:
                continue
            p = s["tbl"][b, : -(-n // page)].long()
            k = (_bytes_at(s["kc"], p).double() * s["ks"][p].double()[:, None, :, None]).flatten(0, 1)[:n]
            v = (_bytes_at(s["vc"], p).double() * s["vs"][p].double()[:, None, :, None]).flatten(0, 1)[:n]
            t = torch.arange(n, device=DEV)
            for i in range(Q):
                j = t - (n - Q)
                see = j <= i if s["tree"] is None else (j < 0) | ((s["tree"][b, i] >> j.clamp(0, 63)) & 1 == 1)
                if not bool(see.any()):
                    continue
                x = torch.einsum("kgd,tkd->kgt", q[b, i].view(-1, G, D), k[see]) / math.sqrt(D)
                out[b, i] = torch.einsum("kgt,tkd->kgd", torch.softmax(x, -1), v[see]).reshape(H, D)
        return out

    def compact(s):
        """Sequence by sequence; what an 8-bit number stands for is given before its rounding."""
        c = s["case"]
        Q, page = c["q_len"], c["page"]
        ctx, acc, n_acc, tbl = s["ctx"].tolist(), s["accept"].tolist(), s["n_acc"].tolist(), s["tbl"].tolist()
        got = dict(ctx=None)
        for name in "kv":
            cache, scale = s[name + "c"].double(), s[name + "s"].double()
            for b, n in enumerate(ctx):
                base = n - Q
                at = [divmod(base + a, page) for a in acc[b][: n_acc[b]]]
                for col in sorted({(base + j) // page for j in range(n_acc[b])}):
                    p, js = tbl[b][col], [j for j in range(n_acc[b]) if (base + j) // page == col]
                    rows = torch.stack([cache[:, tbl[b][at[j][0]], at[j][1]] for j in js], 1)
                    frm = torch.stack([scale[:, tbl[b][at[j][0]]] for j in js], 1)
                    vals = rows * frm[..., None]
                    new = torch.maximum(scale[:, p], vals.abs().amax((1, 3)) / 448)
                    first = (base + js[0]) % page
                    cache[:, p, :first] *= (scale[:, p] / new)[:, None, :, None]
                    cache[:, p, first: first + len(js)] = vals / new[:, None, :, None]
                    scale[:, p] = new
            got[name + "c"], got[name + "s"] = cache, scale
        return got

    s = prepare(case, seed)
    op = case["op"]
    if op == "rope":
        return turn(s["x"], s["pos"], s["table"], case["layout"], case["inverse"])
    if op == "append":
        return append(s)
    if op == "attend":
        return attend(s)
    if op == "compact":
        return compact(s)
    return None     # whole numbers and copies: nothing is computed
