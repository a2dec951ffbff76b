"""Cases of the operators for bounded caches, beams and normalised heads: what a pass reads and returns.

  norm     the RMS norm of every query and key head and its rotary turn in one pass, forward, or forward
           and backward (gradients of both inputs and both weights)
  select   a beam search's step: log-softmax of the beams' logits, added to their scores, and the best
           candidates of each request over all its beams and the vocabulary
  reorder  the beams' other states (token histories, lengths, recurrent states) moved to their parents' rows
  mass     the attention weight that the newest tokens give each cached token, added to a running sum
           (the cache holds 8-bit numbers with one fp32 scale for each page and KV head)
  evict    the tokens of least accumulated weight dropped from that cache, head by head, the kept ones
           moved together under their pages' new scales

`own` False: plain torch operations.  `own` True: this package's operators.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
FLOATS = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
CACHES = {"int8": (torch.int8, 127.0), "e4m3": (torch.float8_e4m3fn, 448.0)}
EPS = 1e-6


def listed():
    return [
        # one new token of one request, the head layout of this repository's stack
        dict(name="norm one token", op="norm", rows=1, heads=32, kv=8, dim=128, rot=128, layout="half", dtype="fp16",
             grad=False, n_pos=4096),
        # a prompt batch, interleaved pairs over the first half of each head
        dict(name="norm prompt", op="norm", rows=8190, heads=32, kv=8, dim=128, rot=64, layout="interleaved",
             dtype="bf16", grad=False, n_pos=32768),
        # a training step's sequence: both outputs and the four gradients
        dict(name="norm training", op="norm", rows=4093, heads=32, kv=8, dim=128, rot=128, layout="half",
             dtype="bf16", grad=True, n_pos=8192),
        # one request of four beams: latency
        dict(name="select one request", op="select", batch=1, beams=4, vocab=32000, n=4, dtype="fp16", masked=0.0,
             done=False, first=False),
        # 32 requests of 8 beams, an odd vocabulary, twice as many candidates as beams
        dict(name="select many beams", op="select", batch=32, beams=8, vocab=127999, n=16, dtype="bf16", masked=0.0,
             done=True, first=False),
        # 8 requests of 4 beams: token histories, lengths, flags
        dict(name="reorder histories", op="reorder", batch=8, beams=4, length=2000, width=0, dtype="fp16"),
        # 48 requests of 8 beams with recurrent states beside the histories
        dict(name="reorder states", op="reorder", batch=48, beams=8, length=1021, width=65544, dtype="bf16"),
        # one token of one short request: latency
        dict(name="mass one short", op="mass", batch=1, q_len=1, kv=8, group=4, dim=128, page=16, cache="int8",
             dtype="fp16", ctx_min=37, ctx_max=37, decay=1.0),
        # decoding 32 requests of ragged lengths
        dict(name="mass ragged decode", op="mass", batch=32, q_len=1, kv=8, group=4, dim=128, page=64, cache="e4m3",
             dtype="bf16", ctx_min=1, ctx_max=8192, decay=0.99),
        # the last 64 tokens of two long prompts look back over them
        dict(name="mass prompt window", op="mass", batch=2, q_len=64, kv=8, group=4, dim=128, page=32, cache="int8",
             dtype="fp16", ctx_min=12000, ctx_max=16384, decay=1.0),
        # 8 requests outgrow their budget, one layer
        dict(name="evict step", op="evict", batch=8, kv=8, dim=128, page=16, layers=1, ctx_max=700, keep=256,
             recent=32),
        # prompts cut down in all of a small model's layers
        dict(name="evict prompts", op="evict", batch=12, kv=8, dim=128, page=32, layers=4, ctx_max=2500, keep=1024,
             recent=128),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))


def draw(rng):
    op = rng.choice(("norm", "select", "reorder", "mass", "mass", "evict"))
    dim = rng.choice((64, 128, 128))
    kv = rng.choice((1, 2, 4, 8))
    page = rng.choice((8, 16, 32, 64, 128))
    dtype = rng.choice(("fp16", "bf16"))
    if op == "norm":
        dtype, grad = rng.choice(("fp16", "bf16", "fp32")), rng.random() < 0.5
        dim = rng.choice((64, 128, 128, 256))
        heads, kv = rng.randint(1, 32), rng.randint(1, 8)
        most = (4093 if grad else 8190) * 40 * 128 // ((heads + kv) * dim) // (2 if dtype == "fp32" else 1)
        return dict(op=op, rows=_log(rng, 1, min(most, 8190)), heads=heads, kv=kv, dim=dim,
                    rot=rng.choice((dim, dim, dim // 2)), layout=rng.choice(("half", "interleaved")), dtype=dtype,
                    grad=grad, n_pos=_log(rng, 1024, 65536))
    if op == "select":
        dtype = rng.choice(("fp16", "bf16", "fp32"))
        beams, vocab = _log(rng, 1, 16), _log(rng, 200, 200000)
        most = 32 * 8 * 127999 // (beams * vocab) // (2 if dtype == "fp32" else 1)
        return dict(op=op, batch=_log(rng, 1, max(1, min(64, most))), beams=beams, vocab=vocab,
                    n=beams * rng.choice((1, 2)), dtype=dtype, masked=rng.choice((0.0, 0.0, 0.5, 0.999)),
                    done=rng.random() < 0.5, first=rng.random() < 0.25)
    if op == "reorder":
        batch, beams = _log(rng, 1, 48), _log(rng, 2, 16)
        most = 48 * 8 * 65544 // (batch * beams)
        return dict(op=op, batch=batch, beams=beams, length=_log(rng, 1, 2000),
                    width=rng.choice((0, _log(rng, 1, min(65544, most)))), dtype=dtype)
    if op == "mass":
        batch, q_len, group = _log(rng, 1, 32), rng.choice((1, _log(rng, 1, 64))), rng.choice((1, 2, 4, 8))
        even = rng.random() < 0.33       # all contexts of one length, or spread below the longest
        most = 32 * (4000 if even else 8000) * 8 * 128 // (batch * kv * dim)
        most = min(most, 2 * 64 * 4 * 14000 * 8 * 128 // (batch * q_len * group * kv * dim))
        hi = _log(rng, q_len + 1, max(q_len + 2, min(32768, most)))
        return dict(op=op, batch=batch, q_len=q_len, kv=kv, group=group, dim=dim, page=page,
                    cache=rng.choice(("int8", "e4m3")), dtype=dtype, ctx_min=hi if even else rng.choice((1, q_len)),
                    ctx_max=hi, decay=rng.choice((1.0, 0.9)))
    batch, layers = _log(rng, 1, 12), _log(rng, 1, 4)
    ctx_max = _log(rng, 32, min(8192, 12 * 4 * 2500 * 8 * 128 // (batch * layers * kv * dim)))
    keep = _log(rng, 16, max(16, min(1024, ctx_max - 1)))
    return dict(op=op, batch=batch, kv=kv, dim=dim, page=page, layers=layers, ctx_max=ctx_max, keep=keep,
                recent=rng.choice((0, 1, keep // 8, keep // 2, keep)))


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


def _tables(g, B, C, extra):
    P = B * C + extra
    return P, torch.randperm(P, generator=g, device=DEV, dtype=torch.int64)[: B * C].to(torch.int32).view(B, C)


def prepare(case, seed):
    g, c = _gen(seed), case
    op = case["op"]
    if op == "norm":
        T, H, KV, D = c["rows"], c["heads"], c["kv"], c["dim"]
        dt = FLOATS[c["dtype"]]
        qkv = (torch.randn(T, (H + 2 * KV) * D, generator=g, device=DEV) * 1.5).to(dt)   # a projection's rows
        s = dict(case=case, q=qkv[:, : H * D].view(T, H, D), k=qkv[:, H * D: (H + KV) * D].view(T, KV, D),
                 qw=(1 + 0.2 * torch.randn(D, generator=g, device=DEV)).to(dt),
                 kw=(1 + 0.2 * torch.randn(D, generator=g, device=DEV)).to(dt),
                 pos=_randint(g, 0, c["n_pos"], (T,)), table=_table(c["n_pos"], c["rot"]))
        if c["grad"]:
            s["gq"] = torch.randn(T, H, D, generator=g, device=DEV).to(dt)
            s["gk"] = torch.randn(T, KV, D, generator=g, device=DEV).to(dt)
            for name in ("q", "k", "qw", "kw"):
                s[name].requires_grad_(True)
        return s
    if op == "select":
        B, K, V = c["batch"], c["beams"], c["vocab"]
        logits = torch.randn(B * K, V, generator=g, device=DEV) * 3
        # some tokens stand out in each row, as they do for a trained model
        peak = torch.randn(B * K, V, generator=g, device=DEV)
        logits += torch.where(peak > 3.0, 4 * (peak - 2), torch.zeros_like(peak))
        if c["masked"]:      # a grammar allows few tokens
            logits.masked_fill_(torch.rand(B * K, V, generator=g, device=DEV) < c["masked"], -torch.inf)
        scores = -torch.rand(B, K, generator=g, device=DEV) * 20
        if c["first"]:       # the beams of a request are alike: only the first counts
            scores[:, 1:] = -torch.inf
        done = torch.rand(B * K, generator=g, device=DEV) < 0.15 if c["done"] else None
        return dict(case=case, logits=logits.to(FLOATS[c["dtype"]]), scores=scores, done=done)
    if op == "reorder":
        B, K = c["batch"], c["beams"]
        R = B * K
        first = (torch.arange(R, device=DEV) // K) * K
        parent = (first + _randint(g, 0, K, (R,))).to(torch.int32)
        keep = _randint(g, 0, 4, (R,)) == 0          # some beams go on in their own row
        parent = torch.where(keep, torch.arange(R, device=DEV, dtype=torch.int32), parent)
        states = [_randint(g, 0, 1 << 17, (R, c["length"])), _randint(g, 1, 1 << 12, (R,)),
                  _randint(g, 0, 2, (R,)).bool()]
        if c["width"]:
            states.append(torch.randn(R, c["width"], generator=g, device=DEV).to(FLOATS[c["dtype"]]))
        return dict(case=case, parent=parent, states=states)
    page, kv, D = c["page"], c["kv"], c["dim"]
    if op == "mass":
        B, Q, H = c["batch"], c["q_len"], kv * c["group"]
        ctx = _randint(g, c["ctx_min"], c["ctx_max"] + 1, (B,))
        ctx[0] = c["ctx_max"]
        C = -(-c["ctx_max"] // page)
        P, tbl = _tables(g, B, C, 3)
        return dict(case=case, q=torch.randn(B, Q, H, D, generator=g, device=DEV).to(FLOATS[c["dtype"]]),
                    kc=_stored(g, (P, page, kv, D), c["cache"]), ks=_scales(g, (P, kv), c["cache"]), tbl=tbl, ctx=ctx,
                    mass=torch.rand(B, kv, C * page, generator=g, device=DEV))
    # evict: accumulated weights as attention leaves them: few large, many small, some tokens never seen
    B, L = c["batch"], c["layers"]
    ctx = _randint(g, max(1, c["ctx_max"] // 2), c["ctx_max"] + 1, (B,))
    ctx[0] = c["ctx_max"]
    C = -(-c["ctx_max"] // page)
    P, tbl = _tables(g, B, C, 3)
    mass = torch.rand(L, B, kv, C * page, generator=g, device=DEV) ** 8 * 10
    mass[torch.rand(L, B, kv, C * page, generator=g, device=DEV) < 0.02] = 0.0
    return dict(case=case, kc=_stored(g, (L, P, page, kv, D), "e4m3"), vc=_stored(g, (L, P, page, kv, D), "e4m3"),
                ks=_scales(g, (L, P, kv), "e4m3"), vs=_scales(g, (L, P, kv), "e4m3"), tbl=tbl, ctx=ctx, mass=mass)


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


def _own_norm(s):
    c = s["case"]
    q, k = _specq().qk_norm_rope(s["q"], s["k"], s["qw"], s["kw"], s["pos"], s["table"], eps=EPS, layout=c["layout"])
    if not c["grad"]:
        return dict(q=q, k=k)
    dq, dk, dqw, dkw = torch.autograd.grad((q, k), (s["q"], s["k"], s["qw"], s["kw"]), (s["gq"], s["gk"]))
    return dict(q=q.detach(), k=k.detach(), dq=dq, dk=dk, dqw=dqw, dkw=dkw)


def _own_select(s):
    c = s["case"]
    scores, parent, token = _specq().beam_select(s["logits"], s["scores"], n=c["n"], done=s["done"], pad=1)
    return dict(scores=scores, parent=parent, token=token)


def _own_reorder(s):
    _specq().beam_reorder(s["states"], s["parent"], s["case"]["beams"])
    return s["states"]


def _own_mass(s):
    return _specq().attention_mass_blocks(s["q"], s["kc"], s["ks"], s["tbl"], s["ctx"], s["mass"],
                                          decay=s["case"]["decay"])


def _own_evict(s):
    c = s["case"]
    ctx = _specq().kv_evict_blocks(s["kc"], s["vc"], s["ks"], s["vs"], s["tbl"], s["ctx"], s["mass"], c["keep"],
                                   c["recent"])
    return dict(ctx=ctx, kc=s["kc"], vc=s["vc"], ks=s["ks"], vs=s["vs"], mass=s["mass"])


# ---- the plain forms ---------------------------------------------------------------------------
def _rotate(x, pos, table, layout, sign=1.0):
    """x [T, H, D]: the first `rot` elements of each head turned by the position's angles (sign -1: back)."""
    rot = table.shape[1]
    h = rot // 2
    t = table[pos.long()].to(x.dtype)[:, None]
    c, n = t[..., :h], t[..., h:] * sign
    if layout == "half":
        a, b = x[..., :h], x[..., h:rot]
        return torch.cat([a * c - b * n, b * c + a * n, x[..., rot:]], -1)
    a, b = x[..., 0:rot:2], x[..., 1:rot:2]
    return torch.cat([torch.stack([a * c - b * n, b * c + a * n], -1).flatten(-2), x[..., rot:]], -1)


def _plain_norm(s):
    c, out = s["case"], {}
    with torch.no_grad():
        for name in "qk":
            x, w = s[name].float(), s[name + "w"].float()
            r = 1 / (x.square().mean(-1, keepdim=True) + EPS).sqrt()
            out[name] = _rotate(x * r * w, s["pos"], s["table"], c["layout"]).to(s[name].dtype)
            if c["grad"]:
                u = _rotate(s["g" + name].float(), s["pos"], s["table"], c["layout"], -1.0)
                hat, uw = x * r, u * w
                out["d" + name] = (r * (uw - hat * (uw * hat).mean(-1, keepdim=True))).to(s[name].dtype)
                out["d" + name + "w"] = (u * hat).sum((0, 1), dtype=torch.float64).to(s[name + "w"].dtype)
    return out


def _plain_select(s):
    c = s["case"]
    B, K, V, n = c["batch"], c["beams"], c["vocab"], c["n"]
    # in 64 bits: candidates of two beams may lie a few fp32 steps apart, and their order is an output
    x = s["logits"].double()
    top = x.amax(-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, torch.zeros_like(top))
    logp = x - top - (x - top).exp().sum(-1, keepdim=True).log()
    logp = torch.where(x == -torch.inf, torch.full_like(x, -torch.inf), logp)
    if s["done"] is not None:       # a finished beam stays as it is, by its pad token
        stay = torch.full((V,), -torch.inf, dtype=torch.float64, device=x.device)
        stay[1] = 0.0
        logp = torch.where(s["done"][:, None], stay, logp)
    total = (s["scores"].double().view(B, K, 1) + logp.view(B, K, V)).view(B, K * V)
    best, at = torch.sort(total, dim=-1, descending=True, stable=True)
    if K * V < n:
        best = torch.cat([best, best.new_full((B, n - K * V), -torch.inf)], 1)
        at = torch.cat([at, at.new_zeros((B, n - K * V))], 1)
    best, at = best[:, :n], at[:, :n]
    none = best == -torch.inf
    first = torch.arange(B, device=x.device)[:, None] * K
    parent = torch.where(none, first + torch.arange(n, device=x.device) % K, first + at // V)
    token = torch.where(none, torch.ones_like(at), at % V)
    return dict(scores=best.float(), parent=parent.to(torch.int32), token=token.to(torch.int32))


def _plain_reorder(s):
    at = s["parent"].long()
    for x in s["states"]:
        x.copy_(x[at])
    return s["states"]


def _bytes_at(cache, idx):
    return cache.view(torch.uint8)[idx].view(cache.dtype)


def _plain_mass(s):
    c, q = s["case"], s["q"]
    B, Q, H, D = q.shape
    kv = c["kv"]
    idx = s["tbl"].long()
    k = (_bytes_at(s["kc"], idx).float() * s["ks"][idx][:, :, None, :, None]).view(B, -1, kv, D)
    x = torch.einsum("bqkgd,btkd->bkgqt", q.float().view(B, Q, kv, H // kv, D), k) * D ** -0.5
    t = torch.arange(k.shape[1], device=q.device)
    n = s["ctx"].long()[:, None, None]
    see = t <= n - Q + torch.arange(Q, device=q.device)[:, None]                      # [B, Q, T]
    x = x.masked_fill(~see[:, None, None], -torch.inf)
    top = x.amax(-1, keepdim=True)
    p = (x - torch.where(torch.isfinite(top), top, torch.zeros_like(top))).exp()
    total = p.sum(-1, keepdim=True)
    w = torch.where(total > 0, p / total.clamp(min=1e-30), torch.zeros_like(p)).sum((2, 3))
    live = (t < s["ctx"][:, None])[:, None]
    m = s["mass"]
    m.copy_(torch.where(live, m * c["decay"] + w, m))
    return m


def _plain_evict(s):
    c = s["case"]
    L, B, KV, D, page = c["layers"], c["batch"], c["kv"], c["dim"], c["page"]
    keep, recent = c["keep"], c["recent"]
    N = s["mass"].shape[-1]
    C = N // page
    t = torch.arange(N, device=DEV)
    n = s["ctx"].long()[None, :, None, None]
    # the newest tokens count as heaviest of all, what is past the end as nothing
    m = s["mass"]
    worth = torch.where(t >= n - recent, torch.full_like(m, torch.inf), m)
    worth = torch.where(t >= n, torch.full_like(m, -torch.inf), worth)
    order = torch.sort(worth, dim=-1, descending=True, stable=True).indices[..., :keep]
    at = torch.sort(order, -1).values                                                  # [L, B, KV, k]
    k = at.shape[-1]
    j = torch.arange(k, device=DEV)
    cut = n > keep
    at = torch.where(cut, at, j.expand_as(at))
    moved = torch.where(cut, m.gather(-1, at), m[..., :k])
    new_mass = torch.where(cut & (t >= keep) & (t < n), torch.zeros_like(m), m)
    new_mass[..., :k] = moved
    m.copy_(new_mass)
    lay = torch.arange(L, device=DEV)[:, None, None, None]
    head = torch.arange(KV, device=DEV)[None, None, :, None]
    pages = s["tbl"].long()[None, :, None, :].expand(L, B, KV, C)
    src, dst = pages.gather(-1, at // page), pages[..., : -(-k // page)].repeat_interleave(page, -1)[..., :k]
    for cache, scale in ((s["kc"], s["ks"]), (s["vc"], s["vs"])):
        was = scale[lay, src, head]                                                    # [L, B, KV, k]
        pad = (-k) % page
        per_page = torch.cat([was, was.new_zeros(L, B, KV, pad)], -1).view(L, B, KV, -1, page).amax(-1)
        new = per_page.repeat_interleave(page, -1)[..., :k]
        raw = cache.view(torch.uint8)
        num = raw[lay, src, at % page, head].view(cache.dtype)
        out = (num.float() * (was / new)[..., None]).to(cache.dtype)
        here = cut.expand(L, B, KV, k)
        slot = (j % page).expand(L, B, KV, k)
        old = raw[lay, dst, slot, head]
        raw[lay, dst, slot, head] = torch.where(here[..., None], out.view(torch.uint8), old)
        first = pages[..., : per_page.shape[-1]]
        scale[lay, first, head] = torch.where(cut, per_page, scale[lay, first, head])
    return dict(ctx=s["ctx"].clamp(max=keep), kc=s["kc"], vc=s["vc"], ks=s["ks"], vs=s["vs"], mass=m)


_PLAIN = dict(norm=_plain_norm, select=_plain_select, reorder=_plain_reorder, mass=_plain_mass, evict=_plain_evict)
_OWN = dict(norm=_own_norm, select=_own_select, reorder=_own_reorder, mass=_own_mass, evict=_own_evict)


# ---- what a pass cannot do without ---------------------------------------------------------------
def work(case):
    c = case
    op = c["op"]
    el = 4 if c.get("dtype") == "fp32" else 2
    if op == "norm":
        n = c["rows"] * (c["heads"] + c["kv"]) * c["dim"]
        b, f = n * el * 2 + c["rows"] * (4 + c["rot"] * 4), n * 7
        if c["grad"]:
            b, f = b + n * el * 3 + c["rows"] * (4 + c["rot"] * 4), f + n * 16
        return dict(bytes=b, flops=f)
    if op == "select":
        rows = c["batch"] * c["beams"]
        return dict(bytes=rows * (c["vocab"] * el * (1 / c["beams"] if c["first"] else 1) + 4) + c["batch"] * c["n"] * 12,
                    flops=rows * c["vocab"] * 3)
    if op == "reorder":
        rows = c["batch"] * c["beams"] * 0.75 * (1 - 1 / c["beams"])
        return dict(bytes=2 * rows * (c["length"] * 4 + 5 + c["width"] * 2) + c["batch"] * c["beams"] * 4, flops=0)
    kv, page, D = c["kv"], c["page"], c["dim"]
    if op == "mass":
        tokens = c["ctx_max"] + (c["batch"] - 1) * (c["ctx_min"] + c["ctx_max"]) / 2
        rows = c["q_len"] * kv * c["group"]
        return dict(bytes=tokens * kv * (D + 4 / page + 8) + tokens / page * 4 + c["batch"] * rows * D * 2,
                    flops=2 * tokens * rows * D)
    # evict: the mean length is three quarters of the longest
    n = c["ctx_max"] * 0.75
    heads = c["layers"] * c["batch"] * kv
    kept = min(c["keep"], n)
    return dict(bytes=heads * (n * 4 + kept * 4 + (kept * (D + 4 / page) * 2) * 2), flops=heads * kept * D * 2)


# ---- the definition in 64 bits ---------------------------------------------------------------------
def exact(case, seed):
    """Written apart from the plain form; an 8-bit number is given as the value before its rounding."""
    c = case

    def norm(s):
        """Pairs as complex numbers times e^(i angle); the gradients by differentiation of that."""
        rot = c["rot"]
        t = s["table"].double()[s["pos"].long()]
        turn = torch.complex(t[:, : rot // 2], t[:, rot // 2:])[:, None]
        out = {}
        for name in "qk":
            x = s[name].detach().double().requires_grad_(c["grad"])
            w = s[name + "w"].detach().double().requires_grad_(c["grad"])
            y = x * w / torch.sqrt((x * x).sum(-1, keepdim=True) / c["dim"] + EPS)
            if c["layout"] == "half":
                z = torch.complex(y[..., : rot // 2], y[..., rot // 2: rot]) * turn
                y = torch.cat([z.real, z.imag, y[..., rot:]], -1)
            else:
                z = torch.view_as_complex(y[..., :rot].unflatten(-1, (-1, 2)).contiguous()) * turn
                y = torch.cat([torch.view_as_real(z).flatten(-2), y[..., rot:]], -1)
            out[name] = y.detach()
            if c["grad"]:
                out["d" + name], out["d" + name + "w"] = torch.autograd.grad(y, (x, w), s["g" + name].double())
        return out

    def select(s):
        """Request by request; the order of candidates is no number, their scores are."""
        best = torch.full((c["batch"], c["n"]), -torch.inf, dtype=torch.float64, device=DEV)
        for b in range(c["batch"]):
            rows = range(b * c["beams"], (b + 1) * c["beams"])
            found = []
            for r in rows:
                score = s["scores"].view(-1)[r].double()
                if s["done"] is not None and bool(s["done"][r]):
                    found.append(score.view(1))
                else:
                    found.append(torch.log_softmax(s["logits"][r].double(), -1).topk(min(c["n"], c["vocab"])).values + score)
            found = torch.cat(found).nan_to_num(nan=-torch.inf, neginf=-torch.inf).sort(descending=True).values[: c["n"]]
            best[b, : found.numel()] = found
        return dict(scores=best, parent=None, token=None)

    def mass(s):
        q, page, G = s["q"].double(), c["page"], c["group"]
        Q, D = q.shape[1], q.shape[3]
        out = s["mass"].double()
        for b, n in enumerate(s["ctx"].tolist()):
            p = s["tbl"][b, : -(-n // page)].long()
            k = (_bytes_at(s["kc"], p).double() * s["ks"][p].double()[:, None, :, None]).flatten(0, 1)[:n]
            out[b, :, :n] *= c["decay"]
            for i in range(Q):
                e = n - Q + i + 1
                if e > 0:
                    x = torch.einsum("kgd,tkd->kgt", q[b, i].view(-1, G, D), k[:e]) / math.sqrt(D)
                    out[b, :, :e] += torch.softmax(x, -1).sum(1)
        return out

    def evict(s):
        """Head by head, page by page of the kept tokens."""
        page, keep, recent = c["page"], c["keep"], c["recent"]
        got = dict(ctx=None, mass=s["mass"].double())
        src = {}
        for x in "kv":
            got[x + "c"], got[x + "s"] = s[x + "c"].double(), s[x + "s"].double()
            src[x] = (s[x + "c"], s[x + "s"])
        for b, n in enumerate(s["ctx"].tolist()):
            if n <= keep:
                continue
            tbl = s["tbl"][b].long()
            dst = torch.arange(keep, device=DEV)
            edge = torch.arange(0, keep, page)
            for l in range(c["layers"]):
                for h in range(c["kv"]):
                    m = s["mass"][l, b, h, : n - recent].double()
                    heavy = torch.argsort(-m, dim=0, stable=True)[: keep - recent]
                    at = torch.cat([heavy.sort().values, torch.arange(n - recent, n, device=DEV)])
                    got["mass"][l, b, h, :n] = 0
                    got["mass"][l, b, h, :keep] = s["mass"][l, b, h, at].double()
                    p = tbl[at // page]
                    for x in "kv":
                        cache, scale = src[x]
                        own_scale = scale[l, p, h].double()
                        wide = torch.nn.functional.pad(own_scale, (0, (-keep) % page)).view(-1, page).amax(1)
                        value = _bytes_at(cache, (l, p, at % page, h)).double() * own_scale[:, None]
                        got[x + "c"][l, tbl[dst // page], dst % page, h] = value / wide[dst // page][:, None]
                        got[x + "s"][l, tbl[: edge.numel()], h] = wide
        return got

    s = prepare(case, seed)
    if case["op"] == "reorder":     # copies; whole numbers are no computed ones
        if not c["width"]:
            return None
        at = s["parent"].long().cpu()
        return [x.cpu()[at].to(x.device) if x.is_floating_point() else None for x in s["states"]]
    return dict(norm=norm, select=select, mass=mass, evict=evict)[case["op"]](s)
