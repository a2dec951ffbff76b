"""Plain numpy forms of the operators around a bounded cache, beams and normalised heads, in 64 bits.

  norm_turn, norm_turn_grad   RMS norm of heads with their rotary turn; its gradients
  beam_select                 the best continuations of each request
  attention_mass              the weight that the newest tokens give each cached one
  evict_choice, evict         the kept tokens of one row; a cache cut down (numbers as the kernels round them)
"""
import numpy as np

from .block_oracle import turn


def norm_turn(x, w, table, pos, layout, eps):
    """x [T, H, D], w [D] or None."""
    x = np.asarray(x, np.float64)
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    return turn(y if w is None else y * w, table, pos, layout, False)


def norm_turn_grad(x, w, g, table, pos, layout, eps):
    """dx, dw from g, the gradient of norm_turn's output."""
    x, g = np.asarray(x, np.float64), np.asarray(g, np.float64)
    r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    u = turn(g, table, pos, layout, True)
    uw = u if w is None else u * w
    hat = x * r
    return r * (uw - hat * (uw * hat).mean(-1, keepdims=True)), (u * hat).sum((0, 1))


def beam_totals(logits, scores, done, pad):
    """Totals of every candidate, [B, K * V]; -inf: none.  logits [B * K, V], scores [B, K]."""
    B, K = scores.shape
    x = np.asarray(logits, np.float64)
    x = np.where(np.isnan(x), -np.inf, np.minimum(x, np.finfo(np.float32).max))
    with np.errstate(all="ignore"):
        top = x.max(-1, keepdims=True)
        z = np.where(np.isfinite(top), top, 0.0)
        logp = x - z - np.log(np.exp(x - z).sum(-1, keepdims=True))
        logp = np.where(np.isfinite(x), logp, -np.inf)
    if done is not None:
        stay = np.full(x.shape[1], -np.inf)
        stay[pad] = 0.0
        logp = np.where(np.asarray(done).reshape(-1, 1), stay, logp)
    s = np.asarray(scores, np.float64).reshape(-1, 1)
    total = np.where(np.isfinite(s), s, 0.0) + logp
    return np.where(np.isfinite(s), total, -np.inf).reshape(B, -1)


def beam_select(logits, scores, n, done=None, pad=0):
    """scores', parent, token, each [B, n]."""
    B, K = scores.shape
    V = logits.shape[1]
    total = beam_totals(logits, scores, done, pad)
    out, parent, token = np.full((B, n), -np.inf), np.zeros((B, n), np.int64), np.full((B, n), pad, np.int64)
    for b in range(B):
        order = np.argsort(-total[b], kind="stable")[:n]
        for j in range(n):
            parent[b, j] = b * K + j % K
            if j < len(order) and total[b, order[j]] > -np.inf:
                out[b, j], parent[b, j], token[b, j] = total[b, order[j]], b * K + order[j] // V, order[j] % V
    return out, parent, token


def gather(cache, scale, pages, n):
    """The first n tokens of a row: [n, H_KV, D] in 64 bits; a page outside the cache gives NaN."""
    out = []
    for p in pages:
        if 0 <= p < cache.shape[0]:
            out.append(np.asarray(cache[p], np.float64) * np.asarray(scale[p], np.float64)[None, :, None])
        else:
            out.append(np.full(cache.shape[1:], np.nan))
    return np.concatenate(out, 0)[:n] if out else np.zeros((0,) + cache.shape[2:])


def attention_mass(q, kc, ks, tbl, ctx, mass, n_rows=None, decay=1.0, sm_scale=None):
    """q [B, Q, H, D], kc [P, page, KV, D] (numbers), mass [B, KV, N] -> (mass', largest sum of |q k| sm_scale)."""
    B, Q, H, D = q.shape
    page, KV = kc.shape[1], kc.shape[2]
    G, sm = H // KV, D ** -0.5 if sm_scale is None else sm_scale
    out, size = np.array(mass, np.float64), 0.0
    for b in range(B):
        n = min(int(ctx[b]), tbl.shape[1] * page)
        rows = Q if n_rows is None else min(max(int(n_rows[b]), 0), Q)
        if n <= 0 or rows == 0:
            continue
        k = gather(kc, ks, tbl[b, : -(-n // page)], n)
        out[b, :, :n] *= decay
        for i in range(rows):
            e = n - rows + i + 1
            if e <= 0:
                continue
            for h in range(KV):
                kk = k[:e, h]
                here = ~np.isnan(kk[:, 0])
                for g in range(G):
                    v = np.asarray(q[b, i, h * G + g], np.float64)
                    if not np.isfinite(v).all() or not here.any():
                        continue
                    s = kk[here] @ v * sm
                    size = max(size, float((np.abs(kk[here]) @ np.abs(v)).max() * sm))
                    p = np.exp(s - s.max())
                    out[b, h, :e][here] += p / p.sum()
    return out, size


def evict_choice(mass, n, keep, recent):
    """Kept tokens of a row of n > keep, in order: the newest `recent` and the heaviest others."""
    m = np.asarray(mass[: n - recent], np.float64)
    m = np.where(np.isnan(m), -np.inf, m)
    heavy = np.sort(np.argsort(-m, kind="stable")[: keep - recent])
    return np.concatenate([heavy, np.arange(n - recent, n)])


def evict(cache, scale, tbl, ctx, mass, keep, recent, requant):
    """One layer's K or V cut down in place: cache [P, page, KV, D] of numbers (fp32), scale fp32 [P, KV].
    requant(numbers, ratio fp32) rounds as the cache's type does.  mass is only read."""
    page = cache.shape[1]
    src, was = cache.copy(), scale.copy()
    for b, n in enumerate(ctx):
        if n <= keep:
            continue
        for h in range(cache.shape[2]):
            at = evict_choice(mass[b, h], n, keep, recent)
            for c in range(-(-keep // page)):
                mine = at[c * page: (c + 1) * page]
                pages = tbl[b, mine // page]
                s = was[pages, h]
                new = s.max()
                dst = tbl[b, c]
                for j, (t, p) in enumerate(zip(mine, pages)):
                    row = src[p, t % page, h]
                    cache[dst, j, h] = row if s[j] == new else requant(row, np.float32(s[j]) / np.float32(new))
                scale[dst, h] = new
