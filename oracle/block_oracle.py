"""Oracle of the block-scaled KV-cache operators, in numpy, from their formulas.

Attention and rotary positions are in float64.  Append and compaction are defined in fp32 with
stated roundings (numpy's float32 arithmetic is IEEE, one rounding an operation), so their 8-bit
numbers and scales are exact; the page pool is integers.  An 8-bit number is carried as the value
it stands for before the scale (int8: -127..127, e4m3: its value).
"""
from __future__ import annotations

import numpy as np

F = np.float32
QMAX = {"int8": F(127.0), "e4m3": F(448.0)}
FLOOR = F(1e-8)


def e4m3_round(y):
    """Round fp32 to e4m3 (nearest even, saturated at +-448), as float32 values."""
    y = np.asarray(y, F)
    a = np.abs(y.astype(np.float64))
    e = np.floor(np.log2(np.maximum(a, 2.0 ** -40)))
    e = np.maximum(e, -6.0)                          # subnormals share the least exponent
    step = 2.0 ** (e - 3)
    q = np.rint(a / step) * step                     # numpy rounds half to even
    return (np.sign(y) * np.minimum(q, 448.0)).astype(F)


def store(y, cache):
    y = np.asarray(y, F)
    if cache == "int8":
        return np.rint(np.clip(y, F(-127), F(127))).astype(F)
    return e4m3_round(y)


def inv_qmax(cache):
    return F(1.0) / QMAX[cache]


def turn(x, table, pos, layout, inverse=False):
    """x [T, H, D] -> float64, rotated by row pos[t] of table [n_pos, rot] (cosines | sines)."""
    x = np.array(x, np.float64)
    rot = table.shape[1]
    h = rot // 2
    t = np.asarray(table, np.float64)[np.asarray(pos)]
    c, s = t[:, None, :h], t[:, None, h:] * (-1.0 if inverse else 1.0)
    if layout == "half":
        ia, ib = np.arange(h), np.arange(h) + h
    else:
        ia, ib = 2 * np.arange(h), 2 * np.arange(h) + 1
    a, b = x[..., ia].copy(), x[..., ib].copy()
    x[..., ia] = a * c - b * s
    x[..., ib] = b * c + a * s
    return x


def append(x, cache, scale, tbl, ctx, q_len, kind):
    """x [B * q_len, H, D] fp32 into cache [P, page, H, D] / scale [P, H], in place."""
    page = cache.shape[1]
    inv = inv_qmax(kind)
    for b in range(len(ctx)):
        base = int(ctx[b]) - q_len
        for col in range(base // page, (int(ctx[b]) - 1) // page + 1):
            p = tbl[b, col]
            lo, hi = max(base, col * page), min(int(ctx[b]), (col + 1) * page)
            rows = np.asarray(x[b * q_len + lo - base: b * q_len + hi - base], F)
            fin = np.where(np.isfinite(rows), np.abs(rows), F(0))
            need = np.maximum(fin.max(axis=(0, 2)), FLOOR) * inv
            fresh = lo == col * page
            new = need if fresh else np.maximum(scale[p], need)
            for h in range(cache.shape[2]):
                if not fresh and new[h] > scale[p, h]:
                    r = F(scale[p, h]) / F(new[h])
                    cache[p, : lo - col * page, h] = store(cache[p, : lo - col * page, h] * r, kind)
            rs = F(1.0) / new.astype(F)
            with np.errstate(invalid="ignore", over="ignore"):
                y = rows * rs[None, :, None]
            cache[p, lo - col * page: hi - col * page] = store(np.nan_to_num(y, nan=0.0, posinf=1e30, neginf=-1e30), kind)
            scale[p] = new


def compact(cache, scale, tbl, ctx, q_len, accept, n_accept, kind):
    """cache [P, page, H, D], scale [P, H] in place; returns the new lengths."""
    page = cache.shape[1]
    inv = inv_qmax(kind)
    for b in range(len(ctx)):
        base, n = int(ctx[b]) - q_len, int(n_accept[b])
        src = [divmod(base + int(a), page) for a in accept[b][:n]]
        for col in sorted({(base + j) // page for j in range(n)}):
            p = tbl[b, col]
            js = [j for j in range(n) if (base + j) // page == col]
            rows = np.stack([cache[tbl[b, src[j][0]], src[j][1]] for j in js])       # [n, H, D]
            frm = np.stack([scale[tbl[b, src[j][0]]] for j in js])                   # [n, H]
            need = (np.abs(rows).max(-1) * inv) * frm
            other = np.array([src[j][0] != col for j in js])
            need = np.where(other[:, None], need, F(0)).max(0)
            new = np.maximum(scale[p], need).astype(F)
            first = (base + js[0]) % page
            for h in range(cache.shape[2]):
                if new[h] > scale[p, h]:
                    cache[p, :first, h] = store(cache[p, :first, h] * (F(scale[p, h]) / new[h]), kind)
                for i in range(len(js)):
                    r = F(frm[i, h]) / new[h]
                    cache[p, first + i, h] = rows[i, h] if r == 1 else store(rows[i, h] * r, kind)
            scale[p] = new
    return np.asarray(ctx) - q_len + np.asarray(n_accept)


def attention(q, kc, vc, ks, vs, tbl, ctx, tree=None, sm_scale=None):
    """q [B, Q, H, D] -> (out, sum p |v| / l, max score error bound's sum |q||k| sm_scale), float64."""
    q = np.asarray(q, np.float64)
    B, Q, H, D = q.shape
    page, KV = kc.shape[1], kc.shape[2]
    G = H // KV
    sm = D ** -0.5 if sm_scale is None else sm_scale
    out, mag, size = np.zeros_like(q), np.zeros_like(q), np.zeros((B, Q, H))
    for b in range(B):
        n = int(ctx[b])
        if n <= 0:
            continue
        p = tbl[b, : -(-n // page)]
        k = (kc[p].astype(np.float64) * ks[p].astype(np.float64)[:, None, :, None]).reshape(-1, KV, D)[:n]
        v = (vc[p].astype(np.float64) * vs[p].astype(np.float64)[:, None, :, None]).reshape(-1, KV, D)[:n]
        t = np.arange(n)
        for i in range(Q):
            j = t - (n - Q)
            if tree is None:
                see = j <= i
            else:
                word = int(tree[b, i]) & ((1 << 64) - 1)
                see = np.array([x < 0 or (word >> int(x)) & 1 == 1 for x in j])
            if not see.any():
                continue
            for h in range(H):
                x = k[see, h // G] @ q[b, i, h] * sm
                w = np.exp(x - x.max())
                w /= w.sum()
                out[b, i, h] = w @ v[see, h // G]
                mag[b, i, h] = w @ np.abs(v[see, h // G])
                size[b, i, h] = (np.abs(k[see, h // G]) @ np.abs(q[b, i, h])).max() * sm
    return out, mag, size


class Pool:
    """The page pool, one step at a time."""

    def __init__(self, ref, tbl, held):
        self.ref, self.tbl, self.held = (np.array(x) for x in (ref, tbl, held))

    def _free(self):
        return [int(p) for p in np.nonzero(self.ref == 0)[0]]

    def release(self, drop):
        for r in np.nonzero(drop)[0]:
            for c in range(self.held[r]):
                self.ref[self.tbl[r, c]] -= 1
            self.tbl[r] = -1
            self.held[r] = 0

    def reserve(self, want, page):
        need = [max(-(-int(w) // page) - int(h), 0) for w, h in zip(want, self.held)]
        free = self._free()
        if sum(need) > len(free):
            return sum(need) - len(free)
        at = 0
        for r, n in enumerate(need):
            for _ in range(n):
                self.tbl[r, self.held[r]] = free[at]
                self.ref[free[at]] = 1
                self.held[r] += 1
                at += 1
        return 0

    def fork(self, parent, length, page):
        """-> (missing, [(from page, to page, filled slots)])"""
        S = len(self.held)
        rows = [r for r in range(S) if 0 <= parent[r] < S and parent[r] != r]
        parts = [r for r in rows if length[parent[r]] % page]
        free = self._free()
        if len(parts) > len(free):
            return len(parts) - len(free), []
        old_tbl, old_held = self.tbl.copy(), self.held.copy()
        copies = []
        for r in rows:
            p, n = int(parent[r]), int(length[parent[r]])
            new = [int(x) for x in old_tbl[p, : n // page]]
            if n % page:
                to = free[len(copies)]
                copies.append((int(old_tbl[p, n // page]), to, n % page))
                new.append(to)
            for x in new:
                self.ref[x] += 1
            for c in range(old_held[r]):
                self.ref[old_tbl[r, c]] -= 1
            self.tbl[r] = -1
            self.tbl[r, : len(new)] = new
            self.held[r] = len(new)
        return 0, copies
