"""Tree-speculative serving over the block-scaled cache: every operator of it, used together.

A scheduler tick of a small server, on random projections in place of a model's:

  pages_reserve            each live row's pages for its tokens and the drafts to come
  per layer:
    kv_append_blocks       the draft tree's K (turned to the nodes' depths) and V into the pages, the
                           queries turned
    paged_attention_blocks verification of the whole tree in one call
  a path of each tree is accepted (here: drawn at random)
  kv_compact_blocks        the accepted nodes' K and V move together, in every layer
  pages_fork               now and then a row is continued twice (a beam): pages shared, the last copied
  pages_release            requests that end give their pages back

Nothing waits for the host between the calls; lengths, tables and counts live on the device.

    python -m specq.tree_serve [--steps 20] [--rows 8] [--layers 4] [--nodes 21] [--check]

--check compares each attention output with a plain one over the dequantised cache and the pool's
counts with its tables, after every tick.
"""
from __future__ import annotations

import argparse
import json
import random
import time

import torch

from . import _lib, blocks


class BlockCache:
    """The tensors of a block-scaled cache of several layers and of its page pool."""

    def __init__(self, layers, n_pages, page, kv_heads, head_dim, rows, max_len, dtype=torch.int8, device="cuda"):
        self.page, self.rows = page, rows
        shape = (layers, n_pages, page, kv_heads, head_dim)
        self.kc = torch.zeros(shape, dtype=torch.uint8, device=device).view(dtype)
        self.vc = torch.zeros(shape, dtype=torch.uint8, device=device).view(dtype)
        self.ks = torch.ones((layers, n_pages, kv_heads), device=device)
        self.vs = torch.ones((layers, n_pages, kv_heads), device=device)
        i32 = dict(dtype=torch.int32, device=device)
        self.ref = torch.zeros(n_pages, **i32)
        self.tbl = torch.full((rows, -(-max_len // page)), -1, **i32)
        self.held = torch.zeros(rows, **i32)
        self.ctx = torch.zeros(rows, **i32)     # tokens of each row

    def layer(self, i):
        return self.kc[i], self.vc[i], self.ks[i], self.vs[i]

    def pool(self):
        return self.ref, self.tbl, self.held


def draw_tree(rng, nodes):
    """Parents, depths, ancestor bit sets and one root-to-leaf path of a random draft tree whose nodes
    stand in the order of their depth."""
    parent, depth, mask = [-1], [0], [1]
    for j in range(1, nodes):
        p = rng.randrange(max(0, j - 4), j)
        parent.append(p)
        depth.append(depth[p] + 1)
        mask.append(mask[p] | 1 << j)
    path, j = [], rng.randrange(nodes)
    while j >= 0:
        path.append(j)
        j = parent[j]
    return depth, mask, path[::-1]


class Server:
    def __init__(self, rows=8, layers=4, nodes=21, heads=32, kv_heads=8, head_dim=128, page=16, max_len=2048,
                 dtype=torch.int8, seed=0, device="cuda"):
        self.H, self.KV, self.D, self.nodes, self.layers, self.max_len = heads, kv_heads, head_dim, nodes, layers, max_len
        cols = -(-max_len // page)
        self.cache = BlockCache(layers, rows * cols, page, kv_heads, head_dim, rows, max_len, dtype, device)
        self.table = blocks.rope_table(max_len, head_dim, base=500000.0, device=device,
                                       scaling={"type": "llama3", "factor": 8.0, "original": 8192})
        self.rng = random.Random(seed)
        self.gen = torch.Generator(device=device).manual_seed(seed)
        self.device = device
        self.len = [0] * rows                   # the host's copy, for the choices that it makes

    def _i32(self, x):
        return torch.tensor(x, dtype=torch.int32, device=self.device)

    def admit(self, row, prompt):
        """A prompt into an empty row: reserve its pages and append its tokens, layer by layer."""
        c = self.cache
        want = [0] * c.rows
        want[row] = prompt
        short = blocks.pages_reserve(*c.pool(), self._i32(want), c.page)
        ctx = self._i32([prompt])
        for i in range(self.layers):
            k, v = (torch.randn(prompt, self.KV, self.D, generator=self.gen, device=self.device).half() for _ in range(2))
            blocks.kv_append_blocks(k, v, *c.layer(i), c.tbl[row:row + 1], ctx, prompt, table=self.table)
        c.ctx[row] = prompt
        self.len[row] = prompt
        return short

    def tick(self, check=False):
        """One verification step of every row -> accepted tokens of each."""
        c, Q, B = self.cache, self.nodes, self.cache.rows
        trees = [draw_tree(self.rng, Q) for _ in range(B)]
        depth = self._i32([d for t in trees for d in t[0]])
        tree = torch.tensor([[m - (1 << 64) if m >> 63 else m for m in t[1]] for t in trees], dtype=torch.int64,
                            device=self.device)
        accept = self._i32([t[2] + [0] * (Q - len(t[2])) for t in trees])
        n_accept = self._i32([len(t[2]) for t in trees])
        with_drafts = c.ctx + Q
        pos = (c.ctx[:, None] + depth.view(B, Q)).flatten()
        short = blocks.pages_reserve(*c.pool(), with_drafts, c.page)
        worst = 0.0
        for i in range(self.layers):
            qkv = torch.randn(B * Q, (self.H + 2 * self.KV) * self.D, generator=self.gen, device=self.device).half()
            q, k, v = (x.unflatten(1, (-1, self.D)) for x in
                       qkv.split([self.H * self.D, self.KV * self.D, self.KV * self.D], 1))
            q = blocks.kv_append_blocks(k, v, *c.layer(i), c.tbl, with_drafts, Q, q=q, table=self.table, pos=pos)
            out = blocks.paged_attention_blocks(q, *c.layer(i), c.tbl, with_drafts, q_len=Q, tree=tree)
            if check:
                worst = max(worst, self._attention_error(out, q, i, with_drafts, tree))
        c.ctx = blocks.kv_compact_blocks(c.kc, c.vc, c.ks, c.vs, c.tbl, with_drafts, Q, accept, n_accept)
        for b, t in enumerate(trees):
            self.len[b] += len(t[2])
        return [len(t[2]) for t in trees], short, worst

    def fork(self, parent):
        """Row b continues row parent[b] (-1: itself)."""
        c = self.cache
        short = blocks.pages_fork(c.kc, c.vc, c.ks, c.vs, *c.pool(), self._i32(parent), c.ctx)
        src = torch.tensor([b if p < 0 else p for b, p in enumerate(parent)], device=self.device)
        c.ctx = c.ctx[src]
        self.len = [self.len[b if p < 0 else p] for b, p in enumerate(parent)]
        return short

    def retire(self, rows):
        c = self.cache
        drop = torch.zeros(c.rows, dtype=torch.bool, device=self.device)
        drop[torch.tensor(rows, device=self.device)] = True
        blocks.pages_release(*c.pool(), drop)
        c.ctx = torch.where(drop, torch.zeros_like(c.ctx), c.ctx)
        for b in rows:
            self.len[b] = 0

    # ---- checks -------------------------------------------------------------------------------
    def _attention_error(self, out, q, layer, ctx, tree):
        """Largest |difference| from plain attention in fp32 over the dequantised cache."""
        kc, vc, ks, vs = self.cache.layer(layer)
        Q, G, worst = self.nodes, self.H // self.KV, 0.0
        for b, n in enumerate(ctx.tolist()):
            p = self.cache.tbl[b, : -(-n // self.cache.page)].long()
            k = (kc[p].float() * ks[p][:, None, :, None]).flatten(0, 1)[:n].repeat_interleave(G, 1)
            v = (vc[p].float() * vs[p][:, None, :, None]).flatten(0, 1)[:n].repeat_interleave(G, 1)
            j = torch.arange(n, device=self.device) - (n - Q)
            see = (j[None] < 0) | (((tree[b][:, None] >> j.clamp(min=0)[None]) & 1) == 1)
            x = torch.einsum("qhd,thd->hqt", q[b * Q: (b + 1) * Q].float(), k) * self.D ** -0.5
            ref = torch.einsum("hqt,thd->qhd", torch.softmax(x.masked_fill(~see, -torch.inf), -1), v)
            worst = max(worst, (out[b * Q: (b + 1) * Q].float() - ref).abs().max().item())
        return worst

    def check_pool(self):
        """Every page's count is the number of rows that hold it, and rows hold pages for their tokens."""
        c = self.cache
        count = torch.zeros(c.ref.shape[0] + 1, dtype=torch.int64, device=self.device)
        held = torch.arange(c.tbl.shape[1], device=self.device) < c.held[:, None]
        count.index_add_(0, torch.where(held, c.tbl, torch.full_like(c.tbl, -1)).flatten().long() % count.shape[0],
                         held.flatten().long())
        assert torch.equal(count[:-1], c.ref.long()), "the pool's counts and tables differ"
        assert bool((c.held * c.page >= c.ctx).all()) and c.ctx.tolist() == self.len, "rows without pages for their tokens"


def run(steps=20, rows=8, layers=4, nodes=21, seed=0, check=False, dtype=torch.int8):
    s = Server(rows=rows, layers=layers, nodes=nodes, seed=seed, dtype=dtype)
    _lib.get_status(clear=True)
    shorts = [s.admit(b, s.rng.randint(1, 600)) for b in range(rows)]
    accepted, worst, forks, ended = 0, 0.0, 0, 0
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    for step in range(steps):
        got, short, err = s.tick(check)
        accepted += sum(got)
        worst = max(worst, err)
        shorts.append(short)
        if step % 5 == 3:                       # the first row is continued in place of the last
            shorts.append(s.fork([0 if b == rows - 1 else -1 for b in range(rows)]))
            forks += 1
        full = [b for b in range(rows) if s.len[b] + 2 * nodes > s.max_len]
        if step % 7 == 6 and not full:
            full = [s.rng.randrange(rows)]
        if full:
            s.retire(full)
            ended += len(full)
            shorts += [s.admit(b, s.rng.randint(1, 600)) for b in full]
        if check:
            s.check_pool()
    torch.cuda.synchronize()
    missing = max(int(x.item()) for x in shorts)
    status = _lib.get_status(clear=True)
    return {"steps": steps, "rows": rows, "layers": layers, "nodes": nodes, "cache": str(dtype)[6:],
            "accepted_tokens": accepted, "forks": forks, "ended": ended,
            "ms_per_step": (time.perf_counter() - t0) / steps * 1e3,
            "missing_pages": missing, "status": status, "max_abs_error": worst if check else None}


def main():
    ap = argparse.ArgumentParser(description="tree-speculative serving over the block-scaled cache")
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--rows", type=int, default=8)
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--nodes", type=int, default=21)
    ap.add_argument("--seed", type=int, default=0)
    ap.add_argument("--fp8", action="store_true", help="an e4m3 cache (default int8)")
    ap.add_argument("--check", action="store_true")
    a = ap.parse_args()
    print(json.dumps(run(a.steps, a.rows, a.layers, a.nodes, a.seed, a.check,
                         torch.float8_e4m3fn if a.fp8 else torch.int8)))


if __name__ == "__main__":
    main()
