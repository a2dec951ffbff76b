"""Beam search over a bounded block-scaled cache: the operators of heads, beams, eviction and pages together.

On random projections and logits in place of a model's, for requests of several beams each:

  a prompt (the request's first beam)
    per layer: qk_norm_rope, kv_append_blocks, attention_mass_blocks of its last tokens
    kv_evict_blocks        the prompt cut down to a budget, in all layers
    pages_release          the pages past the budget go back to the pool
    pages_fork             the other beams continue the first, sharing its pages
  a step of every beam
    pages_reserve; per layer: qk_norm_rope, kv_append_blocks, paged_attention_blocks
    beam_select            the best continuations of each request
    pages_fork             the cache follows the beams
    beam_reorder           so do token histories, lengths and flags

Nothing waits for the host between the calls; scores, parents, lengths and tables live on the device.

    python -m specq.beam_serve [--steps 20] [--requests 4] [--beams 4] [--layers 2] [--keep 96] [--check]

--check compares each attention output with a plain one over the dequantised cache, the pool's counts with its tables, and
the histories with a replay of the parents and tokens on the host.
"""
from __future__ import annotations

import argparse
import json
import random
import time

import torch

from . import _lib, beams, blocks, heads
from .tree_serve import BlockCache

EOS = 1


class BeamServer:
    def __init__(self, requests=4, beams=4, layers=2, keep=96, heads=32, kv_heads=8, head_dim=128, page=16, max_len=1024, vocab=5003,
                 dtype=torch.int8, seed=0, device="cuda"):
        self.B, self.K, self.layers, self.keep, self.vocab = requests, beams, layers, keep, vocab
        self.H, self.KV, self.D, self.max_len = heads, kv_heads, head_dim, max_len
        rows, cols = requests * beams, -(-max_len // page)
        self.cache = BlockCache(layers, rows * cols, page, kv_heads, head_dim, rows, max_len, dtype, device)
        self.mass = torch.zeros(layers, rows, kv_heads, cols * page, device=device)
        self.table = blocks.rope_table(4 * max_len, head_dim, device=device)
        self.rng = random.Random(seed)
        self.gen = torch.Generator(device=device).manual_seed(seed)
        self.device = device
        self.norm = [(self._randn(head_dim) * 0.1 + 1).half() for _ in range(2 * layers)]
        self.scores = torch.full((requests, beams), -torch.inf, device=device)
        self.history = torch.zeros(rows, max_len, dtype=torch.int32, device=device)
        self.new = torch.zeros(rows, dtype=torch.int32, device=device)     # tokens written after the prompt
        self.pos = torch.zeros(rows, dtype=torch.int32, device=device)     # true positions, whatever is kept of them
        self.done = torch.zeros(rows, dtype=torch.bool, device=device)

    def _randn(self, *shape):
        return torch.randn(*shape, generator=self.gen, device=self.device)

    def _i32(self, x):
        return torch.tensor(x, dtype=torch.int32, device=self.device)

    def _heads(self, layer, tokens, pos):
        """A projection's rows: q and k normalised and turned, v as it is."""
        qkv = self._randn(tokens, (self.H + 2 * self.KV) * self.D).half()
        q, k, v = (x.unflatten(1, (-1, self.D)) for x in
                   qkv.split([self.H * self.D, self.KV * self.D, self.KV * self.D], 1))
        q, k = heads.qk_norm_rope(q, k, self.norm[2 * layer], self.norm[2 * layer + 1], pos, self.table, q_out=q, k_out=k)
        return q, k, v

    def admit(self, request, prompt, window=16):
        """A prompt into the first beam of an empty request; the other beams continue it."""
        c, row = self.cache, request * self.K
        rows = c.rows
        want = [0] * rows
        want[row] = prompt
        shorts = [blocks.pages_reserve(*c.pool(), self._i32(want), c.page)]
        tbl, ctx, pos = c.tbl[row:row + 1], self._i32([prompt]), torch.arange(prompt, dtype=torch.int32, device=self.device)
        mass = self.mass[:, row:row + 1]
        mass.zero_()
        w = min(window, prompt)
        for i in range(self.layers):
            q, k, v = self._heads(i, prompt, pos)
            blocks.kv_append_blocks(k, v, *c.layer(i), tbl, ctx, prompt)
            blocks.attention_mass_blocks(q[prompt - w:][None], c.kc[i], c.ks[i], tbl, ctx, mass[i])
        blocks.kv_evict_blocks(c.kc, c.vc, c.ks, c.vs, tbl, ctx, mass, self.keep, recent=self.keep // 4, ref=c.ref, ctx_out=ctx)
        c.ctx[row:row + 1] = ctx
        first = torch.zeros(rows, dtype=torch.bool, device=self.device)
        first[row] = True
        blocks.pages_release(*c.pool(), first, c.ctx, c.page)
        parent = [-1] * rows
        parent[row + 1: row + self.K] = [row] * (self.K - 1)
        shorts.append(blocks.pages_fork(c.kc, c.vc, c.ks, c.vs, *c.pool(), self._i32(parent), c.ctx))
        mine = slice(row, row + self.K)
        c.ctx[mine] = c.ctx[row].clone()
        self.pos[mine], self.new[mine], self.done[mine] = prompt, 0, False
        self.scores[request] = -torch.inf
        self.scores[request, 0] = 0.0
        return shorts

    def step(self, check=False):
        """One token of every beam -> (pages that were missing, the parents, the tokens, the largest error of attention)."""
        c, worst = self.cache, 0.0
        ctx = c.ctx + 1
        shorts = [blocks.pages_reserve(*c.pool(), ctx, c.page)]
        for i in range(self.layers):
            q, k, v = self._heads(i, c.rows, self.pos)
            blocks.kv_append_blocks(k, v, *c.layer(i), c.tbl, ctx, 1)
            out = blocks.paged_attention_blocks(q, *c.layer(i), c.tbl, ctx, q_len=1)
            if check:
                worst = max(worst, self._attention_error(out, q, i, ctx))
        logits = (self._randn(c.rows, self.vocab) * 3).half()
        self.scores, parent, token = beams.beam_select(logits, self.scores, done=self.done, pad=EOS)
        shorts.append(blocks.pages_fork(c.kc, c.vc, c.ks, c.vs, *c.pool(), parent.view(-1), ctx))
        c.ctx = ctx
        self.pos += 1
        beams.beam_reorder([self.history, self.new, self.pos, c.ctx, self.done], parent)
        self.history.scatter_(1, self.new.long()[:, None], token.view(-1, 1))
        self.new += 1
        self.done |= token.view(-1) == EOS
        return shorts, parent, token, worst

    def _attention_error(self, out, q, layer, ctx):
        kc, vc, ks, vs = self.cache.layer(layer)
        G, worst = self.H // self.KV, 0.0
        for b, n in enumerate(ctx.tolist()):
            p = self.cache.tbl[b, : -(-n // self.cache.page)].long()
            k = (kc[p].float() * ks[p][:, None, :, None]).flatten(0, 1)[:n].repeat_interleave(G, 1)
            v = (vc[p].float() * vs[p][:, None, :, None]).flatten(0, 1)[:n].repeat_interleave(G, 1)
            w = torch.softmax(torch.einsum("hd,thd->ht", q[b].float(), k) * self.D ** -0.5, -1)
            worst = max(worst, (out[b].float() - torch.einsum("ht,thd->hd", w, v)).abs().max().item())
        return worst

    def check_pool(self):
        """Every page's count is the number of rows that hold it, and rows hold pages for their tokens."""
        c = self.cache
        count = torch.zeros(c.ref.shape[0], dtype=torch.int64)
        held, tbl = c.held.tolist(), c.tbl.cpu()
        for r, n in enumerate(held):
            for p in tbl[r, :n].tolist():
                count[p] += 1
        assert torch.equal(count, c.ref.cpu().long()), "the pool's counts and tables differ"
        assert bool((c.held * c.page >= c.ctx).all()), "rows without pages for their tokens"


def run(steps=20, requests=4, beams=4, layers=2, keep=96, seed=0, check=False, dtype=torch.int8):
    s = BeamServer(requests, beams, layers, keep, seed=seed, dtype=dtype)
    _lib.get_status(clear=True)
    prompts = [s.rng.randint(1, 600) for _ in range(requests)]
    shorts = [x for b, n in enumerate(prompts) for x in s.admit(b, n)]
    replay, worst = [[] for _ in range(s.cache.rows)], 0.0
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    for _ in range(steps):
        missing, parent, token, err = s.step(check)
        shorts += missing
        worst = max(worst, err)
        if check:
            s.check_pool()
            replay = [replay[p] + [t] for p, t in zip(parent.view(-1).tolist(), token.view(-1).tolist())]
            assert [h[: len(replay[0])] for h in s.history.tolist()] == replay, "the histories do not follow the beams"
    torch.cuda.synchronize()
    ms = (time.perf_counter() - t0) / steps * 1e3
    return {"steps": steps, "requests": requests, "beams": beams, "layers": layers, "keep": keep, "cache": str(dtype)[6:],
            "kept": [int(x) for x in s.cache.ctx.view(requests, beams)[:, 0].tolist()], "prompts": prompts, "ms_per_step": ms,
            "finished": int(s.done.sum()), "missing_pages": max(int(x.item()) for x in shorts),
            "status": _lib.get_status(clear=True), "max_abs_error": worst if check else None}


def main():
    ap = argparse.ArgumentParser(description="beam search over a bounded block-scaled cache")
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--requests", type=int, default=4)
    ap.add_argument("--beams", type=int, default=4)
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--keep", type=int, default=96, help="tokens of a prompt that stay in the cache")
    ap.add_argument("--seed", type=int, default=0)
    ap.add_argument("--fp8", action="store_true", help="an e4m3 cache (default int8)")
    ap.add_argument("--check", action="store_true")
    a = ap.parse_args()
    print(json.dumps(run(a.steps, a.requests, a.beams, a.layers, a.keep, a.seed, a.check,
                         torch.float8_e4m3fn if a.fp8 else torch.int8)))


if __name__ == "__main__":
    main()
