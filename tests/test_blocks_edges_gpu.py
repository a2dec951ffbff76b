"""The block-scaled cache's operators at the edges of their inputs: tiny, zero and outlying queries, page numbers
outside the cache, rows that a call does not reach, gradients of the rotation, kernels on each other's heels.

Attention is compared with the 64-bit oracle under the bound derived in test_blocks_gpu.py; a page number
outside the cache takes its tokens out of the window, so there the oracle gets the table without that page."""
import numpy as np
import pytest
import torch

from oracle import block_oracle as BO
from test_blocks_gpu import UNIT, _attend_check, _attend_inputs, _np, _random_tree, _status

pytestmark = pytest.mark.gpu


# ---- page numbers outside the cache -------------------------------------------------------------------
def _without_pages(q, kc, vc, ks, vs, tbl, cl, bad):
    """The 64-bit result where the pages `bad` (lists of columns, one a sequence; whole pages before the
    drafts) are not there, and the bound's parts."""
    page, parts = kc.shape[1], []
    for b, cols in enumerate(bad):
        row = np.delete(tbl[b].cpu().numpy(), cols)[None]
        parts.append(BO.attention(_np(q[b: b + 1]), _np(kc), _np(vc), _np(ks), _np(vs), row, [int(cl[b]) - page * len(cols)]))
    return [np.concatenate(p) for p in zip(*parts)]


def _attend_with_bad_pages(args, bad):
    import specq
    from specq import _lib
    q, kc, vc, ks, vs, tbl, cl = args
    ref, mag, size = _without_pages(q, kc, vc, ks, vs, tbl, cl, bad)
    broken = tbl.clone()
    for b, cols in enumerate(bad):
        for i, c in enumerate(cols):
            broken[b, c] = (-1, kc.shape[0], 1 << 30, -(1 << 31))[(b + i) % 4]
    got = specq.paged_attention_blocks(q, kc, vc, ks, vs, broken, cl)
    assert _status() == _lib.SPECQ_STATUS_BAD_INDEX
    assert torch.isfinite(got).all()
    lim = UNIT[q.dtype] * np.abs(ref) + (2.0 ** -11 + 2 * (132 * 2.0 ** -24 * size[..., None] + 2.0 ** -14)) * mag + 2.0 ** -24
    err = np.abs(_np(got) - ref)
    assert (err <= lim).all(), (err.max(), (err / lim).max())


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("Q,KV,G,D", [(1, 2, 4, 128), (4, 1, 8, 64), (3, 2, 1, 128)])
def test_attention_steps_over_a_bad_page_of_eight(cuda, kind, dtype, Q, KV, G, D):
    """At page 8 two pages share 16 tokens of a tile: a bad even or odd one takes no weight from the other."""
    args = _attend_inputs(31, 5, Q, KV, G, D, 8, kind, dtype, [40, 47, 90, 300, 24 + Q])
    for bad in ([[2], [3], [0, 5], [4, 7, 10, 33], []], [[0, 2], [1], [1, 2], [16, 17, 18], [2]]):
        _attend_with_bad_pages(args, bad)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("Q,KV,G,D,page", [(1, 2, 4, 128, 16), (9, 1, 4, 64, 32), (2, 2, 4, 128, 128), (3, 1, 8, 64, 8)])
def test_attention_reads_nothing_for_a_bad_page(cuda, dtype, Q, KV, G, D, page):
    """Page 0 belongs to no sequence and holds NaN bytes: a bad page number does not bring them in.  A sequence
    without one good page sees nothing."""
    ctx = [3 * page + 7 + Q, 300 + Q, page + Q]
    q, kc, vc, ks, vs, tbl, cl = _attend_inputs(41, 3, Q, KV, G, D, page, "e4m3", dtype, ctx)
    gen = torch.Generator().manual_seed(7)
    tbl = (torch.randperm(kc.shape[0] - 1, generator=gen)[: tbl.numel()] + 1).to(torch.int32).view(tbl.shape).cuda()
    for c in (kc, vc):
        c[0].view(torch.uint8).fill_(0x7F)
    ks[0], vs[0] = float("nan"), float("inf")
    _attend_with_bad_pages((q, kc, vc, ks, vs, tbl, cl), [[1], [0, 2 if page < 64 else 1], [0]])
    import specq
    none = torch.full_like(tbl, kc.shape[0])
    got = specq.paged_attention_blocks(q, kc, vc, ks, vs, none, cl)
    assert (got == 0).all()
    assert _status() != 0


# ---- queries of any size ----------------------------------------------------------------------------
@pytest.mark.parametrize("page", [8, 16, 32])
@pytest.mark.parametrize("Q,KV,G,D", [(1, 2, 4, 128), (5, 1, 4, 64), (9, 2, 4, 128)])
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attention_of_zero_queries(cuda, dtype, kind, Q, KV, G, D, page):
    """Zero queries see every token alike: the mean of V, and 0 where there is no token; in every sequence and
    in one beside others."""
    ctx = [37, 0, 1, 64, 200, Q]
    q, kc, vc, ks, vs, tbl, cl = _attend_inputs(Q + page, len(ctx), Q, KV, G, D, page, kind, dtype, ctx)
    tree = _random_tree(torch.Generator().manual_seed(Q), len(ctx), Q).cuda()
    zero = torch.zeros_like(q)
    for t in (None, tree):
        got = _attend_check(zero, kc, vc, ks, vs, tbl, cl, tree=t)
        assert (got[1] == 0).all()
    q[4] = 0
    _attend_check(q, kc, vc, ks, vs, tbl, cl)
    assert _status() == 0


@pytest.mark.parametrize("page", [8, 16, 64])
@pytest.mark.parametrize("Q,KV,G,D", [(1, 2, 4, 128), (9, 1, 4, 64)])
@pytest.mark.parametrize("power", [-100, -40, -28, 60, 110])
def test_attention_of_scaled_bf16_queries(cuda, power, Q, KV, G, D, page):
    """bf16 queries times a power of two, under sm_scale times its reciprocal, give the same bits (every product
    and sum is scaled by powers of two alone); tiny ones under the same sm_scale, the mean of V."""
    import specq
    q, kc, vc, ks, vs, tbl, cl = _attend_inputs(Q, 5, Q, KV, G, D, page, "int8", torch.bfloat16, [37, 1, 150, 64, Q])
    ref = _attend_check(q, kc, vc, ks, vs, tbl, cl)
    small = (q.float() * 2.0 ** power).bfloat16()
    got = specq.paged_attention_blocks(small, kc, vc, ks, vs, tbl, cl, sm_scale=D ** -0.5 * 2.0 ** -power)
    assert torch.equal(got, ref)
    if power < 0:
        _attend_check(small, kc, vc, ks, vs, tbl, cl)
    assert _status() == 0


@pytest.mark.parametrize("Q,KV,G,D", [(1, 2, 8, 64), (5, 2, 4, 64), (9, 1, 4, 128)])
@pytest.mark.parametrize("size", [2.0 ** 12, 2.0 ** 14, 2.0 ** 16, 2.0 ** 20, 2.0 ** 40, 1e30])
def test_attention_of_an_outlying_row_leaves_the_others_exact(cuda, size, Q, KV, G, D):
    """One finite, very large bf16 query row costs the others nothing: they keep the bound."""
    q, kc, vc, ks, vs, tbl, cl = _attend_inputs(21, 3, Q, KV, G, D, 16, "e4m3", torch.bfloat16, [400, 33, 90])
    import specq
    big = q.clone()
    big[0, Q // 2, 1] *= size
    big[1, 0, 2, 5] = -size
    got = specq.paged_attention_blocks(big, kc, vc, ks, vs, tbl, cl)
    assert torch.isfinite(got).all()
    keep = torch.ones(q.shape[:3], dtype=torch.bool)
    keep[0, Q // 2, 1] = keep[1, 0, 2] = False
    keep = keep.cuda()
    ref = specq.paged_attention_blocks(q, kc, vc, ks, vs, tbl, cl)
    _attend_check(q, kc, vc, ks, vs, tbl, cl, out=torch.where(keep[..., None], got, ref))
    assert _status() == 0


# ---- kernels on each other's heels -----------------------------------------------------------------------
def test_chained_calls_see_each_others_writes(cuda):
    """Reserve, append, attention and compaction in a stream, each reading what the one before it wrote (tables,
    scales, numbers, lengths, parts), give the bits that they give with the GPU idle between them."""
    import specq
    B, Q, KV, G, D, page, C = 6, 9, 2, 4, 128, 16, 96
    gen = torch.Generator(device="cuda").manual_seed(0)
    table = specq.rope_table(C * page, D, device="cuda")
    steps = 12
    rows = [torch.randn(B * Q, (KV * G + 2 * KV), D, generator=gen, device="cuda").mul(1 + 3 * (i % 4)).half() for i in range(steps)]
    prompt = torch.randn(B * 700, 2 * KV, D, generator=gen, device="cuda").half()
    accept = [torch.stack([torch.randperm(Q, generator=gen, device="cuda")[:4].sort().values for _ in range(B)]).int() for _ in range(steps)]
    four = torch.full((B,), 4, dtype=torch.int32, device="cuda")
    start = torch.full((B,), 700, dtype=torch.int32, device="cuda")

    def run(idle):
        wait = torch.cuda.synchronize if idle else (lambda: None)
        kc, vc = (torch.zeros(B * C, page, KV, D, dtype=torch.int8, device="cuda") for _ in range(2))
        ks, vs = (torch.ones(B * C, KV, device="cuda") for _ in range(2))
        ref = torch.zeros(B * C, dtype=torch.int32, device="cuda")
        tbl = torch.full((B, C), -1, dtype=torch.int32, device="cuda")
        held = torch.zeros(B, dtype=torch.int32, device="cuda")
        lens = [start] + [torch.empty_like(start) for _ in range(steps)]
        drafts = [torch.empty_like(start) for _ in range(steps)]
        outs = []
        specq.pages_reserve(ref, tbl, held, start, page)
        specq.kv_append_blocks(prompt[:, :KV], prompt[:, KV:], kc, vc, ks, vs, tbl, start, 700, table=table)
        wait()
        for i in range(steps):
            torch.add(lens[i], Q, out=drafts[i])
            wait()
            specq.pages_reserve(ref, tbl, held, drafts[i], page)
            wait()
            q, k, v = rows[i].split([KV * G, KV, KV], 1)
            q = specq.kv_append_blocks(k, v, kc, vc, ks, vs, tbl, drafts[i], Q, q=q, table=table)
            wait()
            outs.append(specq.paged_attention_blocks(q, kc, vc, ks, vs, tbl, drafts[i], q_len=Q))
            wait()
            specq.kv_compact_blocks(kc, vc, ks, vs, tbl, drafts[i], Q, accept[i], four, ctx_out=lens[i + 1])
            wait()
            outs.append(specq.paged_attention_blocks(q, kc, vc, ks, vs, tbl, lens[i + 1], q_len=Q))
            wait()
        torch.cuda.synchronize()
        return outs + lens + [kc, vc, ks, vs, tbl, held, ref]
    want = run(True)
    for _ in range(4):
        assert all(torch.equal(a, b) for a, b in zip(run(False), want))
    assert _status() == 0


# ---- rows that a call does not reach ----------------------------------------------------------------------
def test_new_outputs_are_zero_where_a_call_does_not_reach(cuda):
    """Queries turned by an append of fewer sequences, or under a plan, and rows past a plan's in rope."""
    import specq
    gen = torch.Generator(device="cuda").manual_seed(1)
    B, Q, KV, H, D, page = 4, 9, 2, 8, 128, 16
    k, v = (torch.randn(B * Q, KV, D, generator=gen, device="cuda").half() for _ in range(2))
    q = torch.randn(B * Q + 3, H, D, generator=gen, device="cuda").half()
    kc, vc = (torch.zeros(B, page, KV, D, dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.ones(B, KV, device="cuda") for _ in range(2))
    tbl = torch.arange(B, dtype=torch.int32, device="cuda")[:, None]
    ctx = torch.full((B,), Q, dtype=torch.int32, device="cuda")
    table = specq.rope_table(64, D, device="cuda")
    pos = torch.arange(B * Q + 3, dtype=torch.int32, device="cuda") % 64

    def poison():
        junk = [torch.full((B * Q + 3, H, D), float("nan"), dtype=torch.half, device="cuda") for _ in range(4)]
        torch.cuda.synchronize()
        del junk
    for kw, n in ((dict(n_seqs=2), 2 * Q), (dict(), B * Q), (dict(n_seqs=0), 0),
                  (dict(plan=torch.tensor([3, 5], dtype=torch.int32, device="cuda")), 15)):
        poison()
        out = specq.kv_append_blocks(k, v, kc, vc, ks, vs, tbl, ctx, Q, q=q, table=table, **kw)
        assert out.shape == q.shape and (out[n:] == 0).all() and torch.isfinite(out).all()
    for n in (0, 5, B * Q + 3):
        poison()
        out = specq.rope(q, pos, table, plan=torch.tensor([n], dtype=torch.int32, device="cuda"))
        assert (out[n:] == 0).all() and torch.equal(out[:n], specq.rope(q, pos, table)[:n])
    assert _status() == 0


# ---- the rotation's gradient ---------------------------------------------------------------------------------
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rope_carries_gradients(cuda, layout, dtype):
    """The gradient of a rotation is the inverse rotation of the output's gradient, and that of the inverse the
    rotation; under a plan the rows past it have none.  Against difference quotients in fp32: a sum of n products
    of size about 1 is off by n 2^-23 at most, the quotient by 2^-23 |f| / h more."""
    import specq
    gen = torch.Generator(device="cuda").manual_seed(2)
    T, H, D, rot = 9, 3, 64, 32
    table = specq.rope_table(64, rot, device="cuda")
    pos = torch.arange(T, dtype=torch.int32, device="cuda") * 5
    x, g, d = (torch.randn(T, H, D, generator=gen, device="cuda").to(dtype) for _ in range(3))
    plan = torch.tensor([4], dtype=torch.int32, device="cuda")
    for inverse in (False, True):
        for kw in (dict(), dict(plan=plan)):
            leaf = x.clone().requires_grad_()
            y = specq.rope(leaf, pos, table, layout=layout, inverse=inverse, **kw)
            assert torch.equal(y.detach(), specq.rope(x, pos, table, layout=layout, inverse=inverse, **kw))
            y.backward(g)
            assert torch.equal(leaf.grad, specq.rope(g, pos, table, layout=layout, inverse=not inverse, **kw))
    if dtype == torch.float32:
        leaf = x.clone().requires_grad_()
        specq.rope(leaf, pos, table, layout=layout).backward(g)
        h = 0.25
        f = lambda t: (g.double() * specq.rope(t, pos, table, layout=layout).double()).sum()  # noqa: E731
        diff = (f(x + h * d) - f(x - h * d)) / (2 * h)
        size = (g.abs() * (x.abs() + d.abs())).sum().item()
        assert abs((diff - (leaf.grad.double() * d.double()).sum()).item()) <= 8 * 2.0 ** -23 * size / h + T * H * D * 2.0 ** -23
        # the gradient's own gradient
        leaf, gl = x.clone().requires_grad_(), g.clone().requires_grad_()
        first, = torch.autograd.grad(specq.rope(leaf, pos, table, layout=layout), leaf, gl, create_graph=True)
        second, = torch.autograd.grad(first, gl, d)
        assert torch.equal(second, specq.rope(d, pos, table, layout=layout))
    leaf = x.clone().requires_grad_()
    with torch.no_grad():
        assert not specq.rope(leaf, pos, table, layout=layout).requires_grad
        buf = torch.empty_like(x)
        assert specq.rope(leaf, pos, table, layout=layout, out=buf) is buf
    assert _status() == 0
