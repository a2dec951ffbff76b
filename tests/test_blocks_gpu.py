"""The block-scaled cache's append, attention, compaction and page pool against the oracle.

Append without a turn, compaction and the pool are defined exactly (fp32 with stated roundings,
integers): equality.  With a turn, K differs from the oracle's float64 turn by at most
4 * 2^-24 (|a| + |b|), so a stored number is within half a step of the exact quotient and that.

Attention, for each element: half a unit of the output's type; p rounded to fp16 (2^-11 of
sum p |v| / l); scores accumulated in fp32 over D <= 128 products, and the exponent's argument
rounded in log2 units (|x| < 2^9 here): delta = (128 + 4) 2^-24 max sum |q||k| sm + 2^-14, twice
(numerator and normaliser) of sum p |v| / l."""
import numpy as np
import pytest
import torch

from oracle import block_oracle as BO

pytestmark = pytest.mark.gpu

CACHES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def _np(t):
    return t.detach().float().cpu().numpy()


def _stored(gen, shape, kind):
    x = torch.randn(shape, generator=gen) * (40 if kind == "int8" else 140)
    top = 127 if kind == "int8" else 448
    x = x.clamp(-top, top)
    return (x.round() if kind == "int8" else x).to(CACHES[kind]).cuda()


def _scales(gen, shape, kind):
    return ((torch.rand(shape, generator=gen) * 2 + 1) / (127 if kind == "int8" else 448)).cuda()


def _table(gen, B, C, P):
    return torch.randperm(P, generator=gen)[: B * C].to(torch.int32).view(B, C).cuda()


def _status():
    import specq
    torch.cuda.synchronize()
    return specq.get_status(clear=True)


# ---- append ------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,KV,page,Q", [(128, 2, 16, 1), (128, 8, 16, 9), (64, 3, 8, 5), (64, 1, 32, 33), (128, 1, 64, 7),
                                         (128, 3, 128, 150), (64, 2, 128, 1), (128, 1, 8, 40)])
def test_append_exact(cuda, kind, dtype, D, KV, page, Q):
    import specq
    gen = torch.Generator().manual_seed(D + KV + page + Q)
    ctx = torch.tensor([Q, Q + 1, Q + page - 1, Q + 3 * page, Q + 2 * page + 5], dtype=torch.int32)
    B = len(ctx)
    C = int(ctx.max() - 1) // page + 1
    tbl = _table(gen, B, C, B * C + 2)
    kc, vc = (_stored(gen, (B * C + 2, page, KV, D), kind) for _ in range(2))
    ks, vs = (_scales(gen, (B * C + 2, KV), kind) for _ in range(2))
    rows = torch.randn(B * Q, 2 * KV * D + 8, generator=gen).mul(2).to(dtype).cuda()
    k, v = rows[:, : KV * D].unflatten(1, (KV, D)), rows[:, KV * D: 2 * KV * D].unflatten(1, (KV, D))
    want = []
    for x, c, s in ((k, kc, ks), (v, vc, vs)):
        c, s = _np(c).copy(), _np(s).copy()
        BO.append(_np(x), c, s, tbl.cpu().numpy(), ctx.numpy(), Q, kind)
        want.append((c, s))
    assert specq.kv_append_blocks(k, v, kc, vc, ks, vs, tbl, ctx.cuda(), Q) is None
    for (c, s), gc, gs in zip(want, (kc, vc), (ks, vs)):
        assert np.array_equal(_np(gs), s)
        assert np.array_equal(_np(gc), c)          # the numbers, old tokens and untouched slots included
    assert _status() == 0


def test_append_grows_and_keeps(cuda):
    """Token by token into one page: the scale grows when a larger token comes and never shrinks; the older
    numbers follow it."""
    import specq
    gen = torch.Generator().manual_seed(0)
    for kind in CACHES:
        kc, vc = (_stored(gen, (2, 16, 1, 64), kind) for _ in range(2))
        ks, vs = (_scales(gen, (2, 1), kind) for _ in range(2))
        tbl = torch.tensor([[1]], dtype=torch.int32).cuda()
        rc, rs = _np(kc).copy(), _np(ks).copy()
        for t, size in enumerate((1.0, 0.1, 3.0, 2.0, 50.0, 0.0)):
            x = (torch.rand(1, 1, 64, generator=gen) * 2 - 1).mul(size).half().cuda()
            ctx = torch.tensor([t + 1], dtype=torch.int32).cuda()
            specq.kv_append_blocks(x, x, kc, vc, ks, vs, tbl, ctx, 1)
            BO.append(_np(x), rc, rs, tbl.cpu().numpy(), [t + 1], 1, kind)
            assert np.array_equal(_np(ks), rs) and np.array_equal(_np(kc), rc)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("D,rot", [(128, 128), (64, 32), (128, 48)])
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_append_turns_keys_and_queries(cuda, layout, D, rot, kind):
    import specq
    gen = torch.Generator().manual_seed(rot)
    B, Q, H, KV, page = 3, 21, 6, 2, 16
    C, P = 6, 20
    tbl = _table(gen, B, C, P)
    ctx = torch.tensor([21, 40, 93], dtype=torch.int32).cuda()
    qkv = torch.randn(B * Q, (H + 2 * KV) * D, generator=gen).half().cuda()
    q, k, v = (x.unflatten(1, (-1, D)) for x in qkv.split([H * D, KV * D, KV * D], 1))
    table = specq.rope_table(96, rot, device="cuda")
    for given in (False, True):
        pos = (ctx[:, None] - Q + torch.arange(Q, device="cuda")).flatten().int()
        if given:
            pos = (pos + torch.randint(-5, 1, pos.shape, generator=gen).cuda()).clamp(0, 95).int()
        kc, vc = (_stored(gen, (P, page, KV, D), kind) for _ in range(2))
        ks, vs = (_scales(gen, (P, KV), kind) for _ in range(2))
        qo = specq.kv_append_blocks(k, v, kc, vc, ks, vs, tbl, ctx, Q, q=q, table=table, pos=pos if given else None,
                                    layout=layout)
        assert torch.equal(qo, specq.rope(q, pos, table, layout=layout))
        want = BO.turn(_np(k), _np(table), pos.cpu().numpy(), layout)
        slop = 8 * 2.0 ** -24 * np.abs(_np(k)).max(-1, keepdims=True)
        num, sc = _np(kc), _np(ks)
        for b in range(B):
            for t in range(Q):
                p_ = int(ctx[b]) - Q + t
                pg, slot = int(tbl[b, p_ // page]), p_ % page
                y = want[b * Q + t] / sc[pg][:, None]
                half = 0.5 if kind == "int8" else np.maximum(2.0 ** -4 * np.abs(y), 2.0 ** -10)
                lim = half * (1 + 2.0 ** -20) + (slop[b * Q + t] + 2.0 ** -22 * np.abs(want[b * Q + t])) / sc[pg][:, None]
                assert (np.abs(num[pg, slot] - y) <= lim).all()
        # queries in place
        mine = qkv.clone()
        qi = mine[:, : H * D].unflatten(1, (H, D))
        specq.kv_append_blocks(k, v, kc, vc, ks, vs, tbl, ctx, Q, q=qi, q_out=qi, table=table,
                               pos=pos if given else None, layout=layout)
        assert torch.equal(qi, qo) and torch.equal(mine[:, H * D:], qkv[:, H * D:])
    assert _status() == 0


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_append_nonfinite_and_bad_pages(cuda, kind):
    import specq
    from specq import _lib
    gen = torch.Generator().manual_seed(1)
    kc, vc = (_stored(gen, (4, 16, 2, 64), kind) for _ in range(2))
    ks, vs = (_scales(gen, (4, 2), kind) for _ in range(2))
    x = torch.randn(2, 2, 64, generator=gen).half()
    x[0, 0, 3], x[0, 0, 4], x[1, 1, 5], x[1, 1, 6] = float("nan"), float("inf"), float("-inf"), float("nan")
    x = x.cuda()
    tbl = torch.tensor([[2]], dtype=torch.int32).cuda()
    ctx = torch.tensor([2], dtype=torch.int32).cuda()
    rc, rs = _np(kc).copy(), _np(ks).copy()
    BO.append(_np(x), rc, rs, tbl.cpu().numpy(), [2], 2, kind)
    specq.kv_append_blocks(x, x, kc, vc, ks, vs, tbl, ctx, 2)
    assert _status() == _lib.SPECQ_STATUS_KV_NONFINITE
    assert np.array_equal(_np(kc), rc) and np.array_equal(_np(ks), rs)
    assert np.isfinite(_np(kc)).all()
    # page numbers outside the cache, contexts outside the table: nothing is written, the status says so
    before = kc.clone().view(torch.uint8)
    y = torch.randn(4, 2, 64, generator=gen).half().cuda()
    for pg, n, code in ((9, 2, _lib.SPECQ_STATUS_BAD_INDEX), (-1, 2, _lib.SPECQ_STATUS_BAD_INDEX),
                        (1, 1, _lib.SPECQ_STATUS_PLAN_CLAMPED), (1, 17, _lib.SPECQ_STATUS_PLAN_CLAMPED)):
        specq.kv_append_blocks(y[:2], y[:2], kc, vc, ks, vs, torch.tensor([[pg]], dtype=torch.int32).cuda(),
                               torch.tensor([n], dtype=torch.int32).cuda(), 2)
        assert _status() == code
        assert torch.equal(kc.view(torch.uint8), before)


def test_append_plan(cuda):
    import specq
    gen = torch.Generator().manual_seed(2)
    B, Q, KV, D, H, page = 4, 9, 2, 128, 8, 16
    tbl = _table(gen, B, 4, 16)
    ctx = torch.tensor([9, 30, 41, 64], dtype=torch.int32).cuda()
    table = specq.rope_table(64, D, device="cuda")
    qkv = torch.randn(B * Q, (H + 2 * KV) * D, generator=gen).half().cuda()
    q, k, v = (x.unflatten(1, (-1, D)) for x in qkv.split([H * D, KV * D, KV * D], 1))
    base = [_stored(gen, (16, page, KV, D), "int8") for _ in range(2)] + [_scales(gen, (16, KV), "int8") for _ in range(2)]
    for n, ql in ((4, 9), (2, 5), (3, 1), (0, 9), (4, 0)):
        a, b = [t.clone() for t in base], [t.clone() for t in base]
        qa = specq.kv_append_blocks(k, v, *a, tbl, ctx, ql, q=q, table=table, n_seqs=n)
        plan = torch.tensor([n, ql], dtype=torch.int32).cuda()
        out = torch.full_like(q.contiguous(), 7.0)
        specq.kv_append_blocks(k, v, *b, tbl, ctx, Q, q=q, q_out=out, table=table, plan=plan)
        assert all(torch.equal(s, t) for s, t in zip(a, b))
        assert torch.equal(out[: n * ql], qa[: n * ql]) and (out[n * ql:] == 7.0).all()
    assert _status() == 0


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("shift", [4, 12])
def test_append_rows_of_eight_byte_alignment(cuda, layout, shift):
    """K and V rows that begin off a 16-byte boundary, or whose stride leaves it, are stored as aligned ones are."""
    import specq
    gen = torch.Generator().manual_seed(shift)
    B, Q, KV, D, page = 3, 19, 2, 128, 16
    tbl = _table(gen, B, 4, 14)
    ctx = torch.tensor([19, 33, 60], dtype=torch.int32).cuda()
    table = specq.rope_table(64, 64, device="cuda")
    wide = torch.randn(B * Q, 2 * KV * D + 2 * shift, generator=gen).half().cuda()
    k, v = (wide[:, shift + i * KV * D: shift + (i + 1) * KV * D].unflatten(1, (KV, D)) for i in range(2))
    base = [_stored(gen, (14, page, KV, D), "int8") for _ in range(2)] + [_scales(gen, (14, KV), "int8") for _ in range(2)]
    a, b = [t.clone() for t in base], [t.clone() for t in base]
    specq.kv_append_blocks(k, v, *a, tbl, ctx, Q, table=table, layout=layout)
    specq.kv_append_blocks(k.contiguous(), v.contiguous(), *b, tbl, ctx, Q, table=table, layout=layout)
    assert all(torch.equal(s, t) for s, t in zip(a, b))
    assert _status() == 0


# ---- attention ---------------------------------------------------------------------------------
UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _attend_check(q, kc, vc, ks, vs, tbl, ctx, tree=None, out=None, sm_scale=None):
    import specq
    got = specq.paged_attention_blocks(q, kc, vc, ks, vs, tbl, ctx, tree=tree, sm_scale=sm_scale) if out is None else out
    ref, mag, size = BO.attention(_np(q), _np(kc), _np(vc), _np(ks), _np(vs), tbl.cpu().numpy(), ctx.cpu().numpy(),
                                  None if tree is None else tree.cpu().numpy(), sm_scale)
    lim = UNIT[q.dtype] * np.abs(ref) + (2.0 ** -11 + 2 * (132 * 2.0 ** -24 * size[..., None] + 2.0 ** -14)) * mag + 2.0 ** -24
    err = np.abs(_np(got) - ref)
    assert np.isfinite(_np(got)).all()
    assert (err <= lim).all(), (err.max(), (err / lim).max())
    return got


def _attend_inputs(seed, B, Q, KV, G, D, page, kind, dtype, ctx, spare=3):
    gen = torch.Generator().manual_seed(seed)
    C = max(1, -(-max(max(ctx), 1) // page))
    P = B * C + spare
    return (torch.randn(B, Q, KV * G, D, generator=gen).to(dtype).cuda(), _stored(gen, (P, page, KV, D), kind),
            _stored(gen, (P, page, KV, D), kind), _scales(gen, (P, KV), kind), _scales(gen, (P, KV), kind),
            _table(gen, B, C, P), torch.tensor(ctx, dtype=torch.int32).cuda())


@pytest.mark.parametrize("kind,dtype", [("int8", torch.float16), ("e4m3", torch.bfloat16), ("e4m3", torch.float16),
                                        ("int8", torch.bfloat16)])
@pytest.mark.parametrize("Q,KV,G,D,page", [(1, 2, 4, 128, 16), (1, 1, 1, 64, 8), (9, 2, 4, 128, 16), (3, 2, 8, 64, 32),
                                           (5, 1, 5, 128, 128), (2, 3, 2, 128, 8), (4, 1, 8, 64, 64), (13, 1, 4, 128, 32),
                                           (8, 1, 8, 128, 16), (11, 1, 8, 64, 16), (40, 1, 4, 128, 64), (70, 1, 2, 64, 16)])
def test_attention_matches_oracle(cuda, kind, dtype, Q, KV, G, D, page):
    """Every variant (1 to 12 groups of 8 query rows, several row chunks), lengths from none over one token and
    the edges of pages and tiles to a few hundred, rows that see nothing included."""
    ctx = [1, Q, page, page + 1, 127, 128, 129, 15, 17, 300, 0]
    _attend_check(*_attend_inputs(Q * 7 + D, len(ctx), Q, KV, G, D, page, kind, dtype, ctx))
    assert _status() == 0


def _random_tree(gen, B, Q):
    rows = []
    for _ in range(B):
        masks = []
        for j in range(Q):
            p = int(torch.randint(-1, j, (1,), generator=gen)) if j else -1
            masks.append((masks[p] if p >= 0 else 0) | (1 << j))
        rows.append([m - (1 << 64) if m >> 63 else m for m in masks])
    return torch.tensor(rows, dtype=torch.int64)


@pytest.mark.parametrize("Q,KV,G,D,page", [(9, 2, 4, 128, 16), (21, 1, 8, 64, 32), (64, 1, 2, 128, 16), (33, 2, 1, 64, 8)])
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_attention_trees(cuda, Q, KV, G, D, page, kind):
    import specq
    ctx = [Q, Q + 1, Q + page, Q + 131, 400, 3]
    args = _attend_inputs(Q, len(ctx), Q, KV, G, D, page, kind, torch.float16, ctx)
    gen = torch.Generator().manual_seed(Q)
    tree = _random_tree(gen, len(ctx), Q).cuda()
    _attend_check(*args, tree=tree)
    empty = tree.clone()
    empty[0] = 0                        # ctx = Q: these rows see nothing
    empty[1, 0] = 0                     # and this one only the token before the drafts
    got = _attend_check(*args, tree=empty)
    assert (got[0] == 0).all()
    chain = torch.tensor([[(1 << (j + 1)) - 1 if j < 63 else -1 for j in range(Q)]] * len(ctx)).cuda()
    causal = specq.paged_attention_blocks(*args)
    # the same window said as a tree (for contexts that hold all drafts): the same arithmetic
    got = specq.paged_attention_blocks(*args, tree=chain)
    assert torch.equal(got[:5], causal[:5])


def test_attention_long_and_cut(cuda):
    """Contexts long enough that a segment is cut over many blocks and joined, short ones beside them."""
    for seed, (B, Q, KV, G, D, page, ctx) in enumerate([(1, 1, 1, 4, 128, 16, [30011]), (2, 9, 2, 4, 128, 64, [9001, 40]),
                                                        (3, 4, 1, 8, 64, 8, [1, 12345, 700])]):
        _attend_check(*_attend_inputs(seed, B, Q, KV, G, D, page, "e4m3" if seed % 2 else "int8", torch.float16, ctx))
    assert _status() == 0


def test_attention_garbage_past_the_end(cuda):
    """Slots at and past ctx_len, pages of no sequence and table entries past the last page hold NaN bytes or
    nonsense; the outputs do not change by a bit."""
    import specq
    ctx = [5, 16, 33, 130, 0]
    for Q in (1, 4):
        q, kc, vc, ks, vs, tbl, cl = _attend_inputs(3, len(ctx), Q, 2, 4, 128, 16, "e4m3", torch.float16, ctx)
        ref = specq.paged_attention_blocks(q, kc, vc, ks, vs, tbl, cl)
        used = torch.zeros(kc.shape[:2], dtype=torch.bool)
        for b, n in enumerate(ctx):
            for t in range(n):
                used[int(tbl[b, t // 16]), t % 16] = True
        for c in (kc, vc):
            raw = c.view(torch.uint8)
            raw[~used.cuda()] = 0x7F
        dead = ~used.any(1).cuda()
        ks[dead], vs[dead] = float("nan"), float("inf")
        for b, n in enumerate(ctx):
            tbl[b, -(-n // 16):] = -7
        assert torch.equal(specq.paged_attention_blocks(q, kc, vc, ks, vs, tbl, cl), ref)
        assert _status() == 0


def test_attention_extreme_values(cuda):
    """Scores of hundreds (rows whose softmax is one token), page scales that differ by 2^20, a V scale of 0 and
    bf16 queries of 2^40: the running maximum is raised across pages of either order."""
    import specq
    for seed in range(4):
        q, kc, vc, ks, vs, tbl, cl = _attend_inputs(seed, 3, 3, 2, 4, 64, 16, "int8", torch.float16, [200, 333, 64])
        gen = torch.Generator().manual_seed(seed)
        if seed == 0:
            q = q * 40
        elif seed == 1:
            vs = vs * torch.exp2(torch.randint(-10, 11, vs.shape, generator=gen).float()).cuda()
        elif seed == 2:
            ks = ks * torch.exp2(torch.randint(-6, 3, ks.shape, generator=gen).float()).cuda()
        else:
            vs[tbl[1, 2].long()] = 0.0
        _attend_check(q, kc, vc, ks, vs, tbl, cl)
    q, kc, vc, ks, vs, tbl, cl = _attend_inputs(9, 2, 2, 1, 4, 128, 16, "int8", torch.bfloat16, [77, 150])
    big = q * 2.0 ** 40
    got = specq.paged_attention_blocks(big, kc, vc, ks, vs, tbl, cl, sm_scale=128 ** -0.5 * 2.0 ** -40)
    assert torch.equal(got, specq.paged_attention_blocks(q, kc, vc, ks, vs, tbl, cl))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_attention_rows_do_not_touch_each_other(cuda, dtype, bad):
    """A query row that holds an infinity or a NaN changes no other row by a bit."""
    import specq
    q, kc, vc, ks, vs, tbl, cl = _attend_inputs(11, 2, 5, 2, 4, 64, 16, "e4m3", dtype, [400, 33])
    ref = specq.paged_attention_blocks(q, kc, vc, ks, vs, tbl, cl)
    q[0, 2, 1, 7] = bad
    got = specq.paged_attention_blocks(q, kc, vc, ks, vs, tbl, cl)
    keep = torch.ones(2, 5, 8, dtype=torch.bool)
    keep[0, 2, 1] = False
    assert torch.equal(got[keep.cuda()], ref[keep.cuda()])


def test_attention_strides_heads_first_and_packed(cuda):
    """A cache laid out [P, H_KV, page, D], scales and queries with other strides, packed rows, out=."""
    import specq
    ctx = [40, 7, 161]
    q, kc, vc, ks, vs, tbl, cl = _attend_inputs(5, 3, 5, 2, 4, 128, 32, "int8", torch.float16, ctx)
    ref = specq.paged_attention_blocks(q, kc, vc, ks, vs, tbl, cl)
    flip = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731
    wide = torch.zeros(3, 9, dtype=torch.int32, device="cuda")
    wide[:, : tbl.shape[1]] = tbl
    got = specq.paged_attention_blocks(flip(q), flip(kc), flip(vc), ks.t().contiguous().t(), vs.t().contiguous().t(),
                                       wide[:, : tbl.shape[1]], cl)
    assert torch.equal(got, ref)
    packed = torch.full((16, 8 * 128 + 64), 3.0, device="cuda").half()
    x = packed[:, : 8 * 128].unflatten(1, (8, 128))
    x[:15] = q.reshape(15, 8, 128)
    out = torch.full((16, 8, 128), 7.0, device="cuda").half()
    specq.paged_attention_blocks(x, kc, vc, ks, vs, tbl, cl, q_len=5, out=out)
    assert torch.equal(out[:15].view(3, 5, 8, 128), ref) and (out[15] == 7.0).all()
    two = specq.paged_attention_blocks(q, kc, vc, ks, vs, tbl, cl, n_seqs=2)
    _attend_check(q[:2], kc, vc, ks, vs, tbl[:2], cl[:2], out=two[:2])
    assert (two[2] == 0).all()


def test_attention_plan_and_repeat(cuda):
    """Under a plan the active rows agree with the oracle and the others are not written; a repeated call gives
    the same bits; a captured graph serves other plans."""
    import specq
    B, Q, KV, G, D, page = 4, 9, 2, 4, 128, 16
    ctx = [300, 41, 9, 777]
    q, kc, vc, ks, vs, tbl, cl = _attend_inputs(6, B, Q, KV, G, D, page, "int8", torch.float16, ctx)
    assert torch.equal(specq.paged_attention_blocks(q, kc, vc, ks, vs, tbl, cl),
                       specq.paged_attention_blocks(q, kc, vc, ks, vs, tbl, cl))
    plan = torch.tensor([B, Q], dtype=torch.int32).cuda()
    x = q.reshape(B * Q, KV * G, D).clone()
    out = torch.full_like(x, 7.0)
    specq.paged_attention_blocks(x, kc, vc, ks, vs, tbl, cl, q_len=Q, out=out, plan=plan)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        specq.paged_attention_blocks(x, kc, vc, ks, vs, tbl, cl, q_len=Q, out=out, plan=plan)
    for n, ql in ((4, 9), (2, 3), (3, 1), (1, 9), (0, 4), (4, 0)):
        out.fill_(7.0)
        plan.copy_(torch.tensor([n, ql], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert (out[n * ql:] == 7.0).all()
        if n * ql:
            _attend_check(x[: n * ql].view(n, ql, KV * G, D), kc, vc, ks, vs, tbl[:n], cl[:n],
                          out=out[: n * ql].view(n, ql, KV * G, D))
    assert _status() == 0
    plan.copy_(torch.tensor([B + 1, Q], dtype=torch.int32))
    graph.replay()
    assert _status() != 0


def test_attention_bad_pages_and_lengths_are_reported(cuda):
    import specq
    from specq import _lib
    q, kc, vc, ks, vs, tbl, cl = _attend_inputs(8, 2, 1, 1, 4, 64, 16, "int8", torch.float16, [40, 20])
    ref = specq.paged_attention_blocks(q, kc, vc, ks, vs, tbl, cl)
    bad = tbl.clone()
    bad[0, 1] = kc.shape[0]
    got = specq.paged_attention_blocks(q, kc, vc, ks, vs, bad, cl)
    assert _status() == _lib.SPECQ_STATUS_BAD_INDEX
    assert torch.equal(got[1], ref[1]) and torch.isfinite(got).all()
    got = specq.paged_attention_blocks(q, kc, vc, ks, vs, tbl, torch.tensor([40, 49], dtype=torch.int32).cuda())
    assert _status() == _lib.SPECQ_STATUS_PLAN_CLAMPED
    assert torch.isfinite(got).all()
    assert specq.paged_attention_blocks(q[:0], kc, vc, ks, vs, tbl[:0], cl[:0]).shape == (0, 1, 4, 64)


def test_attention_on_another_stream(cuda):
    """Calls on two streams at once, each with its own tensors (and so its own workspace)."""
    import specq
    jobs = [_attend_inputs(s, 2, 9, 2, 4, 128, 16, "int8", torch.float16, [5000, 3000]) for s in (1, 2)]
    ref = [specq.paged_attention_blocks(*j) for j in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(specq.paged_attention_blocks(*jobs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, ref[i]) for g in got[i])


def test_offsets_past_32_bits(cuda):
    """A cache of over 2^31 numbers, pages at its end: append, attention, fork and compaction reach them."""
    import specq
    page, KV, D = 64, 8, 128
    P = (1 << 31) // (page * KV * D) + 40
    kc, vc = (torch.empty((P, page, KV, D), dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.empty((P, KV), device="cuda") for _ in range(2))
    gen = torch.Generator().manual_seed(0)
    last = torch.tensor([[P - 1, P - 9, P - 4, 2]], dtype=torch.int32).cuda()
    n = 150
    x = torch.randn(n, KV, D, generator=gen).half().cuda()
    ctx = torch.tensor([n], dtype=torch.int32).cuda()
    small = [torch.zeros((4, page, KV, D), dtype=torch.int8, device="cuda") for _ in range(2)]
    small += [torch.ones((4, KV), device="cuda") for _ in range(2)]
    order = torch.tensor([[0, 1, 2, 3]], dtype=torch.int32).cuda()
    for cache, tbl in (((kc, vc, ks, vs), last), (small, order)):
        specq.kv_append_blocks(x, x.flip(0), *cache, tbl, ctx, n)
    at = last[0].long()
    q = torch.randn(1, 2, 32, D, generator=gen).half().cuda()

    def same():
        for big, lit in zip((kc, vc), small):
            assert torch.equal(big[at].view(-1, KV, D)[:n], lit.view(-1, KV, D)[:n])
        assert torch.equal(specq.paged_attention_blocks(q, kc, vc, ks, vs, last, ctx),
                           specq.paged_attention_blocks(q, *small, order, ctx))
    same()
    acc = torch.tensor([[0, 2, 70, 90]], dtype=torch.int32).cuda()
    m = torch.tensor([4], dtype=torch.int32).cuda()
    for cache, tbl in (((kc, vc, ks, vs), last), (small, order)):
        specq.kv_compact_blocks(*cache, tbl, ctx, 100, acc, m)
    same()
    ref = torch.zeros(P, dtype=torch.int32, device="cuda")
    ref[at] = 1
    ref[: P - 3] += (ref[: P - 3] == 0).int()            # the only free pages are at the end
    tbl = torch.full((2, 4), -1, dtype=torch.int32, device="cuda")
    tbl[0] = last[0]
    held = torch.tensor([3, 0], dtype=torch.int32).cuda()
    specq.pages_fork(kc, vc, ks, vs, ref, tbl, held, torch.tensor([-1, 0], dtype=torch.int32).cuda(),
                     torch.tensor([n, 0], dtype=torch.int32).cuda())
    assert tbl[1].tolist() == [P - 1, P - 9, P - 3, -1]
    assert torch.equal(kc[P - 3, : n % page], kc[P - 4, : n % page]) and torch.equal(vs[P - 3], vs[P - 4])
    assert _status() == 0


# ---- compaction ----------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("D,KV,page,Q,L", [(128, 2, 16, 9, 1), (64, 3, 8, 33, 3), (128, 1, 64, 64, 2), (64, 1, 128, 5, 1),
                                           (128, 2, 32, 40, 1)])
def test_compact_exact(cuda, kind, D, KV, page, Q, L):
    import specq
    gen = torch.Generator().manual_seed(D + page + Q)
    ctx = torch.tensor([Q, Q + 1, Q + page - 1, Q + 3 * page + 3, Q + page // 2, Q + 7, Q + 2], dtype=torch.int32)
    B = len(ctx)
    C = int(ctx.max() - 1) // page + 1
    P = B * C + 1
    tbl = _table(gen, B, C, P)
    kc, vc = (_stored(gen, (L, P, page, KV, D), kind) for _ in range(2))
    ks, vs = (_scales(gen, (L, P, KV), kind) for _ in range(2))
    acc, n_acc = [], []
    for b in range(B):
        keep = [j for j in range(Q) if torch.rand((), generator=gen) < 0.5]
        keep = {0: list(range(Q)), 1: [], 2: [Q - 1]}.get(b, keep)     # all, none, the last
        acc.append(keep + [Q - 1] * (Q - len(keep)))
        n_acc.append(len(keep))
    want = []
    for c, s in ((kc, ks), (vc, vs)):
        c, s = _np(c).copy(), _np(s).copy()
        for layer in range(L):
            n = BO.compact(c[layer], s[layer], tbl.cpu().numpy(), ctx.numpy(), Q, acc, n_acc, kind)
        want.append((c, s))
    args = (tbl, ctx.cuda(), Q, torch.tensor(acc, dtype=torch.int32).cuda(), torch.tensor(n_acc, dtype=torch.int32).cuda())
    if L == 1:      # one layer by itself
        got = specq.kv_compact_blocks(kc[0], vc[0], ks[0], vs[0], *args)
    else:
        got = specq.kv_compact_blocks(kc, vc, ks, vs, *args)
    assert got.tolist() == list(n)
    for (c, s), gc, gs in zip(want, (kc, vc), (ks, vs)):
        assert np.array_equal(_np(gs), s)
        assert np.array_equal(_np(gc), c)
    assert _status() == 0


def test_compact_bad_indices_move_nothing(cuda):
    import specq
    from specq import _lib
    gen = torch.Generator().manual_seed(4)
    kc, vc = (_stored(gen, (6, 16, 2, 64), "int8") for _ in range(2))
    ks, vs = (_scales(gen, (6, 2), "int8") for _ in range(2))
    before = [t.clone() for t in (kc, vc, ks, vs)]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    for tbl, ctx, acc, n in (([[0, 1]], [20], [[1, 1]], [2]), ([[0, 1]], [20], [[2, 1]], [2]), ([[0, 1]], [20], [[1, 5]], [2]),
                             ([[0, 1]], [20], [[-1, 2]], [2]), ([[0, 1]], [20], [[1, 2]], [3]), ([[0, 1]], [20], [[1, 2]], [-1]),
                             ([[0, 9]], [20], [[1, 2]], [2]), ([[0, 1]], [33], [[1, 2]], [2]), ([[0, 1]], [4], [[1, 2]], [2])):
        got = specq.kv_compact_blocks(kc, vc, ks, vs, i32(tbl), i32(ctx), 5, i32(acc), i32(n))
        assert got.tolist() == ctx
        assert _status() == _lib.SPECQ_STATUS_BAD_INDEX
        assert all(torch.equal(a, b) for a, b in zip(before, (kc, vc, ks, vs)))


# ---- the page pool ---------------------------------------------------------------------------------
def _pool_state(gen, S, C, P):
    """Rows of random lengths, some sharing their first pages."""
    perm = torch.randperm(P, generator=gen)
    held = torch.randint(0, C + 1, (S,), generator=gen)
    while int(held.sum()) > P * 3 // 4:
        held //= 2
    tbl = torch.full((S, C), -1)
    at = 0
    for r in range(S):
        n = int(held[r])
        share = min(n, int(held[r - 1])) // 2 if r % 3 else 0
        tbl[r, :share] = tbl[r - 1, :share]
        tbl[r, share:n] = perm[at: at + n - share]
        at += n - share
    ref = torch.zeros(P, dtype=torch.int64)
    ref.index_add_(0, tbl[tbl >= 0], torch.ones(int((tbl >= 0).sum()), dtype=torch.int64))
    return [t.to(torch.int32) for t in (ref, tbl, held)]


@pytest.mark.parametrize("S,C,P,page", [(1, 1, 2, 16), (5, 7, 60, 8), (40, 33, 2000, 16), (1100, 9, 20011, 16), (700, 40, 30000, 8),
                                        (64, 20, 40000, 32)])
def test_pool_against_the_oracle(cuda, S, C, P, page):
    import specq
    gen = torch.Generator().manual_seed(S + P)
    ref, tbl, held = _pool_state(gen, S, C, P)
    if P == 40000:
        ref[:33000] += 1            # the lowest free page is far up
    o = BO.Pool(ref.numpy(), tbl.numpy(), held.numpy())
    ref, tbl, held = ref.cuda(), tbl.cuda(), held.cuda()
    KV, D, L = 2, 64, 2
    kc, vc = (torch.randint(-127, 128, (L, P, page, KV, D), generator=torch.Generator(device="cuda").manual_seed(i),
                            device="cuda", dtype=torch.int16).to(torch.int8) for i in (1, 2))
    ks, vs = (torch.rand((L, P, KV), device="cuda") for _ in range(2))

    def same():
        assert np.array_equal(ref.cpu().numpy(), o.ref)
        assert np.array_equal(tbl.cpu().numpy(), o.tbl)
        assert np.array_equal(held.cpu().numpy(), o.held)
    for step in range(4):
        drop = torch.rand(S, generator=gen) < 0.3
        specq.pages_release(ref, tbl, held, drop.cuda())
        o.release(drop.numpy())
        same()
        want = torch.randint(0, C * page + 1, (S,), generator=gen, dtype=torch.int32)
        short = specq.pages_reserve(ref, tbl, held, want.cuda(), page)
        assert short.item() == o.reserve(want.numpy(), page)
        same()
        parent = torch.randint(-2, S, (S,), generator=gen, dtype=torch.int32)
        length = torch.minimum(torch.randint(0, C * page + 1, (S,), generator=gen),
                               torch.from_numpy(o.held.astype(np.int64)) * page).to(torch.int32)
        before = [t.clone() for t in (kc, vc, ks, vs)]
        short = specq.pages_fork(kc, vc, ks, vs, ref, tbl, held, parent.cuda(), length.cuda())
        missing, copies = o.fork(parent.numpy(), length.numpy(), page)
        assert short.item() == missing
        same()
        for frm, to, n in copies:
            before[0][:, to, :n], before[1][:, to, :n] = before[0][:, frm, :n], before[1][:, frm, :n]
            before[2][:, to], before[3][:, to] = before[2][:, frm], before[3][:, frm]
        assert all(torch.equal(a, b) for a, b in zip(before, (kc, vc, ks, vs)))
    assert _status() == 0


def test_pool_is_all_or_none_and_reports(cuda):
    import specq
    from specq import _lib
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    ref, tbl, held = i32([0, 1, 0, 0]), i32([[1, -1, -1], [-1, -1, -1]]), i32([1, 0])
    state = [t.clone() for t in (ref, tbl, held)]
    assert specq.pages_reserve(ref, tbl, held, i32([48, 32]), 16).item() == 1       # 2 + 2 wanted, 3 free
    assert all(torch.equal(a, b) for a, b in zip(state, (ref, tbl, held)))
    assert specq.pages_reserve(ref, tbl, held, i32([33, -5]), 16).item() == 0
    assert tbl.tolist() == [[1, 0, 2], [-1, -1, -1]] and ref.tolist() == [1, 1, 1, 0] and held.tolist() == [3, 0]
    assert _status() == 0
    specq.pages_reserve(ref, tbl, held, i32([99, 0]), 16)                           # past the table's columns
    assert _status() == _lib.SPECQ_STATUS_PLAN_CLAMPED
    kc = torch.zeros(4, 16, 1, 64, dtype=torch.int8, device="cuda")
    ks = torch.ones(4, 1, device="cuda")
    state = [t.clone() for t in (ref, tbl, held)]
    # a parent outside the table, and a length past the parent's pages: the row stays
    assert specq.pages_fork(kc, kc.clone(), ks, ks.clone(), ref, tbl, held, i32([-1, 7]), i32([40, 0])).item() == 0
    assert _status() == _lib.SPECQ_STATUS_BAD_INDEX
    specq.pages_fork(kc, kc.clone(), ks, ks.clone(), ref, tbl, held, i32([-1, 0]), i32([49, 0]))
    assert _status() == _lib.SPECQ_STATUS_BAD_INDEX
    assert all(torch.equal(a, b) for a, b in zip(state, (ref, tbl, held)))
    # no free page for the copy of a part-filled one
    full = i32([1, 1, 1, 1])
    assert specq.pages_fork(kc, kc.clone(), ks, ks.clone(), full, tbl, held, i32([-1, 0]), i32([40, 0])).item() == 1
    assert full.tolist() == [1, 1, 1, 1] and held.tolist() == [3, 0]
    # a permutation of beams, and a fork of no tokens
    ref, tbl, held = i32([1, 1, 0, 0]), i32([[0], [1]]), i32([1, 1])
    assert specq.pages_fork(kc, kc.clone(), ks, ks.clone(), ref, tbl, held, i32([1, 0]), i32([16, 16])).item() == 0
    assert tbl.tolist() == [[1], [0]] and ref.tolist() == [1, 1, 0, 0]
    assert specq.pages_fork(kc, kc.clone(), ks, ks.clone(), ref, tbl, held, i32([1, -1]), i32([16, 0])).item() == 0
    assert tbl.tolist() == [[-1], [0]] and ref.tolist() == [1, 0, 0, 0] and held.tolist() == [0, 1]
    assert _status() == 0
