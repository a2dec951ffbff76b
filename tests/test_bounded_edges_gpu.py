"""attention_mass_blocks where scores, scales and tables are out of the ordinary, in each form that a call is cut into.

Bounds as in test_bounded_cache_gpu.py, whose oracle, cases' makers and check these tests use."""
import numpy as np
import pytest
import torch

from oracle import bounded_oracle as O
from test_bounded_cache_gpu import _cache, _check_mass, _i32, _numbers, _table

pytestmark = pytest.mark.gpu

# new tokens, heads of a group, tokens of the table: one launch, one launch of a cluster, a stream of tiles (up to 16 rows), a cluster, two
# passes (17 to 95), tcgen05 (96 and more)
FORMS = [(2, 4, 512), (3, 1, 512), (4, 4, 1024), (2, 2, 4608), (4, 4, 4608), (3, 8, 1024), (4, 8, 4608), (3, 32, 1024), (4, 32, 4608)]


@pytest.mark.parametrize("missing", [False, True])
@pytest.mark.parametrize("score", [-100.0, -181.0])
@pytest.mark.parametrize("kind", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("Q,G,tokens", FORMS)
def test_mass_of_very_negative_scores(cuda, Q, G, tokens, kind, score, missing):
    """Every score far below 0, where a row's sum is below 2^-128 of its own and some 32 tokens of a context are seen by none or by the
    later rows only."""
    import specq
    D, page, ctx = 128, 16, [33, 65, 290]
    C = tokens // page
    g = torch.Generator(device="cuda").manual_seed(Q * G)
    kc, _, ks, _ = _cache(3 * C + 1, page, 1, D, kind, g)
    kc.copy_(torch.full(kc.shape, 4.0, device="cuda").to(kind))
    ks.fill_(1.0)
    tbl = _table(3, C, 3 * C + 1, g)
    if missing:
        tbl[0, 2], tbl[1, 2:4], tbl[2, 4:6] = -1, 3 * C + 1, -1     # whole tiles, and the only one that the last row alone sees
    q = torch.full((3, Q, G, D), score / (4 * D ** 0.5), device="cuda").half()
    mass = torch.rand(3, 1, tokens, generator=g, device="cuda")
    m = specq.attention_mass_blocks(q, kc, ks, tbl, _i32(ctx), mass.clone(), decay=0.5)
    specq.get_status()
    _check_mass(m, q, kc, ks, tbl, _i32(ctx), mass, decay=0.5)


@pytest.mark.parametrize("power", [60, 120])
@pytest.mark.parametrize("kind", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("Q,tokens", [(4, 512), (4, 4608), (12, 1024), (12, 4608), (48, 1024), (48, 4608)])
def test_mass_of_a_large_row_beside_ordinary_ones(cuda, Q, tokens, kind, power):
    """Rows of 2^60, or of 2^120 (whose scores are past fp32), and ordinary ones in one call (two heads of a group): a large row puts its
    weight on one token, and the others lose no bits to it, since each row has its own power of two.  The bound is made from the ordinary
    rows alone."""
    import specq
    D, page, ctx = 64, 16, [33, 65, 290]
    C = tokens // page
    g = torch.Generator(device="cuda").manual_seed(Q + 3)
    kc, _, ks, _ = _cache(3 * C, page, 1, D, kind, g)
    tbl = _table(3, C, 3 * C, g)
    q = torch.randn(3, Q, 2, D, generator=g, device="cuda").bfloat16()
    q[:, :, 1] *= 2.0 ** power
    zero = np.zeros((3, 1, tokens))

    def oracle(rows):
        return O.attention_mass(rows.double().cpu().numpy(), _numbers(kc), ks.cpu().numpy(), tbl.cpu().numpy(), ctx, zero)
    plain, size = oracle(q[:, :, :1])
    large, _ = oracle(q[:, :, 1:])
    assert np.isin(large, np.arange(Q + 1)).all()          # no two of a large row's scores meet
    m = specq.attention_mass_blocks(q, kc, ks, tbl, _i32(ctx), torch.zeros(3, 1, tokens, device="cuda"))
    rel = 2 * (D + 4) * 2.0 ** -23 * size + 2.0 ** -20 + 2 * Q * 2.0 ** -24
    err = np.abs(m.double().cpu().numpy() - plain - large)
    bound = rel * plain + 2.0 ** -23 * (plain + large) + 1e-12
    assert (err <= bound).all(), (err / bound).max()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("kind", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("Q,G,tokens", FORMS)
def test_mass_of_pages_of_scale_zero(cuda, Q, G, tokens, kind, dtype):
    """A key of a page of scale 0 has the score 0, in tiles that rows see in part and in tiles that they see whole, beside pages outside
    the cache."""
    import specq
    D, page, ctx = 64, 16, [33, 65, 290]
    C = tokens // page
    g = torch.Generator(device="cuda").manual_seed(Q * G + 1)
    kc, _, ks, _ = _cache(3 * C + 1, page, 1, D, kind, g)
    tbl = _table(3, C, 3 * C + 1, g)
    for b, n in enumerate(ctx):
        ks[tbl[b, [0, (n - 1) // page]].long()] = 0.0
    ks[tbl[2, 4:9].long()] = 0.0                 # whole tiles
    q = torch.randn(3, Q, G, D, generator=g, device="cuda").to(dtype)
    mass = torch.rand(3, 1, tokens, generator=g, device="cuda")
    for missing in (False, True):
        if missing:
            tbl[0, 1], tbl[2, 3], tbl[2, 5] = -1, 3 * C + 1, -1
        m = specq.attention_mass_blocks(q, kc, ks, tbl, _i32(ctx), mass.clone(), decay=0.5)
        _check_mass(m, q, kc, ks, tbl, _i32(ctx), mass, decay=0.5)
    specq.get_status()


@pytest.mark.parametrize("Q,G,tokens", FORMS)
def test_mass_of_tiny_rows_beside_pages_of_zeros(cuda, Q, G, tokens):
    """bf16 rows of 2^-120 and the least scale that the append writes: their product leaves fp32, the score is 0."""
    import specq
    D, page, ctx = 64, 16, [33, 65, 290]
    C = tokens // page
    g = torch.Generator(device="cuda").manual_seed(Q * G + 2)
    kc, _, ks, _ = _cache(3 * C, page, 1, D, torch.int8, g)
    tbl = _table(3, C, 3 * C, g)
    for b, n in enumerate(ctx):
        last = tbl[b, (n - 1) // page].long()
        kc[last], ks[last] = 0, 1e-8 / 127
    q = torch.randn(3, Q, G, D, generator=g, device="cuda").bfloat16()
    q[:, -1] *= 2.0 ** -120
    mass = torch.rand(3, 1, tokens, generator=g, device="cuda")
    m = specq.attention_mass_blocks(q, kc, ks, tbl, _i32(ctx), mass.clone())
    _check_mass(m, q, kc, ks, tbl, _i32(ctx), mass)


@pytest.mark.parametrize("B,Q,KV,G,cols", [
    (17, 4, 8, 4, 8192), (1, 4, 8, 4, 131072),        # a stream of tiles: sequences in three turns, heads in three
    (6, 11, 8, 8, 524288),                            # two passes of 88 rows: sequences in two turns
    (2, 200, 4, 8, 131072), (1, 300, 4, 8, 131072)])  # tcgen05: sequences in two turns, heads in two
def test_mass_of_short_contexts_in_a_wide_table(cuda, B, Q, KV, G, cols):
    """Tables whose scores or sums would fill more than the workspace: sequence by sequence or head by head, with the same result."""
    import specq
    D, page = 64, 16
    ctx = [(37 * b) % 600 for b in range(B - 1)] + [777]
    g = torch.Generator(device="cuda").manual_seed(B)
    kc, _, ks, _ = _cache(B * 50, page, KV, D, torch.int8, g)
    tbl = torch.full((B, cols), -1, dtype=torch.int32, device="cuda")
    tbl[:, :50] = _table(B, 50, B * 50, g)
    rows = [Q - b % 2 for b in range(B)]
    q = torch.randn(B, Q, KV * G, D, generator=g, device="cuda").half()
    mass = torch.zeros(B, KV, cols * page, device="cuda")
    mass[:, :, :800] = torch.rand(B, KV, 800, generator=g, device="cuda")
    before, small = mass.clone(), mass[:, :, :800].contiguous()
    m = specq.attention_mass_blocks(q, kc, ks, tbl, _i32(ctx), mass, n_rows=_i32(rows), decay=0.5)
    _check_mass(m[:, :, :800], q, kc, ks, tbl[:, :50], _i32(ctx), small, n_rows=rows, decay=0.5)
    for b, n in enumerate(ctx):
        assert torch.equal(m[b, :, n:], before[b, :, n:])
    packed = specq.attention_mass_blocks(q.flatten(0, 1), kc, ks, tbl, _i32(ctx), before, q_len=Q, n_rows=_i32(rows), decay=0.5)
    assert torch.equal(packed, m)


def test_what_is_written_in_place_is_known_to_autograd(cuda):
    """A tensor that a call has written counts as changed, so that a backward pass that saved it ends in an error, not in a wrong gradient."""
    import specq
    g = torch.Generator(device="cuda").manual_seed(9)
    D, page = 64, 16
    table, pos = specq.rope_table(32, D), torch.arange(4, dtype=torch.int32, device="cuda")
    w = torch.ones(D, device="cuda", dtype=torch.float16, requires_grad=True)
    q, k, v = (torch.randn(4, 2, D, generator=g, device="cuda").half() for _ in range(3))
    kc, vc, ks, vs = _cache(4, page, 2, D, torch.int8, g)
    tbl, ctx = _i32([[0, 1], [2, 3]]), _i32([20, 18])
    mass, state = torch.zeros(2, 2, 32, device="cuda"), torch.zeros(4, 3, device="cuda")

    def saved(call, *written):
        before = [t._version for t in written]
        call()
        return all(t._version > n for t, n in zip(written, before))
    assert saved(lambda: specq.rope(q, pos, table, out=q), q)
    assert saved(lambda: specq.qk_norm_rope(q, k, None, None, pos, table, q_out=q, k_out=k), q, k)
    assert saved(lambda: specq.kv_append_blocks(k, v, kc, vc, ks, vs, tbl, ctx, 2, q=q, q_out=q, table=table), q, kc, vc, ks, vs)
    out = torch.empty_like(q)
    assert saved(lambda: specq.paged_attention_blocks(q, kc, vc, ks, vs, tbl, ctx, q_len=2, out=out), out)
    assert saved(lambda: specq.attention_mass_blocks(q, kc, ks, tbl, ctx, mass, q_len=2), mass)
    assert saved(lambda: specq.kv_compact_blocks(kc, vc, ks, vs, tbl, ctx, 2, _i32([[0], [1]]), _i32([1, 1])), kc, vc, ks, vs)
    assert saved(lambda: specq.kv_evict_blocks(kc, vc, ks, vs, tbl, ctx, mass, 8, ctx_out=ctx), kc, vc, ks, vs, mass, ctx)
    assert saved(lambda: specq.beam_reorder([state, pos], _i32([[1, 0], [2, 2]])), state, pos)
    ref, held, drop = _i32([1, 1, 1, 1]), _i32([2, 2]), torch.tensor([False, True], device="cuda")
    assert saved(lambda: specq.pages_release(ref, tbl, held, drop), ref, tbl, held)
    assert saved(lambda: specq.pages_reserve(ref, tbl, held, _i32([20, 20]), page), ref, tbl, held)
    assert saved(lambda: specq.pages_fork(kc, vc, ks, vs, ref, tbl, held, _i32([-1, 0]), _i32([20, 20])), kc, vc, ks, vs, ref, tbl, held)
    assert saved(lambda: specq.pages_release(ref, tbl, held, drop, length=_i32([3, 3]), page=page), ref, tbl, held)

    pos = torch.arange(4, dtype=torch.int32, device="cuda")
    for change in (lambda: specq.rope(q, pos, table, out=q), lambda: specq.beam_reorder([pos], _i32([1, 0, 2, 3]), beams=4)):
        a, _ = specq.qk_norm_rope(q, k, w, w, pos, table)
        change()
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            a.sum().backward()
    a, _ = specq.qk_norm_rope(q, k, w, w, pos, table)
    torch.autograd.grad(a.float().sum(), w)
    with torch.inference_mode():                            # tensors without a count
        x = q.clone()
        specq.rope(x, pos, table, out=x)
    specq.rope(x, pos, table, out=x)


@pytest.mark.parametrize("given", [False, True])
def test_evict_of_a_large_budget_goes_in_turns(cuda, given):
    """260 sequences, 8 heads and a budget of 65536 tokens: more places than the workspace has.  As one sequence after another; the pages are
    all alike, so that the masses and lengths alone tell the tokens apart."""
    import specq
    g = torch.Generator(device="cuda").manual_seed(13)
    B, KV, D, page, keep, recent = 260, 8, 64, 128, 65536, 100
    cols = keep // page + 1
    kc, vc = (torch.zeros(B, page, KV, D, dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = torch.ones(B, KV, device="cuda"), torch.ones(B, KV, device="cuda")
    tbl = torch.arange(B, dtype=torch.int32, device="cuda")[:, None].repeat(1, cols)
    ctx = _i32([keep + (b * 7) % (page + 1) - 3 for b in range(B)])
    mass = torch.rand(B, KV, cols * page, generator=g, device="cuda")
    before, old = mass.clone(), ctx.tolist()
    out = specq.kv_evict_blocks(kc, vc, ks, vs, tbl, ctx, mass, keep, recent, ctx_out=ctx if given else None)
    assert out.tolist() == [min(n, keep) for n in old]
    for b in (0, 1, 64, 129, 130, 200, 258, 259):
        one = before[b:b + 1].clone()
        n = specq.kv_evict_blocks(kc, vc, ks, vs, tbl[b:b + 1], _i32(old[b:b + 1]), one, keep, recent)
        assert n.tolist() == [min(old[b], keep)] and torch.equal(one[0], mass[b])
        if old[b] > keep:
            at = O.evict_choice(before[b, 3].cpu().numpy(), old[b], keep, recent)
            assert torch.equal(mass[b, 3, :keep], before[b, 3, torch.from_numpy(at).cuda()]) and not mass[b, 3, keep:old[b]].any()
