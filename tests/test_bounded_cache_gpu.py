"""attention_mass_blocks, kv_evict_blocks and pages_release's tail against the float64 oracle.

Mass: a score of size at most A (the sum of |q k| times the scale) is off by at most (D + 4) 2^-23 A (the tensor
core cuts the sum's bits off, the scales' products round), so a weight by twice that relative to itself (its own score and lse),
with 2^-20 for the exponentials, their sums in groups of 32 and over tiles, and the logarithm.  It adds up over rows, and decay and
the sum round once more.  Eviction: exact, since it chooses by given masses and rounds as the definition says."""
import numpy as np
import pytest
import torch

from oracle import bounded_oracle as O

pytestmark = pytest.mark.gpu

TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def _numbers(cache):
    return cache.float().cpu().numpy()


def _cache(P, page, KV, D, dtype, g, lead=()):
    def one():
        x = (torch.randn(*lead, P, page, KV, D, generator=g, device="cuda") * TOP[dtype] / 4).clamp(-TOP[dtype], TOP[dtype])
        return x.round().to(dtype) if dtype == torch.int8 else x.to(dtype)

    def scale():
        return (torch.rand(*lead, P, KV, generator=g, device="cuda") * 2 + 1) / TOP[dtype]
    return one(), one(), scale(), scale()


def _table(B, C, P, g):
    return torch.randperm(P, generator=g, device="cuda")[: B * C].to(torch.int32).view(B, C)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _check_mass(got, q, kc, ks, tbl, ctx, mass, **kw):
    B, Q, H, D = q.shape
    ref, size = O.attention_mass(q.double().cpu().numpy(), _numbers(kc), ks.cpu().numpy(), tbl.cpu().numpy(), ctx.tolist(),
                                 mass.double().cpu().numpy(), **kw)
    rel = 2 * (D + 4) * 2.0 ** -23 * size + 2.0 ** -20 + Q * (H // kc.shape[2]) * 2.0 ** -24
    added = ref - mass.double().cpu().numpy() * kw.get("decay", 1.0)
    err = np.abs(got.double().cpu().numpy() - ref)
    bound = rel * np.maximum(added, 0) + 2.0 ** -23 * np.abs(ref) + 1e-12
    assert (err <= bound).all(), (err / bound).max()


CASES = [  # B, Q, KV, G, D, page, contexts
    (1, 1, 1, 1, 64, 8, [1]), (1, 1, 8, 4, 128, 16, [37]), (3, 1, 2, 8, 64, 32, [5, 256, 257]), (2, 9, 2, 4, 128, 16, [700, 9]),
    (4, 1, 1, 4, 128, 64, [2000, 1, 0, 513]), (2, 64, 1, 8, 64, 128, [900, 64]), (2, 33, 2, 3, 128, 8, [300, 40]),
    (1, 5, 1, 1, 64, 16, [3]), (2, 300, 1, 2, 64, 32, [400, 300]), (1, 1, 2, 2, 128, 128, [5000]), (3, 2, 4, 1, 64, 64, [4097, 63, 2500]),
    (1, 9, 1, 4, 128, 64, [5000]), (2, 20, 1, 4, 64, 8, [4500, 100]), (1, 48, 1, 8, 128, 16, [4700]), (2, 24, 2, 4, 64, 16, [257, 90])]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("kind", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("B,Q,KV,G,D,page,ctx", CASES)
def test_mass_matches_oracle(cuda, dtype, kind, B, Q, KV, G, D, page, ctx):
    import specq
    g = torch.Generator(device="cuda").manual_seed(B * 100 + Q)
    C = -(-max(ctx) // page) + 1
    P = B * C + 2
    kc, _, ks, _ = _cache(P, page, KV, D, kind, g)
    tbl = _table(B, C, P, g)
    q = torch.randn(B, Q, KV * G, D, generator=g, device="cuda").to(dtype)
    # where no sequence has a token anything may stand
    N = C * page + 5
    mass = torch.rand(B, KV, N, generator=g, device="cuda")
    for decay in (1.0, 0.5):
        m = mass.clone()
        out = specq.attention_mass_blocks(q, kc, ks, tbl, _i32(ctx), m, decay=decay)
        assert out is m
        _check_mass(m, q, kc, ks, tbl, _i32(ctx), mass, decay=decay)
        for b, n in enumerate(ctx):
            assert torch.equal(m[b, :, n:], mass[b, :, n:])
    packed = specq.attention_mass_blocks(q.view(B * Q, KV * G, D), kc, ks, tbl, _i32(ctx), mass.clone(), q_len=Q, decay=0.5)
    assert torch.equal(packed, m)


def test_mass_adds_up_to_the_rows(cuda):
    """Each row's weights sum to 1: the added mass of a head is rows times heads (sums of up to 4096 in fp32)."""
    import specq
    g = torch.Generator(device="cuda").manual_seed(0)
    B, Q, KV, G, D, page, C = 3, 7, 2, 4, 128, 16, 256
    kc, _, ks, _ = _cache(B * C, page, KV, D, torch.int8, g)
    tbl = _table(B, C, B * C, g)
    q = torch.randn(B, Q, KV * G, D, generator=g, device="cuda").half()
    m = specq.attention_mass_blocks(q, kc, ks, tbl, _i32([4096, 7, 1000]), torch.zeros(B, KV, C * page, device="cuda"))
    assert (m.double().sum(-1) - Q * G).abs().max() <= Q * G * 1e-5


def test_mass_counted_rows(cuda):
    """n_rows: a padded batch; none, one and all rows, more than there are, fewer tokens than rows."""
    import specq
    g = torch.Generator(device="cuda").manual_seed(1)
    B, Q, KV, G, D, page, C = 5, 6, 2, 2, 64, 16, 40
    kc, _, ks, _ = _cache(B * C, page, KV, D, torch.float8_e4m3fn, g)
    tbl = _table(B, C, B * C, g)
    q = torch.randn(B, Q, KV * G, D, generator=g, device="cuda").half()
    ctx, rows = [600, 500, 20, 4, 300], [0, 1, 6, 6, 9]
    for b, r in enumerate(rows):
        q[b, max(r, 0):] = float("nan")                 # padding is not looked at
    mass = torch.rand(B, KV, C * page, generator=g, device="cuda")
    m = specq.attention_mass_blocks(q, kc, ks, tbl, _i32(ctx), mass.clone(), n_rows=_i32(rows), decay=0.9)
    ref, size = O.attention_mass(q.double().cpu().numpy(), _numbers(kc), ks.cpu().numpy(), tbl.cpu().numpy(), ctx, mass.double().cpu().numpy(),
                                 n_rows=rows, decay=0.9)
    assert np.abs(m.double().cpu().numpy() - ref).max() <= (2 * (D + 4) * 2.0 ** -23 * size + 2.0 ** -20) * Q * G + 2.0 ** -22
    assert torch.equal(m[0], mass[0])


@pytest.mark.parametrize("ctx", [200, 900])
def test_mass_strange_values(cuda, ctx):
    """Queries of zeros, huge, tiny, with a NaN or an infinity; stale bytes past the end; pages outside the cache."""
    import specq
    g = torch.Generator(device="cuda").manual_seed(2)
    B, Q, KV, G, D, page, C = 2, 8, 1, 2, 64, 16, 64
    for kind in (torch.int8, torch.float8_e4m3fn):
        kc, _, ks, _ = _cache(B * C + 1, page, KV, D, kind, g)
        tbl = _table(B, C, B * C + 1, g)
        q = torch.randn(B, Q, KV * G, D, generator=g, device="cuda").bfloat16()
        q[:, 0] = 0
        q[:, 1] *= 2.0 ** -100
        q[:, 2] *= 2.0 ** -20
        q[0, 3, 0, 5], q[0, 4, 1, 7], q[1, 5, 0, 0] = float("nan"), float("inf"), -float("inf")
        stale = tbl[:, -(-ctx // page):].flatten().long()
        kc.view(torch.uint8)[stale] = 0x7F
        ks[stale] = float("nan")
        mass = torch.rand(B, KV, C * page, generator=g, device="cuda")
        m = specq.attention_mass_blocks(q, kc, ks, tbl, _i32([ctx, ctx - 3]), mass.clone())
        _check_mass(m, q, kc, ks.nan_to_num(), tbl, _i32([ctx, ctx - 3]), mass)
        specq.get_status()
        tbl[0, 3], tbl[1, 0], tbl[1, 2] = -1, B * C + 1, 1 << 30
        m = specq.attention_mass_blocks(q, kc, ks, tbl, _i32([ctx, ctx - 3]), mass.clone())
        assert specq.get_status() == specq._lib.SPECQ_STATUS_BAD_INDEX
        _check_mass(m, q, kc, ks.nan_to_num(), tbl, _i32([ctx, ctx - 3]), mass)
    # one row far larger than the others takes no bits from them
    q = torch.randn(B, Q, KV * G, D, generator=g, device="cuda").bfloat16()
    q[:, 0] *= 2.0 ** 60
    m = specq.attention_mass_blocks(q[:, 1:], kc, ks, tbl, _i32([ctx, ctx - 3]), mass.clone())
    one = specq.attention_mass_blocks(q[:, 1:].contiguous(), kc, ks, tbl, _i32([ctx, ctx - 3]), mass.clone())
    assert torch.equal(m, one)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("kind,D,page", [(torch.int8, 128, 16), (torch.float8_e4m3fn, 64, 8)])
def test_mass_of_many_rows_in_strange_company(cuda, dtype, kind, D, page):
    """Counted rows that end inside a group of 128, dead rows, pages outside the cache, stale bytes, a tile that ends in a page."""
    import specq
    g = torch.Generator(device="cuda").manual_seed(6)
    B, Q, KV, G, C = 4, 50, 2, 4, 1300 // page
    kc, _, ks, _ = _cache(B * C + 1, page, KV, D, kind, g)
    tbl = _table(B, C, B * C + 1, g)
    q = torch.randn(B, Q, KV * G, D, generator=g, device="cuda").to(dtype)
    ctx, rows = [1290, 1025, 30, 600], [50, 33, 50, 0]
    q[0, 7, 1, 3], q[0, 40, 5, 9], q[1, 32, 2, 0] = float("nan"), float("inf"), -float("inf")
    q[0, 20] = 0
    for b, n in enumerate(ctx):
        stale = tbl[b, -(-n // page):].flatten().long()
        kc.view(torch.uint8)[stale] = 0x7F
        ks[stale] = float("nan")
        if n % page:
            kc.view(torch.uint8)[tbl[b, n // page].long(), n % page:] = 0x7F
    tbl[0, 3], tbl[1, 1024 // page], tbl[2, 0] = -1, B * C + 1, 1 << 30
    mass = torch.rand(B, KV, C * page, generator=g, device="cuda")
    specq.get_status()
    m = specq.attention_mass_blocks(q, kc, ks, tbl, _i32(ctx), mass.clone(), n_rows=_i32(rows), decay=0.75)
    assert specq.get_status() == specq._lib.SPECQ_STATUS_BAD_INDEX
    _check_mass(m, q, torch.nan_to_num(kc.float()) if kind != torch.int8 else kc, ks.nan_to_num(), tbl, _i32(ctx), mass, n_rows=rows, decay=0.75)
    assert torch.equal(m[3], mass[3])
    again = specq.attention_mass_blocks(q, kc, ks, tbl, _i32(ctx), mass.clone(), n_rows=_i32(rows), decay=0.75)
    assert torch.equal(m, again)


def test_mass_context_past_its_table(cuda):
    import specq
    g = torch.Generator(device="cuda").manual_seed(3)
    kc, _, ks, _ = _cache(8, 16, 1, 64, torch.int8, g)
    tbl = _table(2, 4, 8, g)
    q = torch.randn(2, 1, 2, 64, generator=g, device="cuda").half()
    mass = torch.zeros(2, 1, 64, device="cuda")
    specq.get_status()
    m = specq.attention_mass_blocks(q, kc, ks, tbl, _i32([65, -3]), mass.clone())
    assert specq.get_status() == specq._lib.SPECQ_STATUS_PLAN_CLAMPED
    _check_mass(m, q, kc, ks, tbl, _i32([64, 0]), mass)


def test_mass_agrees_with_attention(cuda):
    """Over values that are unit vectors of the tokens, attention gives the weights themselves."""
    import specq
    g = torch.Generator(device="cuda").manual_seed(4)
    D, page = 64, 16
    kc, vc, ks, vs = _cache(4, page, 1, D, torch.int8, g)
    vc.zero_()
    tbl = _i32([[2, 0, 3, 1]])
    for t in range(D):
        vc[tbl[0, t // page], t % page, 0, t] = 1
    vs.fill_(1.0)
    q = torch.randn(1, 3, 2, D, generator=g, device="cuda").half()
    out = specq.paged_attention_blocks(q, kc, vc, ks, vs, tbl, _i32([D]))
    m = specq.attention_mass_blocks(q, kc, ks, tbl, _i32([D]), torch.zeros(1, 1, D, device="cuda"))
    # the attention's output has been rounded to fp16, from weights in fp16
    assert (out.float().sum((0, 1, 2)) - m[0, 0]).abs().max() <= 6 * 2.0 ** -10


def test_mass_streams_and_graph(cuda):
    import specq
    g = torch.Generator(device="cuda").manual_seed(5)
    B, Q, KV, G, D, page, C = 2, 4, 2, 4, 128, 32, 40
    kc, _, ks, _ = _cache(B * C, page, KV, D, torch.int8, g)
    tbl, ctx = _table(B, C, B * C, g), _i32([1200, 800])
    q = torch.randn(B, Q, KV * G, D, generator=g, device="cuda").half()
    zero = torch.zeros(B, KV, C * page, device="cuda")
    ref = specq.attention_mass_blocks(q, kc, ks, tbl, ctx, zero.clone())
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        a = specq.attention_mass_blocks(q, kc, ks, tbl, ctx, zero.clone())
    b = specq.attention_mass_blocks(q, kc, ks, tbl, ctx, zero.clone())     # at the same time
    side.synchronize()
    assert torch.equal(a, ref) and torch.equal(b, ref)
    m = zero.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        specq.attention_mass_blocks(q, kc, ks, tbl, ctx, m, decay=0.5)
    m.zero_()
    ctx.copy_(_i32([300, 1280]))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(m, specq.attention_mass_blocks(q, kc, ks, tbl, ctx, zero.clone(), decay=0.5))


# ---- eviction ----------------------------------------------------------------------------------------
def _requant(kind):
    def f(row, ratio):
        x = torch.from_numpy(np.asarray(row, np.float32)) * torch.tensor(ratio, dtype=torch.float32)
        return (x.round().clamp(-127, 127) if kind == torch.int8 else x.to(torch.float8_e4m3fn).float()).numpy()
    return f


def _check_evict(before, after, tbl, ctx, keep, recent, kind, ctx_out):
    """before, after: (kc, vc, ks, vs, mass) with layers."""
    t, m = tbl.cpu().numpy(), before[4].cpu().numpy()
    assert ctx_out.tolist() == [min(n, keep) if n > 0 else n for n in ctx]
    for i in (0, 1):
        num, scale = _numbers(before[i]), before[2 + i].cpu().numpy().copy()
        for l in range(num.shape[0]):
            O.evict(num[l], scale[l], t, ctx, m[l], keep, recent, _requant(kind))
        assert (scale == after[2 + i].cpu().numpy()).all()
        same = (num == _numbers(after[i])) | (np.isnan(num) & np.isnan(_numbers(after[i])))
        assert same.all(), np.argwhere(~same)[:4]
    want = m.copy()
    for l in range(m.shape[0]):
        for b, n in enumerate(ctx):
            if n > keep:
                for h in range(m.shape[2]):
                    at = O.evict_choice(m[l, b, h], n, keep, recent)
                    want[l, b, h, :n] = 0
                    want[l, b, h, :keep] = m[l, b, h, at]
    got = after[4].cpu().numpy()
    assert ((want == got) | (np.isnan(want) & np.isnan(got))).all()


@pytest.mark.parametrize("kind", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("L,B,KV,D,page,ctx,keep,recent", [
    (1, 1, 1, 64, 8, [9], 8, 0), (1, 1, 1, 64, 8, [2], 1, 1), (1, 3, 2, 128, 16, [100, 48, 49], 48, 7), (2, 2, 2, 64, 32, [333, 40], 100, 100),
    (2, 3, 1, 128, 128, [700, 0, 513], 257, 1), (1, 2, 3, 128, 64, [1000, 999], 500, 250), (3, 2, 2, 64, 64, [600, 601], 599, 30),
    (1, 2, 1, 128, 8, [3000, 2999], 1030, 64), (1, 1, 1, 64, 128, [13000], 4000, 500), (1, 2, 2, 128, 32, [2049, 2048], 2048, 0),
    (1, 1, 1, 64, 128, [50000], 300, 20), (1, 40, 8, 64, 128, [12700] + [9, 130, 600] * 13, 100, 30)])
def test_evict_matches_oracle(cuda, kind, L, B, KV, D, page, ctx, keep, recent):
    import specq
    g = torch.Generator(device="cuda").manual_seed(keep + page)
    C = -(-max(ctx) // page) + 1
    P = B * C + 3
    kc, vc, ks, vs = _cache(P, page, KV, D, kind, g, (L,))
    tbl = _table(B, C, P, g)
    mass = torch.rand(L, B, KV, C * page + 3, generator=g, device="cuda") ** 6
    mass[torch.rand(mass.shape, generator=g, device="cuda") < 0.1] = 0.0            # ties
    mass[torch.rand(mass.shape, generator=g, device="cuda") < 0.05] = 0.25
    before = [x.clone() for x in (kc, vc, ks, vs, mass)]
    out = specq.kv_evict_blocks(kc, vc, ks, vs, tbl, _i32(ctx), mass, keep, recent)
    _check_evict(before, (kc, vc, ks, vs, mass), tbl, ctx, keep, recent, kind, out)


@pytest.mark.parametrize("fill", ["zero", "falling", "rising", "strange"])
def test_evict_masses(cuda, fill):
    """All masses alike, in order, NaN, infinities, negative."""
    import specq
    g = torch.Generator(device="cuda").manual_seed(7)
    B, KV, D, page, ctx, keep, recent = 2, 2, 64, 16, [300, 170], 90, 11
    kc, vc, ks, vs = _cache(60, page, KV, D, torch.int8, g)
    tbl = _table(B, 20, 60, g)
    t = torch.arange(320, device="cuda").float().expand(B, KV, -1)
    mass = dict(zero=torch.zeros(B, KV, 320, device="cuda"), falling=(-t).clone(), rising=t.clone(), strange=torch.randn(B, KV, 320, generator=g, device="cuda"))[fill]
    if fill == "strange":
        for i, v in enumerate((float("nan"), float("inf"), -float("inf"), -0.0, 0.0)):
            mass[:, :, i::9] = v
    before = [x.clone()[None] for x in (kc, vc, ks, vs, mass)]
    ctx_t = _i32(ctx)
    out = specq.kv_evict_blocks(kc, vc, ks, vs, tbl, ctx_t, mass, keep, recent, ctx_out=ctx_t)
    assert out is ctx_t
    _check_evict(before, [x[None] for x in (kc, vc, ks, vs, mass)], tbl, ctx, keep, recent, torch.int8, out)


def test_evict_leaves_rows_alone(cuda):
    """Short rows, shared pages (with the pool's counts), pages outside the cache, a context past its table."""
    import specq
    g = torch.Generator(device="cuda").manual_seed(8)
    kc, vc, ks, vs = cache = _cache(40, 16, 2, 64, torch.int8, g)
    tbl = _table(6, 6, 40, g)
    tbl[1, 2] = tbl[0, 1]                              # rows 0 and 1 share a page
    tbl[3, 0], tbl[4, 1] = -1, 40
    ref = torch.zeros(40, dtype=torch.int32, device="cuda")
    for p in tbl.flatten().tolist():
        if 0 <= p < 40:
            ref[p] += 1
    mass = torch.rand(6, 2, 96, generator=g, device="cuda")
    ctx = [90, 80, 70, 60, 60, 97]
    before = [x.clone() for x in (*cache, mass)]
    specq.get_status()
    out = specq.kv_evict_blocks(*cache, tbl, _i32(ctx), mass, 30, 10, ref=ref)
    assert specq.get_status() == specq._lib.SPECQ_STATUS_BAD_INDEX
    assert out.tolist() == [90, 80, 30, 60, 60, 97]
    after = [x.clone() for x in (*cache, mass)]
    only = [0, 0, 70, 0, 0, 0]
    _check_evict([x[None] for x in before], [x[None] for x in after], tbl, only, 30, 10, torch.int8, _i32([0, 0, 30, 0, 0, 0]))
    out = specq.kv_evict_blocks(*cache, tbl[2:3], _i32([90]), mass[2:3], (1 << 31) - 1, (1 << 31) - 1)   # no budget at all
    assert out.tolist() == [90]
    out = specq.kv_evict_blocks(*cache, tbl, _i32([20, 30, 30, 8, 0, 1]), mass, 30, 10, ref=ref)       # nothing to cut
    assert out.tolist() == [20, 30, 30, 8, 0, 1] and specq.get_status() == 0
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(after, (*cache, mass)))


def test_evict_strided_cache_and_graph(cuda):
    """Heads first in a page, layers as views; captured and replayed on other lengths and masses."""
    import specq
    g = torch.Generator(device="cuda").manual_seed(9)
    L, P, page, KV, D, B = 2, 30, 16, 2, 64, 2
    kc, vc, ks, vs = _cache(P, KV, page, D, torch.float8_e4m3fn, g, (L,))           # [L, P, KV, page, D]
    kc, vc = kc.transpose(2, 3), vc.transpose(2, 3)
    ks, vs = (torch.rand(L, P, KV, generator=g, device="cuda") + 0.5 for _ in range(2))
    tbl = _table(B, 12, P, g)
    mass, ctx = torch.rand(L, B, KV, 192, generator=g, device="cuda"), _i32([30, 30])
    out = torch.zeros(B, dtype=torch.int32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    specq.kv_evict_blocks(kc, vc, ks, vs, tbl, ctx, mass, 40, 8)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        specq.kv_evict_blocks(kc, vc, ks, vs, tbl, ctx, mass, 40, 8, ctx_out=out)
    ctx.copy_(_i32([190, 64]))
    before = [x.clone() for x in (kc, vc, ks, vs, mass)]
    graph.replay()
    torch.cuda.synchronize()
    _check_evict(before, (kc, vc, ks, vs, mass), tbl, [190, 64], 40, 8, torch.float8_e4m3fn, out)


def test_release_of_tails(cuda):
    import specq
    ref = torch.zeros(32, dtype=torch.int32, device="cuda")
    tbl = torch.full((5, 6), -1, dtype=torch.int32, device="cuda")
    held = torch.zeros(5, dtype=torch.int32, device="cuda")
    specq.pages_reserve(ref, tbl, held, _i32([96, 40, 16, 0, 90]), 16)
    want_tbl, want_held, want_ref = tbl.clone(), held.clone(), ref.clone()
    drop = torch.tensor([1, 1, 0, 1, 1], dtype=torch.bool, device="cuda")
    specq.pages_release(ref, tbl, held, drop, _i32([17, 200, 0, 5, -2]), 16)
    for r, n in ((0, 2), (4, 0)):
        for c in range(n, int(want_held[r])):
            want_ref[want_tbl[r, c]] -= 1
            want_tbl[r, c] = -1
        want_held[r] = n
    assert torch.equal(tbl, want_tbl) and torch.equal(held, want_held) and torch.equal(ref, want_ref)
    short = specq.pages_reserve(ref, tbl, held, _i32([96, 0, 0, 0, 0]), 16)           # they are free again
    assert short.item() == 0 and held[0] == 6


def test_append_and_attend_after_eviction(cuda):
    """A row cut down goes on: new tokens at its places with their own positions, attention over what is kept."""
    import specq
    g = torch.Generator(device="cuda").manual_seed(10)
    page, KV, H, D, n, keep = 16, 2, 4, 64, 100, 40
    kc, vc, ks, vs = cache = _cache(12, page, KV, D, torch.int8, g)
    tbl = _table(1, 8, 12, g)
    mass = torch.rand(1, KV, 128, generator=g, device="cuda")
    ctx = specq.kv_evict_blocks(*cache, tbl, _i32([n]), mass, keep, 10)
    k, v, q = (torch.randn(1, h, D, generator=g, device="cuda").half() for h in (KV, KV, H))
    table = specq.rope_table(256, D, device="cuda")
    ctx = ctx + 1
    q2 = specq.kv_append_blocks(k, v, *cache, tbl, ctx, 1, q=q, table=table, pos=_i32([n]))
    out = specq.paged_attention_blocks(q2, *cache, tbl, ctx, q_len=1)
    rows = tbl[0, :3].long()
    kk = (kc[rows].double() * ks[rows].double()[:, None, :, None]).flatten(0, 1)[: keep + 1].repeat_interleave(H // KV, 1)
    vv = (vc[rows].double() * vs[rows].double()[:, None, :, None]).flatten(0, 1)[: keep + 1].repeat_interleave(H // KV, 1)
    w = torch.softmax(torch.einsum("hd,thd->ht", q2[0].double(), kk) * D ** -0.5, -1)
    # weights and output in fp16
    assert (out[0].double() - torch.einsum("ht,thd->hd", w, vv)).abs().max() <= 3 * 2.0 ** -11 * vv.abs().max()
    m = specq.attention_mass_blocks(q2[None], kc, ks, tbl, ctx, mass.clone())
    got = (m - mass)[0, :, : keep + 1].double()
    assert (got - w.view(KV, H // KV, -1).sum(1)).abs().max() <= 1e-5 and torch.equal(m[0, :, keep + 1:], mass[0, :, keep + 1:])
