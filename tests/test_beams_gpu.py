"""beam_select and beam_reorder against the float64 oracle.

A total is a score plus a logit less lse.  lse is off by at most 2e-6: ex2 and the product before it lose 2^-21 of a
term, sums of eight 2^-21, and for logits whose difference fp32 rounds, |d| 2^-24 of a term, whose weighted mean is at most ln V
2^-24.  The order of two candidates of different beams is asked for where their totals differ by more than 4e-6; of one beam
always."""
import numpy as np
import pytest
import torch

from oracle import bounded_oracle as O

pytestmark = pytest.mark.gpu

LSE = 2e-6
FLOATS = [torch.float16, torch.bfloat16, torch.float32]


def _check(got, logits, scores, n, done=None, pad=0):
    s, p, t = (x.cpu().numpy() for x in got)
    B, K = scores.shape
    V = logits.shape[1]
    x, sc = logits.float().cpu().numpy(), scores.cpu().numpy()
    dn = None if done is None else done.cpu().numpy()
    rs, rp, rt = O.beam_select(x, sc, n, dn, pad)
    total = O.beam_totals(x, sc, dn, pad)
    none = rs == -np.inf
    assert ((s == -np.inf) == none).all()
    assert (p[none] == rp[none]).all() and (t[none] == pad).all()
    with np.errstate(invalid="ignore"):
        tol = LSE + 2.0 ** -23 * np.abs(rs)
        assert (none | (np.abs(s - rs) <= tol)).all(), np.nanmax(np.abs(s - rs)[~none])
    for b in range(B):
        flat = (p[b].astype(np.int64) - b * K) * V + t[b]
        live = ~none[b]
        assert ((p[b] >= b * K) & (p[b] < (b + 1) * K)).all() and len(set(flat[live].tolist())) == live.sum()
        mine = total[b][flat[live]]                       # the chosen ones' totals are the best ones', in order
        assert (np.abs(mine - rs[b][live]) <= LSE * 2).all()
        same = flat[live] == (rp[b][live] - b * K) * V + rt[b][live]
        for j in np.nonzero(~same)[0]:                    # another candidate only where two beams' totals all but meet
            near = np.abs(total[b] - rs[b][live][j]) <= LSE * 2
            assert len({int(f) // V for f in np.nonzero(near)[0]}) > 1, (b, j)


def _rows(B, K, V, dtype, seed, spread=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return ((torch.randn(B * K, V, generator=g, device="cuda") * spread).to(dtype), -torch.rand(B, K, generator=g, device="cuda") * 10)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("B,K,V,n", [(1, 1, 1, 1), (2, 3, 50, 1), (3, 64, 4, 1), (1, 8, 362, 16), (4, 2, 1299, 4), (1, 3, 25785, 6), (2, 16, 200, 32), (1, 1, 5, 8), (1, 4, 32000, 4), (3, 5, 999, 10), (2, 8, 50257, 16), (2, 3, 16384, 6),
                                     (2, 2, 16385, 128), (5, 64, 333, 128), (1, 64, 20001, 64), (40, 4, 17000, 8), (1, 2, 200003, 4)])
def test_select_matches_oracle(cuda, dtype, B, K, V, n):
    import specq
    x, s = _rows(B, K, V, dtype, B + V)
    _check(specq.beam_select(x, s, n=n), x, s, n)
    if n == K:
        _check(specq.beam_select(x, s.view(-1), beams=K), x, s, n)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("gap", [0, 1, 3, 8])
def test_select_row_strides(cuda, dtype, gap):
    """Rows that begin anywhere in a 16-byte piece: nothing outside the row counts."""
    import specq
    B, K, V = 2, 3, 5003
    g = torch.Generator(device="cuda").manual_seed(gap)
    wide = torch.full((B * K, V + gap + 2), 60.0, device="cuda").to(dtype)
    x = wide[:, 1: V + 1]
    x.copy_(torch.randn(B * K, V, generator=g, device="cuda"))
    s = -torch.rand(B, K, generator=g, device="cuda")
    _check(specq.beam_select(x, s, n=7), x, s, 7)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("V", [300, 40000])
def test_select_ties(cuda, dtype, V):
    """Constant rows, two levels, all masked by the type's lowest number, masked by -inf but for a few."""
    import specq
    K, n = 8, 16
    x, s = _rows(1, K, V, dtype, 3)
    s[:] = -2.0
    x[0] = 1.5
    x[1] = torch.where(torch.arange(V, device="cuda") % 3 == 1, 2.0, -1.0)
    x[2] = torch.finfo(dtype).min
    x[2, V - 3:] = 4.0
    x[3] = -torch.inf
    x[3, [7, V // 2]] = 0.25
    x[4] = -torch.inf
    x[5] = x[0]                                    # a beam like another: equal totals, the lower beam first
    x[6] = 0.0
    x[6, ::2] = -0.0                               # one value
    x[7] = torch.finfo(dtype).min
    for order in (range(8), (2, 7, 2, 7, 2, 7, 2, 7), (0, 5, 0, 5, 0, 5, 0, 5), (4, 4, 4, 4, 4, 4, 3, 4), (6, 6, 6, 6, 6, 6, 6, 6)):
        y = x[list(order)]
        got = specq.beam_select(y, s, n=n, pad=2)
        _check(got, y, s, n, pad=2)
        rs, rp, rt = O.beam_select(y.float().cpu().numpy(), s.cpu().numpy(), n, None, 2)
        if len(set(order)) <= 2:                   # exact ties alone: every index is that of the definition
            assert (got[1].cpu().numpy() == rp).all() and (got[2].cpu().numpy() == rt).all()


def test_select_masks_and_strange_values(cuda):
    import specq
    V, K = 1000, 4
    x, s = _rows(2, K, V, torch.float32, 4)
    x[0, 5], x[0, 6] = float("nan"), float("inf")
    x[1, :] = float("nan")
    x[2, 10:] = -torch.inf
    s[1, 0], s[1, 1], s[1, 2] = -torch.inf, float("nan"), float("inf")
    _check(specq.beam_select(x, s, n=8), x, s, 8)
    got = specq.beam_select(x, s, n=8)
    assert got[2][0, 0] == 6 or (got[1][0] == 0).sum() <= 1          # +inf takes its whole beam's probability
    s[:] = -torch.inf                              # nothing at all: each place its own row
    out, parent, token = specq.beam_select(x, s, n=8, pad=9)
    assert (out == -torch.inf).all() and (token == 9).all()
    assert parent.tolist() == [[0, 1, 2, 3, 0, 1, 2, 3], [4, 5, 6, 7, 4, 5, 6, 7]]


@pytest.mark.parametrize("V", [40, 30000])
def test_select_finished_beams(cuda, V):
    import specq
    x, s = _rows(3, 4, V, torch.bfloat16, 5)
    done = torch.tensor([[1, 0, 0, 1], [1, 1, 1, 1], [0, 0, 0, 0]], dtype=torch.bool, device="cuda").view(-1)
    s[0, 3] = -torch.inf                           # an empty beam, finished or not, has no candidate
    _check(specq.beam_select(x, s, n=8, done=done, pad=3), x, s, 8, done, 3)
    _check(specq.beam_select(x, s, n=8, done=done.to(torch.uint8), pad=3), x, s, 8, done, 3)
    out, parent, token = specq.beam_select(x, s, done=done, pad=3)
    assert sorted(parent[1].tolist()) == [4, 5, 6, 7] and (token[1] == 3).all() and torch.equal(out[1], s[1].sort(descending=True).values)


def test_select_totals_are_those_of_the_definition(cuda):
    """lse of peaked and flat rows, and of one with a wide spread, to the bound above."""
    import specq
    V = 128001
    for dtype in FLOATS:
        for spread in (0.01, 1.0, 6.0):
            x, s = _rows(1, 4, V, dtype, 6, spread)
            _check(specq.beam_select(x, s, n=32), x, s, 32)


def test_select_streams_graph_and_repeats(cuda):
    import specq
    x, s = _rows(4, 4, 30011, torch.float16, 7)
    ref = specq.beam_select(x, s, n=8)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(ref, specq.beam_select(x, s, n=8)))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = specq.beam_select(x, s, n=8)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(ref, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = specq.beam_select(x, s, n=8)
        s2 = held[0][:, :4].contiguous()
        again = specq.beam_select(x, s2, n=8)
    y, t = _rows(4, 4, 30011, torch.float16, 8)
    x.copy_(y)
    s.copy_(t)
    graph.replay()
    torch.cuda.synchronize()
    _check(held, x, s, 8)
    _check(again, x, s2, 8)


def test_select_no_requests(cuda):
    import specq
    out, parent, token = specq.beam_select(torch.zeros(0, 50, device="cuda"), torch.zeros(0, 4, device="cuda"), n=8)
    assert out.shape == parent.shape == token.shape == (0, 8)


# ---- reorder -----------------------------------------------------------------------------------------
def _states(R, g):
    def i(hi, *s, dtype=torch.int32):
        return torch.randint(0, hi, s, generator=g, device="cuda", dtype=dtype)
    wide = torch.randn(R, 3, 40, generator=g, device="cuda")
    return [i(1000, R, 37), i(2, R).bool(), i(100, R, dtype=torch.int64), torch.randn(R, 5, 7, generator=g, device="cuda").half(),
            wide[:, 1], i(255, R, 3, dtype=torch.uint8), torch.randn(R, 2000, generator=g, device="cuda").bfloat16()[:, 1:1999],
            torch.zeros(R, 0, device="cuda"), wide[:, 2], i(255, R, 6, dtype=torch.uint8)[:, 1:5], torch.randn(R, 9, generator=g, device="cuda").double()]


@pytest.mark.parametrize("B,K", [(1, 1), (1, 2), (3, 4), (2, 5), (4, 8), (2, 13), (2, 16), (2, 31), (1, 33), (2, 64)])
def test_reorder_matches_indexing(cuda, B, K):
    import specq
    R = B * K
    g = torch.Generator(device="cuda").manual_seed(K)
    for trial in range(3):
        states = _states(R, g)
        first = torch.arange(R, device="cuda") // K * K
        if trial == 0:
            parent = first + torch.randint(0, K, (R,), generator=g, device="cuda")
        elif trial == 1:                            # a permutation: a cycle through every row
            parent = first + (torch.arange(R, device="cuda") - first + 1) % K
        else:
            parent = first                          # all from one
        ref = [x[parent].clone() for x in states]
        specq.beam_reorder(states, parent.to(torch.int32).view(B, K))
        for a, b in zip(states, ref):
            assert torch.equal(a, b)


def test_reorder_leaves_the_rest(cuda):
    """Gaps between rows, rows that stay, parents that are none or another request's."""
    import specq
    buf = torch.arange(8 * 10, dtype=torch.int32, device="cuda").view(8, 10)
    before = buf.clone()
    x = buf[:, 2:7]
    specq.get_status()
    parent = torch.tensor([1, -1, -7, 2, 0, 5, 8, 7], dtype=torch.int32, device="cuda")
    specq.beam_reorder([x], parent, beams=4)
    assert specq.get_status() == specq._lib.SPECQ_STATUS_BAD_INDEX
    want = before.clone()
    want[0, 2:7], want[3, 2:7] = before[1, 2:7], before[2, 2:7]
    assert torch.equal(buf, want)
    specq.beam_reorder([], parent, beams=4)
    specq.beam_reorder([x], torch.full((8,), -1, dtype=torch.int32, device="cuda"), beams=4)
    assert torch.equal(buf, want) and specq.get_status() == 0


def test_reorder_many_states(cuda):
    """More states than one launch takes."""
    import specq
    g = torch.Generator(device="cuda").manual_seed(1)
    states = [torch.randn(6, 1 + i % 7, generator=g, device="cuda") for i in range(70)]
    parent = torch.tensor([[2, 0, 0], [5, 4, 3]], dtype=torch.int32, device="cuda")
    ref = [x[parent.view(-1).long()].clone() for x in states]
    specq.beam_reorder(states, parent)
    assert all(torch.equal(a, b) for a, b in zip(states, ref))


def test_reorder_in_a_graph_and_beside_select(cuda):
    """A captured step, replayed: scores, parents and tokens feed the histories and the next step."""
    import specq
    B, K, V, L = 3, 4, 5000, 6
    R = B * K
    g = torch.Generator(device="cuda").manual_seed(2)
    steps = [torch.randn(R, V, generator=g, device="cuda").half() for _ in range(L)]
    x, at = torch.empty_like(steps[0]), torch.zeros(1, dtype=torch.int64, device="cuda")
    scores = torch.full((B, K), -torch.inf, device="cuda")
    history, length = torch.zeros(R, L, dtype=torch.int32, device="cuda"), torch.zeros(R, dtype=torch.int32, device="cuda")

    def step():
        s, parent, token = specq.beam_select(x, scores)
        specq.beam_reorder([history, length], parent)
        history.index_copy_(1, at, token.view(R, 1))
        length.add_(1)
        scores.copy_(s)
    x.copy_(steps[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    scores.fill_(-torch.inf)
    scores[:, 0] = 0
    history.zero_()
    length.zero_()
    ref_s, ref_h = scores.cpu().numpy().astype(np.float64), np.zeros((R, 0), np.int64)
    for i, y in enumerate(steps):
        x.copy_(y)
        at.fill_(i)
        graph.replay()
        s, p, t = O.beam_select(y.float().cpu().numpy(), ref_s.astype(np.float32), K)
        ref_h = np.concatenate([ref_h[p.reshape(-1)], t.reshape(-1, 1)], 1)
        ref_s = scores.cpu().numpy().astype(np.float64)
        assert np.abs(ref_s - s).max() <= LSE + 2.0 ** -23 * np.abs(s).max()
    assert (history.cpu().numpy() == ref_h).all() and (length == L).all()
