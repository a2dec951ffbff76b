"""qk_norm_rope and its gradients against the float64 oracle.

Bounds, with e = 2^-24 (fp32) and D elements a head.  The sum of squares loses at most D e of itself, so r loses
(D / 2 + 2) e of itself; with the products, the weight and the turn (three roundings of a pair) an output is off by
at most (D / 2 + 8) e times the pair's size, and half a unit of its type.  dx adds a dot product of D terms: (D + 20) e
times r (|u w| + |xh| mean |u w xh|), |u| being the pair's size.  dw sums T H terms: (T H + D + 20) e of the sum of
their magnitudes."""
import numpy as np
import pytest
import torch

from oracle import bounded_oracle as O
from oracle import block_oracle as BO

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 1e-38, torch.float32: 1e-38}
DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def _np(t):
    return t.detach().double().cpu().numpy()


def _pair(v, rot, layout):
    """Each element's pair size |a| + |b| (of the tail: |a|)."""
    v = np.abs(v)
    out, h = v.copy(), rot // 2
    if layout == "half":
        out[..., :h] = out[..., h:rot] = v[..., :h] + v[..., h:rot]
    else:
        out[..., 0:rot:2] = out[..., 1:rot:2] = v[..., 0:rot:2] + v[..., 1:rot:2]
    return out


def _check_forward(out, x, w, table, pos, layout, eps):
    dt, rot = out.dtype, table.shape[1]
    xs, ws = _np(x), None if w is None else _np(w)
    ref = O.norm_turn(xs, ws, table.cpu().numpy(), pos.cpu().numpy(), layout, eps)
    D = xs.shape[-1]
    y = xs / np.sqrt((xs * xs).mean(-1, keepdims=True) + eps) * (1 if ws is None else ws)
    bound = UNIT[dt] * np.abs(ref) + (D / 2 + 8) * E * (1 + UNIT[dt]) * _pair(y, rot, layout) + TINY[dt]
    err = np.abs(_np(out) - ref)
    assert (err <= bound).all(), (err / bound).max()


def _check_grad(dx, dw, x, w, g, table, pos, layout, eps):
    rot = table.shape[1]
    xs, ws, gs = _np(x), None if w is None else _np(w), _np(g)
    t, p = table.cpu().numpy(), pos.cpu().numpy()
    rx, rw = O.norm_turn_grad(xs, ws, gs, t, p, layout, eps)
    T, H, D = xs.shape
    r = 1 / np.sqrt((xs * xs).mean(-1, keepdims=True) + eps)
    u, hat = _pair(gs, rot, layout), np.abs(xs * r)          # |u| is at most its pair's size
    uw = u if ws is None else u * np.abs(ws)
    if dx is not None:
        bound = UNIT[dx.dtype] * np.abs(rx) + (D + 20) * E * r * (uw + hat * (uw * hat).mean(-1, keepdims=True)) + TINY[dx.dtype]
        err = np.abs(_np(dx) - rx)
        assert (err <= bound).all(), (err / bound).max()
    if dw is not None:
        bound = UNIT[dw.dtype] * np.abs(rw) + (T * H + D + 20) * E * (u * hat).sum((0, 1)) + TINY[dw.dtype]
        err = np.abs(_np(dw) - rw)
        assert (err <= bound).all(), (err / bound).max()


def _make(T, H, KV, D, rot, dtype, seed=0, weights="same", n_pos=300):
    import specq
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def r(*s):
        return torch.randn(*s, generator=gen, device="cuda")
    q, k = r(T, H, D).to(dtype), (2 * r(T, KV, D)).to(dtype)
    wt = torch.float32 if weights == "fp32" else dtype
    qw, kw = (None, None) if weights is None else ((1 + 0.3 * r(D)).to(wt), (0.5 + 0.3 * r(D)).to(wt))
    pos = torch.randint(0, n_pos, (T,), generator=gen, device="cuda", dtype=torch.int32)
    return q, k, qw, kw, pos, specq.rope_table(n_pos, rot, device="cuda"), r


SHAPES = [(1, 1, 1, 128, 128), (1, 32, 8, 128, 128), (7, 5, 2, 64, 64), (33, 6, 3, 128, 64), (5, 3, 1, 256, 256), (9, 2, 2, 512, 256),
          (4, 3, 1, 96, 96), (6, 2, 1, 80, 48), (3, 1, 1, 10, 6), (2, 2, 1, 33, 32), (2, 1, 1, 2048, 2048), (700, 32, 8, 64, 64),
          (301, 7, 3, 128, 128)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("T,H,KV,D,rot", SHAPES)
def test_forward_matches_oracle(cuda, dtype, layout, T, H, KV, D, rot):
    import specq
    for weights in ("same", "fp32", None) if D <= 128 else ("same",):
        q, k, qw, kw, pos, table, _ = _make(T, H, KV, D, rot, dtype, T + D, weights)
        a, b = specq.qk_norm_rope(q, k, qw, kw, pos, table, eps=1e-5, layout=layout)
        _check_forward(a, q, qw, table, pos, layout, 1e-5)
        _check_forward(b, k, kw, table, pos, layout, 1e-5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("T,H,KV,D,rot", SHAPES)
def test_gradients_match_oracle(cuda, dtype, layout, T, H, KV, D, rot):
    import specq
    for weights in ("same", "fp32", None) if D == 64 else ("same",):
        q, k, qw, kw, pos, table, r = _make(T, H, KV, D, rot, dtype, T + D + 1, weights)
        gq, gk = r(T, H, D).to(dtype), r(T, KV, D).to(dtype)
        leaves = [t for t in (q, k, qw, kw) if t is not None]
        for t in leaves:
            t.requires_grad_(True)
        a, b = specq.qk_norm_rope(q, k, qw, kw, pos, table, eps=1e-5, layout=layout)
        got = list(torch.autograd.grad((a, b), leaves, (gq, gk)))
        dqw, dkw = (got[2], got[3]) if weights is not None else (None, None)
        assert got[0].dtype == dtype and (weights is None or dqw.dtype == qw.dtype)
        _check_grad(got[0], dqw, q, qw, gq, table, pos, layout, 1e-5)
        _check_grad(got[1], dkw, k, kw, gk, table, pos, layout, 1e-5)
        again = torch.autograd.grad(specq.qk_norm_rope(q, k, qw, kw, pos, table, eps=1e-5, layout=layout), leaves, (gq, gk))
        assert all(torch.equal(x, y) for x, y in zip(got, again))          # the same bits


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_gradient_is_the_difference(cuda, layout):
    """Central differences of <g, y> along random directions, fp32 with step 2^-6: the quotient of a sum of n = T H D
    outputs of size about 1 has an error of n^(1/2) 2^-24 / h from rounding (20 of them allowed) and h^2 times a third derivative of
    at most some 10 sum |g|."""
    import specq
    T, H, KV, D, rot, h = 5, 3, 2, 64, 48, 2.0 ** -6
    q, k, qw, kw, pos, table, r = _make(T, H, KV, D, rot, torch.float32, 3)
    gq, gk = r(T, H, D), r(T, KV, D)

    def f(ts):
        a, b = specq.qk_norm_rope(*ts, pos, table, layout=layout)
        return (gq.double() * a.double()).sum() + (gk.double() * b.double()).sum()
    leaves = [t.clone().requires_grad_(True) for t in (q, k, qw, kw)]
    grads = torch.autograd.grad(specq.qk_norm_rope(*leaves, pos, table, layout=layout), leaves, (gq, gk))
    size = float(gq.abs().sum() + gk.abs().sum())
    for _ in range(6):
        ds = [r(*t.shape) / t.numel() ** 0.5 for t in (q, k, qw, kw)]
        diff = (f([t + h * d for t, d in zip((q, k, qw, kw), ds)]) - f([t - h * d for t, d in zip((q, k, qw, kw), ds)])) / (2 * h)
        dot = sum((g.double() * d.double()).sum() for g, d in zip(grads, ds))
        n = (T * (H + KV) * D) ** 0.5
        assert abs(float(diff - dot)) <= 20 * n * E / h + h * h * 10 * size / n


@pytest.mark.parametrize("offset,gap", [(0, 64), (1, 0), (3, 5), (8, 8)])
def test_strided_rows_and_in_place(cuda, offset, gap):
    """Heads of a packed projection row, aligned or not, in place; nothing beside them moves."""
    import specq
    T, H, KV, D = 19, 6, 2, 64
    table = specq.rope_table(100, D, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(3)
    rows = torch.randn(T, offset + (H + 2 * KV) * D + gap, generator=gen, device="cuda").half()
    before = rows.clone()
    w = torch.rand(D, generator=gen, device="cuda").half() + 0.5
    pos = torch.arange(T, dtype=torch.int32, device="cuda")
    q = rows[:, offset: offset + H * D].unflatten(1, (H, D))
    k = rows[:, offset + H * D: offset + (H + KV) * D].unflatten(1, (KV, D))
    ref = specq.qk_norm_rope(q.contiguous(), k.contiguous(), w, w, pos, table)
    _check_forward(ref[0], q, w, table, pos, "half", 1e-6)
    got = specq.qk_norm_rope(q, k, w, w, pos, table, q_out=q, k_out=k)
    # an unaligned row takes another kernel, whose sums have another order
    assert got[0] is q and got[1] is k
    _check_forward(got[0], before[:, offset: offset + H * D].unflatten(1, (H, D)), w, table, pos, "half", 1e-6)
    _check_forward(got[1], before[:, offset + H * D: offset + (H + KV) * D].unflatten(1, (KV, D)), w, table, pos, "half", 1e-6)
    assert torch.equal(rows[:, :offset], before[:, :offset])
    assert torch.equal(rows[:, offset + (H + KV) * D:], before[:, offset + (H + KV) * D:])


def test_strided_and_broadcast_gradients(cuda):
    """Inputs expanded over heads get the sum of the heads' gradients; gradients of any strides are read."""
    import specq
    T, H, D = 11, 4, 64
    q1, _, qw, kw, pos, table, r = _make(T, 1, 1, D, D, torch.float32, 5)
    gq, gk = r(T, D, H).transpose(1, 2), r(1, 1, D).expand(T, H, D)
    q1.requires_grad_(True)
    a, b = specq.qk_norm_rope(q1.expand(T, H, D), q1.expand(T, H, D), qw, kw, pos, table)
    (got,) = torch.autograd.grad((a, b), (q1,), (gq, gk))
    full = q1.detach().expand(T, H, D).contiguous()
    t, p = table.cpu().numpy(), pos.cpu().numpy()
    ref = sum(O.norm_turn_grad(_np(full), _np(w), _np(g), t, p, "half", 1e-6)[0] for w, g in ((qw, gq), (kw, gk))).sum(1, keepdims=True)
    size = sum(np.abs(_np(g)).sum(1, keepdims=True).max() for g in (gq, gk)) * 8
    assert np.abs(_np(got) - ref).max() <= (D + 40) * E * size * float(1 / q1.detach().square().mean(-1).sqrt().min())


def test_only_the_wanted_gradients(cuda):
    import specq
    q, k, qw, kw, pos, table, r = _make(9, 3, 2, 64, 64, torch.bfloat16, 6)
    gq, gk = r(9, 3, 64).bfloat16(), r(9, 2, 64).bfloat16()
    leaves = (q, k, qw, kw)
    for t in leaves:
        t.requires_grad_(True)
    every = torch.autograd.grad(specq.qk_norm_rope(q, k, qw, kw, pos, table), leaves, (gq, gk))
    for i, t in enumerate(leaves):
        for u in leaves:
            u.requires_grad_(u is t)
        out = specq.qk_norm_rope(q, k, qw, kw, pos, table)
        (one,) = torch.autograd.grad([o for o in out if o.requires_grad], (t,), (gq, gk))
        assert torch.equal(one, every[i])
    for u in leaves:                                  # one output used
        u.requires_grad_(True)
    a, _ = specq.qk_norm_rope(q, k, qw, kw, pos, table)
    got = torch.autograd.grad(a, leaves, gq)
    assert torch.equal(got[0], every[0]) and torch.equal(got[2], every[2]) and not got[1].any() and not got[3].any()
    with torch.no_grad():
        assert not specq.qk_norm_rope(q, k, qw, kw, pos, table)[0].requires_grad


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_large_and_small_rows(cuda, dtype):
    """A row whose squares leave fp32, a row of zeros, one far below eps, beside an ordinary one; the rows do not
    touch one another, a NaN or an infinity stays in its head."""
    import specq
    for D in (64, 20):
        q, k, qw, kw, pos, table, r = _make(8, 2, 1, D, D, dtype, 7)
        for row, s in ((0, 2.0 ** 62), (1, 2.0 ** 100), (2, 0.0), (3, 2.0 ** -60), (4, 2.0 ** 64)):
            q[row] *= s
        q[5, 0, 3], q[6, 1, 0] = float("nan"), float("inf")
        for fn in ("forward", "grad"):
            if fn == "forward":
                a, _ = specq.qk_norm_rope(q, k, qw, kw, pos, table)
                _check_forward(a[:5], q[:5], qw, table, pos[:5], "half", 1e-6)
                _check_forward(a[5:7, :, :][[0, 1], [1, 0]][:, None], q[5:7][[0, 1], [1, 0]][:, None], qw, table, pos[5:7], "half", 1e-6)
                assert a[5, 0].isnan().any() and a[6, 1].isnan().any()
            else:
                x = q[:5].clone().requires_grad_(True)
                g = r(5, 2, D).to(dtype)
                (dx,) = torch.autograd.grad(specq.qk_norm_rope(x, k[:5], qw, kw, pos[:5], table)[0], x, g)
                _check_grad(dx, None, x, qw, g, table, pos[:5], "half", 1e-6)


def test_differentiable_once(cuda):
    """A graph of the gradients is no zero but an error, where it is used."""
    import specq
    q, k, qw, kw, pos, table, r = _make(5, 2, 1, 64, 64, torch.float32, 12)
    q.requires_grad_(True)
    a, _ = specq.qk_norm_rope(q, k, qw, kw, pos, table)
    g = r(5, 2, 64)
    (plain,) = torch.autograd.grad(a, q, g, retain_graph=True)
    (dq,) = torch.autograd.grad(a, q, g, create_graph=True)
    assert torch.equal(plain, dq)
    with pytest.raises(RuntimeError, match="differentiable once"):
        dq.sum().backward()


def test_inputs_changed_before_backward_are_an_error(cuda):
    import specq
    q, k, qw, kw, pos, table, r = _make(5, 2, 1, 64, 64, torch.float32, 13)
    qw.requires_grad_(True)
    a, _ = specq.qk_norm_rope(q, k, qw, kw, pos, table)
    q.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(a, qw, r(5, 2, 64))


def test_plan_and_empty_calls(cuda):
    import specq
    q, k, qw, kw, pos, table, r = _make(12, 3, 2, 64, 64, torch.float16, 8)
    plan = torch.tensor([7], dtype=torch.int32, device="cuda")
    full = specq.qk_norm_rope(q, k, qw, kw, pos, table)
    part = specq.qk_norm_rope(q, k, qw, kw, pos, table, plan=plan)
    for f, p in zip(full, part):
        assert torch.equal(p[:7], f[:7]) and not p[7:].any()
    qo, ko = torch.full_like(q, 5), torch.full_like(k, 6)
    specq.qk_norm_rope(q, k, qw, kw, pos, table, q_out=qo, k_out=ko, plan=plan)
    assert torch.equal(qo[:7], full[0][:7]) and (qo[7:] == 5).all() and torch.equal(ko[:7], full[1][:7]) and (ko[7:] == 6).all()
    leaves = (q, k, qw, kw)
    for t in leaves:
        t.requires_grad_(True)
    gq, gk = r(12, 3, 64).half(), r(12, 2, 64).half()
    got = torch.autograd.grad(specq.qk_norm_rope(q, k, qw, kw, pos, table, plan=plan), leaves, (gq, gk))
    x, y = q[:7].detach().requires_grad_(True), k[:7].detach().requires_grad_(True)
    ref = torch.autograd.grad(specq.qk_norm_rope(x, y, qw, kw, pos[:7], table), (x, y, qw, kw), (gq[:7], gk[:7]))
    assert torch.equal(got[0][:7], ref[0]) and not got[0][7:].any() and torch.equal(got[1][:7], ref[1]) and not got[1][7:].any()
    _check_grad(None, got[2], x, qw, gq[:7], table, pos[:7], "half", 1e-6)
    # no rows, no heads: weights get zeros
    e = torch.empty(0, 3, 64, dtype=torch.float16, device="cuda").requires_grad_(True)
    f = torch.empty(0, 2, 64, dtype=torch.float16, device="cuda")
    a, b = specq.qk_norm_rope(e, f, qw, kw, pos[:0], table)
    d = torch.autograd.grad((a, b), (e, qw, kw), (a.detach(), b.detach()))
    assert d[0].shape == e.shape and not d[1].any() and not d[2].any()
    none = torch.empty(12, 0, 64, dtype=torch.float16, device="cuda")
    a, b = specq.qk_norm_rope(q, none, qw, kw, pos, table)
    assert torch.equal(a, full[0]) and b.shape == (12, 0, 64)


def test_positions_outside_the_table_are_clamped(cuda):
    import specq
    q, k, qw, kw, _, table, _ = _make(3, 2, 1, 64, 64, torch.float16, 9, n_pos=50)
    specq.get_status()
    pos = torch.tensor([-4, 7, 50], dtype=torch.int32, device="cuda")
    got = specq.qk_norm_rope(q, k, qw, kw, pos, table)
    assert specq.get_status() == specq._lib.SPECQ_STATUS_PLAN_CLAMPED
    ref = specq.qk_norm_rope(q, k, qw, kw, pos.clamp(0, 49), table)
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])


def test_streams_and_graphs(cuda):
    """On another stream, and forward and backward captured and replayed on new inputs."""
    import specq
    q, k, qw, kw, pos, table, r = _make(40, 4, 2, 128, 128, torch.bfloat16, 10)
    gq, gk = r(40, 4, 128).bfloat16(), r(40, 2, 128).bfloat16()

    def step(q, k, qw, kw):
        a, b = specq.qk_norm_rope(q, k, qw, kw, pos, table)
        return (a, b, *torch.autograd.grad((a, b), (q, k, qw, kw), (gq, gk)))
    leaves = [t.requires_grad_(True) for t in (q, k, qw, kw)]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = step(*leaves)
    side.synchronize()
    ref = step(*leaves)
    assert all(torch.equal(x, y) for x, y in zip(got, ref))
    del got, ref
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(*leaves)
    with torch.no_grad():
        q.copy_(r(40, 4, 128))
        kw.mul_(1.5)
    graph.replay()
    torch.cuda.synchronize()
    got = [t.detach().clone() for t in held]
    assert all(torch.equal(x, y) for x, y in zip(got, step(*leaves)))


def test_appended_keys_need_no_table(cuda):
    """Normalised and turned rows go to the cache and to attention as they are."""
    import specq
    B, Q, H, KV, D, page = 3, 5, 8, 2, 64, 16
    q, k, qw, kw, _, table, r = _make(B * Q, H, KV, D, D, torch.float16, 11)
    v = r(B * Q, KV, D).half()
    ctx = torch.full((B,), Q, dtype=torch.int32, device="cuda")
    pos = torch.arange(Q, dtype=torch.int32, device="cuda").repeat(B)
    tbl = torch.arange(B * 2, dtype=torch.int32, device="cuda").view(B, 2)
    cache = [torch.zeros(6, page, KV, D, dtype=torch.int8, device="cuda") for _ in range(2)] + [torch.ones(6, KV, device="cuda") for _ in range(2)]
    q2, k2 = specq.qk_norm_rope(q, k, qw, kw, pos, table)
    specq.kv_append_blocks(k2, v, *cache, tbl, ctx, Q)
    stored = (cache[0][tbl[:, 0].long()].float() * cache[2][tbl[:, 0].long()][:, None, :, None])[:, :Q]
    # half a step of the page's scale, and what the division by it loses
    step = cache[2][tbl[:, 0].long()][:, None, :, None]
    assert ((stored - k2.view(B, Q, KV, D).float()).abs() <= 0.5001 * step).all()
    out = specq.paged_attention_blocks(q2, *cache, tbl, ctx, q_len=Q)
    assert out.shape == q2.shape and out.isfinite().all()


def test_other_device_is_refused(cuda):
    import specq
    q, k, qw, kw, pos, table, _ = _make(2, 1, 1, 64, 64, torch.float16)
    for i in range(6):
        a = [q, k, qw, kw, pos, table]
        a[i] = a[i].cpu()
        with pytest.raises(ValueError, match="CUDA"):
            specq.qk_norm_rope(*a)


def test_oracle_turn_is_the_pair_formula():
    assert BO.turn(np.ones((1, 1, 2)), np.array([[0.0, 1.0]], np.float32), np.array([0]), "half").tolist() == [[[-1.0, 1.0]]]
