"""Rotary positions against the float64 oracle.

Bound of each element: the fp32 products and sum of a pair cost at most 4 * 2^-24 (|a| + |b|)
(three roundings, cosines and sines at most 1), the store half a unit of the row's type."""
import numpy as np
import pytest
import torch

from oracle import block_oracle as BO

pytestmark = pytest.mark.gpu

UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 1e-38, torch.float32: 1e-38}


def _bound(x, ref, rot, dtype):
    size = np.abs(x).max(-1, keepdims=True) * 2
    return UNIT[dtype] * np.abs(ref) + 4 * 2.0 ** -24 * size + TINY[dtype]


def _check(out, x, table, pos, layout, inverse, rot, dtype):
    xs = x.double().cpu().numpy()
    ref = BO.turn(xs, table.cpu().numpy(), pos.cpu().numpy(), layout, inverse)
    err = np.abs(out.double().cpu().numpy() - ref)
    assert (err <= _bound(xs, ref, rot, dtype)).all(), err.max()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("T,H,D,rot", [(1, 1, 128, 128), (1, 40, 128, 128), (7, 3, 64, 32), (33, 5, 96, 80),
                                       (5, 2, 64, 6), (3, 1, 10, 2), (640, 33, 128, 64)])
def test_matches_oracle(cuda, dtype, layout, T, H, D, rot):
    import specq
    g = torch.Generator().manual_seed(T * 1000 + H)
    table = specq.rope_table(512, rot, device="cuda")
    x = torch.randn(T, H, D, generator=g).to(dtype).cuda()
    pos = torch.randint(0, 512, (T,), generator=g, dtype=torch.int32).cuda()
    for inverse in (False, True):
        out = specq.rope(x, pos, table, layout=layout, inverse=inverse)
        _check(out, x, table, pos, layout, inverse, rot, dtype)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("offset,gap", [(0, 64), (1, 0), (3, 5), (8, 8)])
def test_strided_rows_and_in_place(cuda, layout, offset, gap):
    """Heads of a packed projection row, aligned or not, turned in place; nothing beside them moves."""
    import specq
    T, H, D, rot = 19, 6, 64, 64
    table = specq.rope_table(100, rot, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(3)
    rows = torch.randn(T, offset + H * D + gap, generator=g, device="cuda").half()
    before = rows.clone()
    x = rows[:, offset: offset + H * D].unflatten(1, (H, D))
    pos = torch.arange(T, dtype=torch.int32, device="cuda")
    ref = specq.rope(x.contiguous(), pos, table, layout=layout)
    got = specq.rope(x, pos, table, layout=layout, out=x)
    assert got is x and torch.equal(x, ref)
    assert torch.equal(rows[:, :offset], before[:, :offset]) and torch.equal(rows[:, offset + H * D:], before[:, offset + H * D:])
    # heads in another order of strides
    y = before[:, offset: offset + H * D].unflatten(1, (H, D)).transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(specq.rope(y, pos, table, layout=layout), ref)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_inverse_is_the_gradient(cuda, layout):
    """<g, R d> by central differences equals <R^T g, d>; R^T R = 1.  fp32: a sum of n products of size
    about 1 has an error of at most n 2^-23, the difference quotient one of 2^-23 |f| / h more."""
    import specq
    T, H, D, rot = 9, 4, 64, 48
    table = specq.rope_table(64, rot, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(5)
    x, g, d = (torch.randn(T, H, D, generator=gen, device="cuda") for _ in range(3))
    pos = torch.arange(T, dtype=torch.int32, device="cuda") * 7
    h = 0.25

    def f(v):
        return (g.double() * specq.rope(v, pos, table, layout=layout).double()).sum()
    diff = (f(x + h * d) - f(x - h * d)) / (2 * h)
    grad = (specq.rope(g, pos, table, layout=layout, inverse=True).double() * d.double()).sum()
    n = T * H * D
    size = (g.abs() * (x.abs() + d.abs())).sum().item()
    assert abs((diff - grad).item()) <= 8 * 2.0 ** -23 * size / h + n * 2.0 ** -23
    back = specq.rope(specq.rope(x, pos, table, layout=layout), pos, table, layout=layout, inverse=True)
    # two rotations, and cos^2 + sin^2 of fp32 table entries is 1 to 2^-23
    assert ((back - x).abs() <= 16 * 2.0 ** -24 * 2 * x.abs().amax(-1, keepdim=True)).all()


def test_plan_clamps_and_streams(cuda):
    import specq
    T, H, D = 12, 2, 64
    table = specq.rope_table(16, D, device="cuda")
    x = torch.randn(T, H, D, device="cuda")
    pos = torch.arange(T, dtype=torch.int32, device="cuda")
    full = specq.rope(x, pos, table)
    out = torch.full_like(x, 7.0)
    plan = torch.tensor([5], dtype=torch.int32, device="cuda")
    specq.get_status(clear=True)
    specq.rope(x, pos, table, out=out, plan=plan)
    assert torch.equal(out[:5], full[:5]) and (out[5:] == 7.0).all()
    assert specq.get_status(clear=True) == 0
    # positions outside the table are clamped into it and reported
    bad = pos.clone()
    bad[0], bad[1] = -3, 99
    got = specq.rope(x, bad, table)
    torch.cuda.synchronize()
    assert specq.get_status(clear=True) != 0
    ok = pos.clone()
    ok[0], ok[1] = 0, 15
    assert torch.equal(got, specq.rope(x, ok, table))
    # a side stream's own tensors
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = specq.rope(x, pos, table)
    s.synchronize()
    assert torch.equal(y, full)
    assert specq.rope(x[:0], pos[:0], table).shape == (0, H, D)


def test_graph_capture(cuda):
    import specq
    table = specq.rope_table(64, 64, device="cuda")
    x = torch.randn(8, 4, 64, device="cuda").half()
    pos = torch.arange(8, dtype=torch.int32, device="cuda")
    out = torch.empty_like(x)
    specq.rope(x, pos, table, out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        specq.rope(x, pos, table, out=out)
    x.copy_(torch.randn(8, 4, 64, device="cuda"))
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, specq.rope(x, pos, table))
