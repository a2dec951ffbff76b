"""Normalised heads, beams and the bounded cache without a GPU: what is refused before anything is launched, and
the oracle against its own definitions.  (Tensors on the CPU are refused last, with "CUDA" in the message, so a
refusal that names something else comes from the arguments.)"""
import numpy as np
import pytest
import torch

import specq
from oracle import bounded_oracle as O
from specq import _lib

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def _heads(T=4, H=4, KV=2, D=64, dtype=F16):
    return torch.zeros(T, H, D, dtype=dtype), torch.zeros(T, KV, D, dtype=dtype), torch.ones(D, dtype=dtype), torch.ones(D, dtype=dtype)


def _cache(P=6, page=16, KV=2, D=64, dtype=torch.int8, layers=None):
    lead = () if layers is None else (layers,)
    kc = torch.zeros(*lead, P, page, KV, D, dtype=torch.uint8).view(dtype)
    return kc, kc.clone(), torch.ones(*lead, P, KV), torch.ones(*lead, P, KV)


# ---- qk_norm_rope ------------------------------------------------------------------------------------
@pytest.mark.parametrize("change,error,match", [
    (dict(q=torch.zeros(4, 4, 64)), ValueError, "one type"),
    (dict(k=torch.zeros(3, 2, 64, dtype=F16)), ValueError, "as many rows"),
    (dict(k=torch.zeros(4, 2, 32, dtype=F16)), ValueError, "elements a head"),
    (dict(q=torch.zeros(4, 4, 64, dtype=torch.int32)), TypeError, "float16"),
    (dict(q=torch.zeros(4, 256, dtype=F16)), ValueError, "rows, heads, dim"),
    (dict(q=torch.zeros(4, 64, 4, dtype=F16).transpose(1, 2)), ValueError, "unit inner stride"),
    (dict(qw=torch.ones(32, dtype=F16)), ValueError, "weights must be contiguous"),
    (dict(qw=torch.ones(128, dtype=F16)[::2]), ValueError, "weights must be contiguous"),
    (dict(qw=torch.ones(64, dtype=BF16)), TypeError, "weights must be"),
    (dict(qw=torch.ones(64)), TypeError, "of one type"),
    (dict(pos=_i32(3)), ValueError, "pos"),
    (dict(pos=torch.zeros(4, dtype=torch.int64)), TypeError, "pos"),
    (dict(table=torch.zeros(8, 128)), ValueError, "table"),
    (dict(table=torch.zeros(8, 63)), ValueError, "table"),
    (dict(eps=0.0), ValueError, "eps"),
    (dict(eps=-1.0), ValueError, "eps"),
    (dict(eps=1e-60), ValueError, "eps"),
    (dict(eps=float("inf")), ValueError, "eps"),
    (dict(eps=float("nan")), ValueError, "eps"),
    (dict(layout="pairs"), ValueError, "layout"),
    (dict(q_out=torch.zeros(4, 4, 64)), ValueError, "q_out"),
    (dict(q_out=torch.zeros(1, 4, 64, dtype=F16).expand(4, -1, -1)), ValueError, "q_out .*expanded"),
    (dict(k_out=torch.zeros(4, 1, 64, dtype=F16).expand(-1, 2, -1)), ValueError, "k_out .*expanded"),
    (dict(plan=torch.zeros(1)), TypeError, "plan"),
    (dict(plan=_i32(0)), ValueError, "plan"),
    (dict(table=torch.zeros(8, 64, requires_grad=True)), ValueError, "table has no gradient"),
    (dict(), ValueError, "CUDA"),
    (dict(qw=None, kw=None), ValueError, "CUDA"),
    (dict(qw=torch.ones(64), kw=torch.ones(64)), ValueError, "CUDA"),
    (dict(qw=torch.ones(64), kw=None), ValueError, "CUDA"),
])
def test_heads_refusals(change, error, match):
    q, k, qw, kw = _heads()
    a = dict(q=q, k=k, qw=qw, kw=kw, pos=_i32(4), table=torch.zeros(8, 64), eps=1e-6, layout="half", q_out=None, k_out=None, plan=None)
    a.update(change)
    with pytest.raises(error, match=match):
        specq.qk_norm_rope(a["q"], a["k"], a["qw"], a["kw"], a["pos"], a["table"], a["eps"], a["layout"], a["q_out"], a["k_out"], a["plan"])


def test_heads_refuse_an_output_where_a_gradient_is_wanted():
    q, k, qw, kw = _heads()
    for t in (q, k, qw, kw):
        t.requires_grad_(True)
        with pytest.raises(ValueError, match="gradient is wanted"):
            specq.qk_norm_rope(q, k, qw, kw, _i32(4), torch.zeros(8, 64), q_out=torch.zeros(4, 4, 64, dtype=F16))
        with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
            specq.qk_norm_rope(q, k, qw, kw, _i32(4), torch.zeros(8, 64), q_out=torch.zeros(4, 4, 64, dtype=F16))
        with pytest.raises(ValueError, match="CUDA"):
            specq.qk_norm_rope(q, k, qw, kw, _i32(4), torch.zeros(8, 64))
        t.requires_grad_(False)


def _views(shape, *slices):
    x = torch.zeros(shape, dtype=F16)
    return [x[s] for s in slices]


ALL = slice(None)


@pytest.mark.parametrize("names,views,match", [
    ("q q_out", _views((5, 4, 64), slice(0, 4), slice(1, 5)), "q_out may be q"),
    ("k q_out", _views((4, 4, 64), (ALL, slice(0, 2)), ALL), "q_out may be q"),
    ("q k_out", _views((4, 4, 64), ALL, (ALL, slice(1, 3))), "k_out may be k"),
    ("q q_out", _views((4, 4, 96), (ALL, ALL, slice(0, 64)), (ALL, ALL, slice(32, 96))), "q_out may be q"),
    ("q_out k_out", _views((4, 4, 64), ALL, (ALL, slice(2, 4))), "q_out and k_out"),
    # allowed, so that the next refusal is met: the heads of one projection's rows, and heads side by side
    ("q k q_out k_out", _views((4, 8, 64), (ALL, slice(0, 4)), (ALL, slice(4, 6)), (ALL, slice(0, 4)), (ALL, slice(4, 6))), "CUDA"),
    ("q k k_out", _views((4, 8, 64), (ALL, slice(0, 4)), (ALL, slice(4, 6)), (ALL, slice(6, 8))), "CUDA"),
    ("q q_out", _views((4, 4, 2, 64), (ALL, ALL, 0), (ALL, ALL, 1)), "CUDA"),
])
def test_heads_refuse_outputs_over_inputs(names, views, match):
    a = dict(q=torch.zeros(4, 4, 64, dtype=F16), k=torch.zeros(4, 2, 64, dtype=F16), q_out=None, k_out=None)
    a.update(zip(names.split(), views))
    with pytest.raises(ValueError, match=match):
        specq.qk_norm_rope(a["q"], a["k"], None, None, _i32(4), torch.zeros(8, 64), q_out=a["q_out"], k_out=a["k_out"])


def test_heads_library_refuses():
    lib = _lib.load()

    def call(D=64, rot=64, eps=1e-6, layout=0, T=1, q=16, out=16, ot=64, dtype=0):
        return lib.specq_qk_norm_rope(q, 64, 64, out, ot, 64, 16, 64, 64, 32, 64, 64, dtype, None, None, 0, eps, 16, 16, 8, T, 1, 1, D, rot,
                                      layout, None, None)
    assert call(D=4096) == _lib.SPECQ_ERR_UNSUPPORTED
    for bad in (dict(rot=63), dict(rot=66), dict(eps=0.0), dict(eps=float("nan")), dict(layout=2), dict(T=-1), dict(q=None), dict(ot=128),
                dict(dtype=3)):
        assert call(**bad) == _lib.SPECQ_ERR_INVALID_ARG, bad
    assert lib.specq_qk_norm_rope_grad(16, 64, 64, 16, 64, 64, None, 0, 0, 16, 64, 64, 16, 64, 64, None, 0, 0, 0, None, None, 16, None, 0, 1e-6,
                                       16, 16, 8, 1, 1, 1, 64, 64, 0, None, None, 0, None) == _lib.SPECQ_ERR_INVALID_ARG   # dqw without weights


# ---- beams -------------------------------------------------------------------------------------------
@pytest.mark.parametrize("change,error,match", [
    (dict(logits=torch.zeros(4, 10, dtype=torch.float64)), TypeError, "logits"),
    (dict(logits=torch.zeros(40)), ValueError, "logits"),
    (dict(logits=torch.zeros(10, 4).T), ValueError, "unit inner stride"),
    (dict(logits=torch.zeros(1, 10).expand(4, -1)), ValueError, "overlap"),
    (dict(logits=torch.zeros(5, 10)), ValueError, "scores"),
    (dict(scores=torch.zeros(2, 2, dtype=F16)), ValueError, "scores"),
    (dict(scores=torch.zeros(2, 4)[:, ::2]), ValueError, "contiguous"),
    (dict(scores=torch.zeros(4)), ValueError, "give beams"),
    (dict(scores=torch.zeros(4), beams=3), ValueError, "no requests"),
    (dict(beams=4), ValueError, "no requests"),
    (dict(beams=0), ValueError, "no requests"),
    (dict(n=0), ValueError, "n=0"),
    (dict(pad=-1), ValueError, "pad"),
    (dict(pad=10), ValueError, "pad"),
    (dict(done=torch.zeros(4)), ValueError, "done"),
    (dict(done=torch.zeros(3, dtype=torch.bool)), ValueError, "done"),
    (dict(logits=torch.zeros(4, 10, requires_grad=True)), ValueError, "gradient"),
    (dict(logits=torch.zeros(4, 0)), ValueError, "vocabulary"),
    (dict(), ValueError, "CUDA"),
    (dict(scores=torch.zeros(4), beams=2), ValueError, "CUDA"),
])
def test_select_refusals(change, error, match):
    a = dict(logits=torch.zeros(4, 10), scores=torch.zeros(2, 2), n=None, done=None, pad=0, beams=None)
    a.update(change)
    with pytest.raises(error, match=match):
        specq.beam_select(**a)


def test_select_library_refuses():
    lib = _lib.load()

    def call(B=1, K=2, V=10, n=2, pad=0, ld=10, dtype=1):
        return lib.specq_beam_select(16, ld, dtype, 16, None, pad, 16, 16, 16, B, K, V, n, 16, 1 << 20, None)
    for bad in (dict(K=65), dict(n=129), dict(K=64, V=1 << 26), dict(B=40000), dict(K=1, V=0x7ffffff0)):
        assert call(**bad) == _lib.SPECQ_ERR_UNSUPPORTED, bad
    for bad in (dict(K=0), dict(V=0), dict(n=0), dict(B=-1), dict(pad=10), dict(ld=9), dict(dtype=3)):
        assert call(**bad) == _lib.SPECQ_ERR_INVALID_ARG, bad


@pytest.mark.parametrize("states,error,match", [
    (torch.zeros(4, 3), TypeError, "list"),
    ([np.zeros(4)], TypeError, "state"),
    ([torch.zeros(3, 3)], ValueError, "rows"),
    ([torch.zeros(())], ValueError, "state 0"),
    ([torch.zeros(4, 6)[:, ::2]], ValueError, "contiguous"),
    ([torch.zeros(4, 3, 5).transpose(1, 2)], ValueError, "contiguous"),
    ([torch.zeros(1, 3).expand(4, -1)], ValueError, "share memory"),
    ([torch.zeros(4, 3, requires_grad=True)], ValueError, "requires grad"),
])
def test_reorder_refuses_states(states, error, match):
    with pytest.raises(error, match=match):
        specq.beam_reorder(states, _i32(2, 2))


def test_reorder_refuses_the_rest():
    x = torch.zeros(4, 6)
    with pytest.raises(ValueError, match="share memory"):
        specq.beam_reorder([x, x], _i32(2, 2))
    with pytest.raises(ValueError, match="share memory"):
        specq.beam_reorder([x[:, :4], x[:, 3:]], _i32(2, 2))
    with pytest.raises(ValueError, match="share memory"):
        specq.beam_reorder([x.view(-1)[:8].view(4, 2), x.view(-1)[6:14].view(4, 2)], _i32(2, 2))
    with pytest.raises(ValueError, match="CUDA"):       # columns of one buffer are two states
        specq.beam_reorder([x[:, :4], x[:, 4:]], _i32(2, 2))
    parent = _i32(2, 2)
    with pytest.raises(ValueError, match="parent share memory"):
        specq.beam_reorder([parent.view(4)], parent)
    with pytest.raises(ValueError, match="parent"):
        specq.beam_reorder([x], torch.zeros(2, 2, dtype=torch.int64))
    with pytest.raises(ValueError, match="beams"):
        specq.beam_reorder([x], _i32(4))
    with pytest.raises(ValueError, match="beams"):
        specq.beam_reorder([x], _i32(4), beams=3)
    with pytest.raises(ValueError, match="CUDA"):
        specq.beam_reorder([x], _i32(4), beams=2)


# ---- mass and eviction -------------------------------------------------------------------------------
@pytest.mark.parametrize("change,error,match", [
    (dict(q=torch.zeros(2, 3, 4, 64)), TypeError, "float16"),
    (dict(q=torch.zeros(6, 4, 64, dtype=F16)), ValueError, "q_len"),
    (dict(q=torch.zeros(5, 4, 64, dtype=F16), q_len=3), ValueError, "2 sequences"),
    (dict(q=torch.zeros(1, 3, 4, 64, dtype=F16).expand(2, -1, -1, -1)), ValueError, "expanded"),
    (dict(q=torch.zeros(2, 3, 3, 64, dtype=F16)), ValueError, "heads"),
    (dict(q=torch.zeros(2, 3, 4, 128, dtype=F16)), ValueError, "heads"),
    (dict(q=torch.zeros(2, 3, 64, 4, dtype=F16).transpose(2, 3)), ValueError, "heads|unit"),
    (dict(mass=torch.zeros(2, 2, 47)), ValueError, "mass"),
    (dict(mass=torch.zeros(2, 3, 48)), ValueError, "mass"),
    (dict(mass=torch.zeros(1, 2, 48)), ValueError, "mass"),
    (dict(mass=torch.zeros(2, 2, 48, dtype=F16)), TypeError, "mass"),
    (dict(mass=torch.zeros(2, 2, 96)[:, :, ::2]), ValueError, "unit stride"),
    (dict(mass=torch.zeros(1, 2, 48).expand(2, -1, -1)), ValueError, "expanded"),
    (dict(mass=torch.zeros(2, 2, 48, requires_grad=True)), ValueError, "requires grad"),
    (dict(n_rows=_i32(1)), ValueError, "n_rows"),
    (dict(decay=1.5), ValueError, "decay"),
    (dict(decay=float("nan")), ValueError, "decay"),
    (dict(sm_scale=0.0), ValueError, "sm_scale"),
    (dict(ks=torch.ones(6, 3)), ValueError, "scale"),
    (dict(), ValueError, "CUDA"),
    (dict(q=torch.zeros(6, 4, 64, dtype=BF16), q_len=3), ValueError, "CUDA"),
])
def test_mass_refusals(change, error, match):
    kc, _, ks, _ = _cache()
    a = dict(q=torch.zeros(2, 3, 4, 64, dtype=F16), kc=kc, ks=ks, block_tbl=_i32(2, 3), ctx_len=_i32(2), mass=torch.zeros(2, 2, 48))
    a.update(change)
    with pytest.raises(error, match=match):
        specq.attention_mass_blocks(**a)


@pytest.mark.parametrize("change,error,match", [
    (dict(keep=0), ValueError, "keep"),
    (dict(recent=-1), ValueError, "recent"),
    (dict(recent=9), ValueError, "recent"),
    (dict(mass=torch.zeros(2, 2, 47)), ValueError, "mass"),
    (dict(mass=torch.zeros(1, 2, 2, 48)), ValueError, "mass"),
    (dict(ref=_i32(5)), ValueError, "ref"),
    (dict(ctx_out=_i32(1)), ValueError, "ctx_out"),
    (dict(), ValueError, "CUDA"),
    (dict(ref=_i32(6)), ValueError, "CUDA"),
])
def test_evict_refusals(change, error, match):
    a = dict(zip(("kc", "vc", "ks", "vs"), _cache()), block_tbl=_i32(2, 3), ctx_len=_i32(2), mass=torch.zeros(2, 2, 48), keep=8, recent=2)
    a.update(change)
    with pytest.raises(error, match=match):
        specq.kv_evict_blocks(**a)


def test_evict_of_layers_wants_a_mass_of_layers():
    cache = _cache(layers=3)
    with pytest.raises(ValueError, match="mass"):
        specq.kv_evict_blocks(*cache, _i32(2, 3), _i32(2), torch.zeros(2, 2, 48), 8)
    with pytest.raises(ValueError, match="mass"):
        specq.kv_evict_blocks(*cache, _i32(2, 3), _i32(2), torch.zeros(2, 2, 2, 48), 8)
    with pytest.raises(ValueError, match="CUDA"):
        specq.kv_evict_blocks(*cache, _i32(2, 3), _i32(2), torch.zeros(3, 2, 2, 48), 8)
    with pytest.raises(ValueError, match="expanded"):
        specq.kv_evict_blocks(*cache, _i32(2, 3), _i32(2), torch.zeros(1, 2, 2, 48).expand(3, -1, -1, -1), 8)


def test_bounded_cache_library_refuses():
    lib = _lib.load()

    def mass(D=64, page=16, B=1, cols=2, cache=0, q=16, kv=64):
        return lib.specq_attention_mass(q, 64, 64, 64, 0, 16, kv, 64, 64, cache, 4, 16, 1, 1, 16, 2, cols, 16, None, 0.1, 1.0, 16, 64, 64, B, 1, 1,
                                        1, D, page, None, 0, None)
    for bad in (dict(D=96), dict(page=24), dict(page=4), dict(page=256), dict(B=70000), dict(cols=1 << 27, page=128), dict(q=8), dict(kv=24)):
        assert mass(**bad) == _lib.SPECQ_ERR_UNSUPPORTED, bad
    for bad in (dict(cache=2), dict(B=-1), dict(q=None), dict(cols=1000)):    # (the last: no workspace)
        assert mass(**bad) == _lib.SPECQ_ERR_INVALID_ARG, bad

    def evict(D=64, page=16, L=1, keep=8, recent=2, ws=16, n=1 << 20, kv=64, pages=4):
        return lib.specq_block_evict(16, 16, 64, kv, 64, 64, 0, L, pages, 16, 16, 1, 1, 1, 16, 2, 2, 16, None, 16, 64, 64, 64, keep, recent, 16, 1,
                                     1, D, page, ws, n, None)
    for bad in (dict(D=96), dict(page=24), dict(L=70000), dict(kv=24), dict(pages=1 << 28)):
        assert evict(**bad) == _lib.SPECQ_ERR_UNSUPPORTED, bad
    for bad in (dict(L=0), dict(keep=0), dict(recent=9), dict(recent=-1), dict(ws=None), dict(n=8), dict(ws=8)):
        assert evict(**bad) == _lib.SPECQ_ERR_INVALID_ARG, bad


def test_release_of_a_tail_refusals():
    ref, tbl, held, drop = _i32(8), _i32(2, 4), _i32(2), torch.zeros(2, dtype=torch.bool)
    with pytest.raises(ValueError, match="together"):
        specq.pages_release(ref, tbl, held, drop, length=_i32(2))
    with pytest.raises(ValueError, match="together"):
        specq.pages_release(ref, tbl, held, drop, page=16)
    with pytest.raises(ValueError, match="length"):
        specq.pages_release(ref, tbl, held, drop, _i32(1), 16)
    with pytest.raises(ValueError, match="page"):
        specq.pages_release(ref, tbl, held, drop, _i32(2), 0)
    with pytest.raises(ValueError, match="CUDA"):
        specq.pages_release(ref, tbl, held, drop, _i32(2), 16)


# ---- the oracle itself -------------------------------------------------------------------------------
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_oracle_gradients_are_differences(layout):
    """Central differences of a sum of products, 64 bits: error h^2 times the third derivative, about 1e-8 here."""
    rng = np.random.default_rng(1)
    T, H, D, rot, eps, h = 3, 2, 10, 6, 1e-3, 1e-4
    x, g, w = rng.normal(size=(T, H, D)), rng.normal(size=(T, H, D)), rng.normal(size=D)
    table, pos = specq.rope_table(16, rot, device="cpu").numpy(), np.array([0, 5, 9])

    def f(x, w):
        return (O.norm_turn(x, w, table, pos, layout, eps) * g).sum()
    dx, dw = O.norm_turn_grad(x, w, g, table, pos, layout, eps)
    for _ in range(20):
        d, e = rng.normal(size=x.shape), rng.normal(size=D)
        assert abs((f(x + h * d, w) - f(x - h * d, w)) / (2 * h) - (dx * d).sum()) < 1e-5
        assert abs((f(x, w + h * e) - f(x, w - h * e)) / (2 * h) - (dw * e).sum()) < 1e-5


def test_oracle_beams():
    x = np.log(np.array([[0.5, 0.25, 0.25], [0.1, 0.1, 0.8]]))
    s, p, t = O.beam_select(x, np.array([[0.0, np.log(0.5)]]), 4)
    assert t.tolist() == [[0, 2, 1, 2]] and p.tolist() == [[0, 1, 0, 0]]
    np.testing.assert_allclose(np.exp(s), [[0.5, 0.4, 0.25, 0.25]])
    s, p, t = O.beam_select(x, np.array([[0.0, -np.inf]]), 5, done=[True, False], pad=2)
    assert t.tolist() == [[2, 2, 2, 2, 2]] and p.tolist() == [[0, 1, 0, 1, 0]] and s[0, 0] == 0 and (s[0, 1:] == -np.inf).all()


def test_oracle_eviction_keeps_ties_in_order():
    assert O.evict_choice(np.array([1.0, 2.0, 2.0, 2.0, np.nan, 9.0]), 6, 3, 1).tolist() == [1, 2, 5]
    assert O.evict_choice(np.zeros(6), 6, 4, 0).tolist() == [0, 1, 2, 3]
    assert O.evict_choice(np.arange(6.0), 6, 3, 3).tolist() == [3, 4, 5]
