"""The block-scaled cache without a GPU: what is refused, the rotary tables, the oracle itself."""
import math

import numpy as np
import pytest
import torch

import specq
from oracle import block_oracle as BO
from specq import _lib


def _cache(P=6, page=16, KV=2, D=64, dtype=torch.int8):
    kc = torch.zeros(P, page, KV, D, dtype=torch.uint8).view(dtype)
    return kc, kc.clone(), torch.ones(P, KV), torch.ones(P, KV)


def _i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def test_cpu_tensors_are_refused():
    kc, vc, ks, vs = _cache()
    k = torch.zeros(4, 2, 64, dtype=torch.float16)
    tbl, ctx = _i32(2, 3), _i32(2)
    table = specq.rope_table(8, 64, device="cpu")
    with pytest.raises(ValueError, match="CUDA"):
        specq.rope(k, _i32(4), table)
    with pytest.raises(ValueError, match="CUDA"):
        specq.kv_append_blocks(k, k, kc, vc, ks, vs, tbl, ctx, 2)
    with pytest.raises(ValueError, match="CUDA"):
        specq.paged_attention_blocks(k.view(2, 2, 2, 64), kc, vc, ks, vs, tbl, ctx)
    with pytest.raises(ValueError, match="CUDA"):
        specq.kv_compact_blocks(kc, vc, ks, vs, tbl, ctx, 2, _i32(2, 2), _i32(2))
    with pytest.raises(ValueError, match="CUDA"):
        specq.pages_release(_i32(6), tbl, _i32(2), torch.zeros(2, dtype=torch.bool))
    with pytest.raises(ValueError, match="CUDA"):
        specq.pages_reserve(_i32(6), tbl, _i32(2), _i32(2), 16)
    with pytest.raises(ValueError, match="CUDA"):
        specq.pages_fork(kc, vc, ks, vs, _i32(6), tbl, _i32(2), _i32(2), _i32(2))


def test_wrong_tensors_are_refused():
    kc, vc, ks, vs = _cache()
    k = torch.zeros(4, 2, 64, dtype=torch.float16)
    q = k.view(2, 2, 2, 64)
    tbl, ctx = _i32(2, 3), _i32(2)
    table = specq.rope_table(8, 64, device="cpu")
    with pytest.raises(ValueError, match="layout"):
        specq.rope(k, _i32(4), table, layout="neox")
    with pytest.raises(TypeError, match="int32"):
        specq.rope(k, torch.zeros(4, dtype=torch.int64), table)
    with pytest.raises(ValueError, match="pos"):
        specq.rope(k, _i32(3), table)
    with pytest.raises(ValueError, match="rot"):
        specq.rope(k[..., :32], _i32(4), table)
    with pytest.raises(TypeError):
        specq.rope(k.to(torch.int8), _i32(4), table)
    with pytest.raises(ValueError, match="out"):
        specq.rope(k, _i32(4), table, out=k[:3])
    with pytest.raises(TypeError, match="float8"):
        specq.kv_append_blocks(k, k, kc.float(), vc, ks, vs, tbl, ctx, 2)
    with pytest.raises(TypeError, match="float32"):
        specq.kv_append_blocks(k, k, kc, vc, ks.half(), vs, tbl, ctx, 2)
    with pytest.raises(ValueError, match="ks and vs"):
        specq.kv_append_blocks(k, k, kc, vc, ks[:, :1], vs, tbl, ctx, 2)
    with pytest.raises(ValueError, match="rotary table"):
        specq.kv_append_blocks(k, k, kc, vc, ks, vs, tbl, ctx, 2, q=k)
    with pytest.raises(ValueError, match="v must be"):
        specq.kv_append_blocks(k, k[:3], kc, vc, ks, vs, tbl, ctx, 2)
    with pytest.raises(ValueError, match="q_len"):
        specq.kv_append_blocks(k, k, kc, vc, ks, vs, tbl, ctx, -1)
    with pytest.raises(ValueError, match="packed"):
        specq.paged_attention_blocks(k, kc, vc, ks, vs, tbl, ctx)
    with pytest.raises(TypeError, match="float16"):
        specq.paged_attention_blocks(q.float(), kc, vc, ks, vs, tbl, ctx)
    with pytest.raises(ValueError, match="heads"):
        specq.paged_attention_blocks(q[:, :, :1], kc, vc, ks, vs, tbl, ctx)
    with pytest.raises(ValueError, match="tree"):
        specq.paged_attention_blocks(q, kc, vc, ks, vs, tbl, ctx, tree=torch.zeros(2, 1, dtype=torch.int64))
    with pytest.raises(ValueError, match="ctx_len"):
        specq.paged_attention_blocks(q, kc, vc, ks, vs, tbl, ctx[:1])
    with pytest.raises(ValueError, match="out"):
        specq.paged_attention_blocks(q, kc, vc, ks, vs, tbl, ctx, out=q[:1])
    with pytest.raises(ValueError, match="alike"):
        specq.kv_compact_blocks(kc, vc[:, :8], ks, vs, tbl, ctx, 2, _i32(2, 2), _i32(2))
    with pytest.raises(ValueError, match="accept"):
        specq.kv_compact_blocks(kc, vc, ks, vs, tbl, ctx, 2, _i32(1, 2), _i32(2))
    with pytest.raises(ValueError, match="drop"):
        specq.pages_release(_i32(6), tbl, _i32(2), _i32(2))
    with pytest.raises(ValueError, match="page"):
        specq.pages_reserve(_i32(6), tbl, _i32(2), _i32(2), 0)
    with pytest.raises(ValueError, match="held"):
        specq.pages_reserve(_i32(6), tbl, _i32(1), _i32(2), 16)
    with pytest.raises(ValueError, match="pool"):
        specq.pages_fork(kc, vc, ks, vs, _i32(7), tbl, _i32(2), _i32(2), _i32(2))


def _sig(name):
    return len(_lib.SIGNATURES[name][1])


def test_c_entries_refuse_bad_sizes():
    """The C ABI on its own: nothing below reaches a device."""
    lib = _lib.load()
    E, U = _lib.SPECQ_ERR_INVALID_ARG, _lib.SPECQ_ERR_UNSUPPORTED
    rope = dict(x=16, xt=64, xh=64, out=32, ot=64, oh=64, dtype=0, pos=16, table=16, n_pos=4, T=1, H=1, D=64, rot=64,
                layout=0, inverse=0, plan=None, stream=None)

    def r(**kw):
        return lib.specq_rope(*dict(rope, **kw).values())
    assert r(rot=63) == E and r(rot=66) == E and r(rot=0) == E and r(layout=2) == E and r(dtype=3) == E
    assert r(T=-1) == E and r(pos=None) == E and r(n_pos=0) == E
    assert r(out=16, ot=128) == E          # in place with other strides
    assert r(T=0, x=None) == _lib.SPECQ_OK
    app = dict(k=16, kt=64, kh=64, v=16, vt=64, vh=64, q=None, qt=0, qh=0, q_out=None, ot=0, oh=0, dtype=0, table=None,
               n_pos=0, rot=0, layout=0, pos=None, kc=16, vc=16, kv_sp=1024, kv_so=64, kv_sh=64, cache=0, n_pages=1,
               ks=16, vs=16, s_sp=1, s_sh=1, bt=16, bt_sb=1, cols=1, ctx=16, plan=None, B=1, n_seqs=1, q_len=1,
               ql_max=1, H=0, H_KV=1, D=64, page=16, stream=None)
    assert len(app) == _sig("specq_block_append")

    def a(**kw):
        return lib.specq_block_append(*dict(app, **kw).values())
    assert a(D=96) == U and a(page=12) == U and a(page=256) == U and a(cache=2) == E and a(dtype=1) == E
    assert a(n_seqs=2) == E and a(q_len=2) == E and a(k=None) == E and a(kt=62) == U and a(kv_so=68) == U
    assert a(q=16) == E                     # queries without a table
    assert a(table=16, rot=24, n_pos=4) == U and a(table=16, rot=80, n_pos=4) == E
    assert a(q_len=0, k=None) == _lib.SPECQ_OK
    att = dict(q=16, q_sb=64, q_st=64, q_sh=64, dtype=0, kc=16, vc=16, kv_sp=1024, kv_so=64, kv_sh=64, cache=0, n_pages=1,
               ks=16, vs=16, s_sp=1, s_sh=1, bt=16, bt_sb=1, cols=1, ctx=16, tree=None, tree_sb=0, tree_st=0,
               sm=0.125, out=16, o_sb=64, o_st=64, o_sh=64, plan=None, B=1, n_seqs=1, q_len=1, ql_max=1, H=1, H_KV=1,
               D=64, page=16, ws=None, ws_bytes=0, stream=None)
    assert len(att) == _sig("specq_block_attention")

    def t(**kw):
        return lib.specq_block_attention(*dict(att, **kw).values())
    assert t(H=3, H_KV=2) == E and t(D=256) == U and t(page=48) == U and t(dtype=1) == E and t(cache=7) == E
    assert t(kv_so=72) == U and t(q_st=62) == U and t(n_pages=0) == E and t(q=None) == E and t(q_len=2) == E
    assert t(tree=16, q_len=65, ql_max=65) == U
    assert t(B=0, n_seqs=0, q=None) == _lib.SPECQ_OK
    com = dict(kc=16, vc=16, kv_sl=0, kv_sp=1024, kv_so=64, kv_sh=64, cache=0, L=1, n_pages=1, ks=16, vs=16, s_sl=0,
               s_sp=1, s_sh=1, bt=16, bt_sb=1, cols=1, ctx=16, accept=16, acc_sb=1, acc_cols=1, n_accept=16, out=32, B=1,
               q_len=1, H_KV=1, D=64, page=16, stream=None)
    assert len(com) == _sig("specq_block_compact")

    def c(**kw):
        return lib.specq_block_compact(*dict(com, **kw).values())
    assert c(out=16) == E                   # ctx_out over ctx_len
    assert c(L=0) == E and c(D=32) == U and c(page=4) == U and c(kv_sh=24) == U and c(accept=None) == E
    assert lib.specq_pages_release(16, 4, 16, 1, 16, 1, 2, 16, None) == E          # ld < C
    assert lib.specq_pages_reserve(16, 4, 16, 2, 16, 9000, 2, 16, 16, 16, None) == U
    assert lib.specq_pages_reserve(16, 4, 16, 2, 16, 1, 2, 16, 0, 16, None) == E   # page 0
    assert lib.specq_pages_reserve(20, 4, 16, 2, 16, 1, 2, 16, 16, 16, None) == U  # ref not aligned
    assert lib.specq_pages_fork(16, 16, 0, 1024, 64, 64, 1, 16, 16, 0, 1, 1, 16, 4, 16, 2, 16, 1, 2, 16, 16, None, 16, 1,
                                64, 16, None) == E
    assert lib.specq_pages_fork(16, 16, 0, 1024, 64, 64, 1, 16, 16, 0, 1, 1, 16, 4, 16, 2, 16, 1, 2, 16, 16, 16, 16, 1,
                                72, 16, None) == U


def test_rope_tables():
    n, rot = 300, 32
    t = specq.rope_table(n, rot, base=10000.0, device="cpu").double().numpy()
    i = np.arange(rot // 2)
    ang = np.arange(n)[:, None] * 10000.0 ** (-2 * i / rot)
    assert np.abs(t[:, : rot // 2] - np.cos(ang)).max() <= 2.0 ** -24
    assert np.abs(t[:, rot // 2:] - np.sin(ang)).max() <= 2.0 ** -24
    lin = specq.rope_table(n, rot, scaling={"type": "linear", "factor": 4.0}, device="cpu")
    assert np.abs(lin.double().numpy()[:, : rot // 2] - np.cos(ang / 4)).max() <= 2.0 ** -24
    ntk = specq.rope_table(n, rot, scaling={"type": "ntk", "factor": 4.0}, device="cpu").double().numpy()
    base = 10000.0 * 4.0 ** (rot / (rot - 2))
    assert np.abs(ntk[:, rot // 2:] - np.sin(np.arange(n)[:, None] * base ** (-2 * i / rot))).max() <= 2.0 ** -24
    # llama3: fast pairs kept, slow ones divided
    l3 = specq.rope_table(n, rot, base=500000.0, device="cpu",
                          scaling={"type": "llama3", "factor": 8.0, "original": 8192, "low": 1.0, "high": 4.0})
    inv = 500000.0 ** (-2 * i / rot)
    turns = 8192 * inv / (2 * math.pi)
    keep = np.clip((turns - 1) / 3, 0, 1)
    want = inv * keep + inv / 8 * (1 - keep)
    assert keep[0] == 1 and keep[-1] == 0
    assert np.abs(l3.double().numpy()[:, : rot // 2] - np.cos(np.arange(n)[:, None] * want)).max() <= 2.0 ** -23
    ya = specq.rope_table(n, rot, device="cpu", scaling={"type": "yarn", "factor": 4.0, "original": 4096})
    assert abs(ya[0, 0].item() - (0.1 * math.log(4.0) + 1.0)) < 1e-6
    first, last = ya[1, 0].item() / ya[0, 0].item(), ya[200, rot // 2 - 1].item() / ya[0, 0].item()
    assert abs(first - math.cos(1.0)) < 1e-6                                # the fastest pair is kept
    assert abs(last - math.cos(200 * 10000.0 ** (-30 / 32) / 4)) < 1e-6     # the slowest is divided
    for bad in (dict(rot=3), dict(rot=0), dict(n_pos=0), dict(scaling={"type": "cubic", "factor": 2.0})):
        with pytest.raises(ValueError):
            specq.rope_table(**dict(dict(n_pos=8, rot=8, device="cpu"), **bad))


def test_oracle_e4m3_rounding_is_torchs():
    """The oracle's e4m3 rounding on every representable value, on all midpoints and on random numbers."""
    v = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    v = np.sort(v[torch.isfinite(v)].numpy().astype(np.float32))
    g = np.random.default_rng(0)
    x = np.concatenate([v, (v[1:] + v[:-1]) / 2, g.standard_normal(2000) * 100, g.standard_normal(2000) * 0.01])
    x = x.astype(np.float32)
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).float().numpy()
    assert np.array_equal(BO.e4m3_round(x), want)
    assert BO.e4m3_round(np.float32(1e9)) == 448.0


def test_oracle_catches_planted_mistakes():
    """A wrong causal limit or a scale off by a page shows in the oracle's outputs."""
    g = np.random.default_rng(1)
    q = g.standard_normal((1, 3, 2, 8))
    kc, vc = (g.integers(-127, 128, (4, 8, 1, 8)).astype(np.float32) for _ in range(2))
    ks, vs = g.uniform(0.01, 0.02, (4, 1)), g.uniform(0.01, 0.02, (4, 1))
    tbl = np.array([[2, 0, 3]])
    ref, _, _ = BO.attention(q, kc, vc, ks, vs, tbl, [19])
    assert np.abs(BO.attention(q, kc, vc, ks, vs, tbl, [18])[0] - ref).max() > 1e-3
    assert np.abs(BO.attention(q, kc, vc, ks[::-1], vs, tbl, [19])[0] - ref).max() > 1e-3
    tree = np.array([[1, 3, 7]])            # the causal chain as a tree
    assert np.allclose(BO.attention(q, kc, vc, ks, vs, tbl, [19], tree=tree)[0], ref)
    assert np.abs(BO.attention(q, kc, vc, ks, vs, tbl, [19], tree=np.array([[1, 3, 5]]))[0] - ref).max() > 1e-4
