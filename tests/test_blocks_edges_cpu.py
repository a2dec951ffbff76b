"""The block-scaled cache's operators without a GPU: what else is refused before anything is launched, and the
rotary tables at the ends of their rules.  (Tensors on the CPU are refused last, with "CUDA" in the message, so a
refusal that names something else comes from the arguments.)"""
import math

import numpy as np
import pytest
import torch

import specq
from specq import _lib


def _cache(P=6, page=16, KV=2, D=64, dtype=torch.int8):
    kc = torch.zeros(P, page, KV, D, dtype=torch.uint8).view(dtype)
    return kc, kc.clone(), torch.ones(P, KV), torch.ones(P, KV)


def _i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def test_queries_expanded_over_the_sequences_are_refused():
    """A batch stride of 0 means packed rows to the kernels, which would read past the one sequence there is."""
    cache = _cache()
    tbl, ctx = _i32(3, 2), _i32(3)
    one = torch.zeros(1, 2, 4, 64, dtype=torch.float16)
    q = one.expand(3, -1, -1, -1)
    with pytest.raises(ValueError, match="expanded"):
        specq.paged_attention_blocks(q, *cache, tbl, ctx)
    with pytest.raises(ValueError, match="expanded"):
        specq.paged_attention_blocks(q, *cache, tbl, ctx, plan=_i32(2), n_seqs=1)
    # one sequence, tokens or heads of one row each, packed rows of one token: the strides say what is meant
    for ok, kw in ((one, dict()), (one[:, :1].expand(-1, 2, -1, -1), dict()), (one[:, :, :1].expand(-1, -1, 4, -1), dict())):
        with pytest.raises(ValueError, match="CUDA"):
            specq.paged_attention_blocks(ok, *cache, tbl[:1], ctx[:1], **kw)
    with pytest.raises(ValueError, match="CUDA"):
        specq.paged_attention_blocks(q, *cache, tbl, ctx, n_seqs=1)
    with pytest.raises(ValueError, match="CUDA"):
        specq.paged_attention_blocks(one[0, :1].expand(6, -1, -1), *cache, tbl, ctx, q_len=2)


def test_written_tensors_whose_elements_share_memory_are_refused():
    kc, vc, ks, vs = cache = _cache()
    k = torch.zeros(4, 2, 64, dtype=torch.float16)
    q = torch.zeros(2, 2, 4, 64, dtype=torch.float16)
    tbl, ctx = _i32(2, 3), _i32(2)
    table = specq.rope_table(8, 64, device="cpu")
    with pytest.raises(ValueError, match="out .*expanded"):
        specq.rope(k, _i32(4), table, out=k[:1].expand(4, -1, -1))
    with pytest.raises(ValueError, match="out .*expanded"):
        specq.rope(k, _i32(4), table, out=k[:, :1].expand(-1, 2, -1))
    with pytest.raises(ValueError, match="q_out .*expanded"):
        specq.kv_append_blocks(k, k, *cache, tbl, ctx, 2, q=k, q_out=k[:1].expand(4, -1, -1), table=table)
    for dim in range(3):
        shape = [2, 2, 4, 64]
        shape[dim] = 1
        with pytest.raises(ValueError, match="out .*expanded"):
            specq.paged_attention_blocks(q, *cache, tbl, ctx, out=torch.zeros(shape, dtype=torch.float16).expand(2, 2, 4, 64))
    wide = [t[:1].expand_as(t) for t in cache]
    pool = _i32(6), tbl, _i32(2)
    for bad in ((wide[0], wide[1], ks, vs), (kc, vc, wide[2], wide[3]), (kc, vc, ks[:, :1].expand(6, 2), vs[:, :1].expand(6, 2))):
        with pytest.raises(ValueError, match="expanded"):
            specq.kv_append_blocks(k, k, *bad, tbl, ctx, 2)
        with pytest.raises(ValueError, match="expanded"):
            specq.kv_compact_blocks(*bad, tbl, ctx, 2, _i32(2, 2), _i32(2))
        with pytest.raises(ValueError, match="expanded"):
            specq.pages_fork(*bad, *pool, _i32(2), _i32(2))
    # attention only reads the scales: one for all pages is fine
    with pytest.raises(ValueError, match="CUDA"):
        specq.paged_attention_blocks(q, kc, vc, wide[2], wide[3], tbl, ctx)


def test_plans_that_are_too_short_are_refused():
    """rope reads plan[0], append and attention plan[0] and plan[1]."""
    cache = _cache()
    k = torch.zeros(4, 2, 64, dtype=torch.float16)
    tbl, ctx = _i32(2, 3), _i32(2)
    table = specq.rope_table(8, 64, device="cpu")
    for plan in (_i32(0), _i32(1), _i32(8)[::4], _i32(3, 2)[:, 0]):
        with pytest.raises(ValueError, match="plan"):
            specq.kv_append_blocks(k, k, *cache, tbl, ctx, 2, plan=plan)
        with pytest.raises(ValueError, match="plan"):
            specq.paged_attention_blocks(k, *cache, tbl, ctx, q_len=2, plan=plan)
    with pytest.raises(ValueError, match="plan"):
        specq.rope(k, _i32(4), table, plan=_i32(0))
    for plan in (_i32(2), _i32(3), _i32(1, 2).t()):
        with pytest.raises(ValueError, match="CUDA"):
            specq.kv_append_blocks(k, k, *cache, tbl, ctx, 2, plan=plan)
    with pytest.raises(ValueError, match="CUDA"):
        specq.rope(k, _i32(4), table, plan=_i32(1))


def test_query_groups_that_the_row_arithmetic_cannot_hold_are_refused():
    """A row's token is a product by ceil(2^32 / group), exact while rows * group <= 2^32: a group of 279 heads
    goes wrong before the limit of 2^24 query rows does."""
    group, rows = 279, (1 << 24) // 279 * 279
    magic = 0xFFFFFFFF // group + 1
    assert ((rows - 1) * magic) >> 32 != (rows - 1) // group
    lib = _lib.load()
    n = _lib.C.c_int64()

    def size(q_len, H, H_KV):
        return lib.specq_block_attention_workspace(1, 1, q_len, q_len, H, H_KV, 128, 16, 0, 0, n)
    assert size(60000, 279, 1) == _lib.SPECQ_ERR_UNSUPPORTED
    assert size(1 << 15, 512, 1) == _lib.SPECQ_ERR_UNSUPPORTED
    # the largest that are taken: exact for every row (and for the padding of a block)
    for g in (2, 3, 7, 255, 256, 279, 300, 1000):
        most = min((1 << 24) // g, (1 << 32) // (g * g) - 1) * g
        r = np.arange(max(0, most - (1 << 16)), most, dtype=np.uint64)
        assert ((r * np.uint64(0xFFFFFFFF // g + 1)) >> np.uint64(32) == r // np.uint64(g)).all()


def _yarn(n, rot, base, factor, original, fast=32.0, slow=1.0):
    """Angles a position from the method's definition, in 64 bits: the ramp runs over the pair index between the
    pairs that turn `fast` and `slow` times in `original` positions, its ends rounded outwards and kept within
    0 .. rot - 1."""
    def pair(turns):
        return rot * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))
    lo, hi = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), rot - 1)
    i = np.arange(rot // 2)
    inv = base ** (-2.0 * i / rot)
    ramp = np.clip((i - lo) / max(hi - lo, 1e-3), 0, 1)
    return inv * (1 - ramp) + inv / factor * ramp


@pytest.mark.parametrize("base", [10000.0, 500000.0])
@pytest.mark.parametrize("rot", [32, 64, 128])
@pytest.mark.parametrize("original", [2048, 4096, 32768, 65536, 131072, 1 << 20])
def test_yarn_tables_at_any_original_length(original, rot, base):
    """Table entries are fp32 roundings of 64-bit cosines: 2^-24 of the gain, and the angle's own 64-bit error."""
    factor, n = 4.0, 300
    t = specq.rope_table(n, rot, base=base, device="cpu", scaling={"type": "yarn", "factor": factor, "original": original})
    ang = np.arange(n)[:, None] * _yarn(n, rot, base, factor, original)
    gain = 0.1 * math.log(factor) + 1.0
    t = t.double().numpy()
    assert np.abs(t[:, : rot // 2] - np.cos(ang) * gain).max() <= 2.0 ** -23
    assert np.abs(t[:, rot // 2:] - np.sin(ang) * gain).max() <= 2.0 ** -23


def test_yarn_gain_is_one_where_nothing_is_stretched():
    """The default attention factor is 0.1 ln(factor) + 1 above a factor of 1, and 1 up to it."""
    for factor in (0.25, 0.5, 1.0):
        t = specq.rope_table(4, 32, device="cpu", scaling={"type": "yarn", "factor": factor, "original": 4096})
        assert (t[0, :16] == 1.0).all()
    t = specq.rope_table(4, 32, device="cpu", scaling={"type": "yarn", "factor": 0.5, "original": 4096, "attention": 0.75})
    assert (t[0, :16] == 0.75).all()
    t = specq.rope_table(4, 32, device="cpu", scaling={"type": "yarn", "factor": 2.0, "original": 4096})
    assert abs(t[0, 0].item() - (0.1 * math.log(2.0) + 1.0)) <= 2.0 ** -23


def test_rope_refuses_gradients_that_it_does_not_have():
    x, pos, table = torch.zeros(4, 2, 64), _i32(4), specq.rope_table(8, 64, device="cpu")
    leaf = x.clone().requires_grad_()
    with pytest.raises(ValueError, match="requires grad"):
        specq.rope(leaf, pos, table, out=torch.zeros(4, 2, 64))
    with pytest.raises(ValueError, match="requires grad"):
        specq.rope(x, pos, table, out=leaf)
    with pytest.raises(ValueError, match="table has no gradient"):
        specq.rope(x, pos, table.clone().requires_grad_())
    with pytest.raises(ValueError, match="CUDA"):
        specq.rope(leaf, pos, table)
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
        specq.rope(leaf, pos, table, out=torch.zeros(4, 2, 64))
