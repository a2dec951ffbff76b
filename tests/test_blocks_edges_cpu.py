"""The block-scaled cache's operators without a GPU: what else is refused before anything is launched, and the
rotary tables at the ends of their rules.  (Tensors on the CPU are refused last, with "CUDA" in the message, so a
refusal that names something else comes from the arguments.)"""

import pytest
import torch

import specq


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
