"""Normalised heads, beams and the bounded cache without a GPU: workspaces, and gradients that the operators do not have."""
import ctypes

import pytest
import torch
from torch.autograd import forward_ad

import specq
from specq import _lib

SPACE = 512 << 20


def _mass(B, q_len, G, KV, cols, D=128, page=16):
    n = ctypes.c_int64(-1)
    assert _lib.load().specq_attention_mass_workspace(B, q_len, KV * G, KV, D, page, cols, ctypes.byref(n)) == 0
    return n.value


@pytest.mark.parametrize("q_len,G", [(1, 4), (4, 4), (9, 4), (24, 4), (64, 8)])
@pytest.mark.parametrize("tokens", [8192, 131072, 1 << 20])
@pytest.mark.parametrize("B,KV", [(1, 1), (1, 8), (32, 8), (64, 8), (256, 8), (1024, 1), (7, 32)])
def test_workspace_of_a_wide_table_is_bounded(B, KV, tokens, q_len, G):
    """At most 512 MB or what one KV head of one sequence takes, and never less than that."""
    one, got = _mass(1, q_len, G, 1, tokens // 16), _mass(B, q_len, G, KV, tokens // 16)
    assert min(one, 1) <= got <= max(SPACE, one), (one, got)


def _evict(L, B, KV, keep):
    n = ctypes.c_int64(-1)
    assert _lib.load().specq_block_evict_workspace(L, B, KV, keep, ctypes.byref(n)) == 0
    return n.value


@pytest.mark.parametrize("L,B,KV,keep", [(32, 64, 8, 131072), (80, 256, 8, 32768), (1, 65535, 1, 4096), (64, 3, 8, 1 << 20)])
def test_workspace_of_a_large_budget_is_bounded(L, B, KV, keep):
    one, got = _evict(L, 1, KV, keep), _evict(L, B, KV, keep)
    assert one <= got <= max(SPACE, one), (one, got)


def test_workspace_of_ordinary_calls():
    """Nothing for what a cluster holds; 8 bytes a row and block and 4 a row and token for a stream of tiles; the sums alone for many rows."""
    assert _mass(1, 1, 4, 8, 4) == 0
    assert _mass(32, 1, 4, 8, 512) == 32 * 8 * 4 * (8192 * 4 + 8192 // 2048 * 8)
    assert _mass(2, 64, 4, 8, 1024) == 2 * 8 * 256 * (16384 // 256 * 8 + 4)
    assert _mass(0, 1, 4, 8, 512) == 0
    assert _evict(4, 12, 8, 1024) == 4 * 12 * 8 * 1025 * 4
    assert _evict(4, 0, 8, 1024) == 0


@pytest.mark.parametrize("what", ["q", "k", "q_weight", "k_weight", "x", "logits", "scores", "state", "mass"])
@pytest.mark.parametrize("grad", [False, True])
def test_tangents_are_refused(what, grad):
    """A dual tensor's tangent would be lost without a word."""
    F16 = torch.float16
    pos, table, kc = torch.zeros(4, dtype=torch.int32), torch.zeros(8, 64), torch.zeros(2, 16, 2, 64, dtype=torch.int8)
    a = {"q": torch.zeros(4, 4, 64, dtype=F16), "k": torch.zeros(4, 2, 64, dtype=F16), "q_weight": torch.ones(64, dtype=F16),
         "k_weight": torch.ones(64, dtype=F16), "x": torch.zeros(4, 4, 64), "logits": torch.zeros(4, 10), "scores": torch.zeros(2, 2),
         "state": torch.zeros(4, 3), "mass": torch.zeros(1, 2, 32)}
    i32 = torch.zeros(1, 2, dtype=torch.int32)

    def call(a):
        if what in ("q", "k", "q_weight", "k_weight"):
            return specq.qk_norm_rope(a["q"], a["k"], a["q_weight"], a["k_weight"], pos, table)
        if what == "x":
            return specq.rope(a["x"], pos, table)
        if what in ("logits", "scores"):
            return specq.beam_select(a["logits"], a["scores"])
        if what == "state":
            return specq.beam_reorder([a["state"]], pos, beams=2)
        return specq.attention_mass_blocks(a["q"][:1, None], kc, torch.ones(2, 2), i32, i32[:, 0], a["mass"])
    if grad and what in ("q", "k", "q_weight", "k_weight", "x"):
        a[what].requires_grad_(True)
    with forward_ad.dual_level():
        dual = dict(a, **{what: forward_ad.make_dual(a[what], torch.ones_like(a[what]))})
        with pytest.raises(ValueError, match="forward-mode"):
            call(dual)
        with forward_ad._set_fwd_grad_enabled(False), pytest.raises(ValueError, match="CUDA"):
            call(dual)
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
        call(a)


@pytest.mark.parametrize("sm_scale", [float("inf"), 1e39, float("nan"), -1.0, 0.0])
def test_mass_refuses_a_scale_that_is_not_finite(sm_scale):
    """An infinite scale times a score of 0 would be NaN."""
    kc, i32 = torch.zeros(2, 16, 2, 64, dtype=torch.int8), torch.zeros(1, 2, dtype=torch.int32)
    with pytest.raises(ValueError, match="sm_scale"):
        specq.attention_mass_blocks(torch.zeros(1, 1, 4, 64).half(), kc, torch.ones(2, 2), i32, i32[:, 0], torch.zeros(1, 2, 32), sm_scale=sm_scale)
    assert _lib.load().specq_attention_mass(16, 64, 64, 64, 0, 16, 64, 64, 64, 0, 4, 16, 1, 1, 16, 2, 2, 16, None, sm_scale, 1.0, 16, 64, 64, 1, 1, 1,
                                            1, 64, 16, None, 0, None) == _lib.SPECQ_ERR_INVALID_ARG


@pytest.mark.parametrize("same", ["vc", "vs"])
def test_evict_refuses_one_cache_for_keys_and_values(same):
    """Both would be moved at once."""
    kc, i32 = torch.zeros(2, 16, 2, 64, dtype=torch.int8), torch.zeros(1, 2, dtype=torch.int32)
    a = {"kc": kc, "vc": kc.clone(), "ks": torch.ones(2, 2), "vs": torch.ones(2, 2)}
    with pytest.raises(ValueError, match="CUDA"):
        specq.kv_evict_blocks(*a.values(), i32, i32[:, 0], torch.zeros(1, 2, 32), 8)
    a[same] = a["k" + same[1]]
    with pytest.raises(ValueError, match="same memory"):
        specq.kv_evict_blocks(*a.values(), i32, i32[:, 0], torch.zeros(1, 2, 32), 8)
