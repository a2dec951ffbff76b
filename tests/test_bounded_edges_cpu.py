"""The workspace of the operators around a bounded cache, without a GPU."""
import ctypes

import pytest

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


def test_workspace_of_ordinary_calls():
    """Nothing for what a cluster holds; 8 bytes a row and block and 4 a row and token for a stream of tiles; the sums alone for many rows."""
    assert _mass(1, 1, 4, 8, 4) == 0
    assert _mass(32, 1, 4, 8, 512) == 32 * 8 * 4 * (8192 * 4 + 8192 // 2048 * 8)
    assert _mass(2, 64, 4, 8, 1024) == 2 * 8 * 256 * (16384 // 256 * 8 + 4)
    assert _mass(0, 1, 4, 8, 512) == 0
