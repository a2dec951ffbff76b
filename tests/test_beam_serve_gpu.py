"""The operators of heads, beams, eviction and pages run together as a server would run them."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("requests,beams,keep,dtype", [(3, 4, 96, torch.int8), (2, 2, 33, torch.float8_e4m3fn), (1, 1, 700, torch.int8)])
def test_beam_server(cuda, requests, beams, keep, dtype):
    from specq import beam_serve
    r = beam_serve.run(steps=12, requests=requests, beams=beams, layers=2, keep=keep, seed=requests, check=True, dtype=dtype)
    assert r["missing_pages"] == 0 and r["status"] == 0
    # averages of normal draws (the largest below 6): weights and output in fp16
    assert r["max_abs_error"] <= 2.0 ** -11 * (3 + 3 * 6)
    assert r["kept"] == [min(n, keep) + 12 for n in r["prompts"]]
