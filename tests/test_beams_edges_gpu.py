"""beam_select with more candidates than its merge holds in shared memory, against the float64 oracle (bounds as in test_beams_gpu.py)."""
import pytest
import torch

from oracle import bounded_oracle as O
from test_beams_gpu import FLOATS, _check, _rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("B,V", [(1, 128000), (2, 40003)])
def test_select_of_more_candidates_than_are_staged(cuda, dtype, B, V):
    """64 beams, 128 places and two slices or more a row are past 96 KB.  Beams that are finished, empty, alike, and rows of ties."""
    import specq
    K, n = 64, 128
    x, s = _rows(B, K, V, dtype, V)
    _check(specq.beam_select(x, s, n=n), x, s, n)
    x[1] = 1.5
    x[2] = torch.where(torch.arange(V, device="cuda") % 1009 == 1, 9.0, -1.0)
    x[5] = x[2]
    x[4] = -torch.inf
    x[6] = -torch.inf
    x[6, [3, V - 1]] = 0.25
    s[:, :8] = -2.0
    s[:, 7] = -torch.inf
    done = torch.zeros(B * K, dtype=torch.bool, device="cuda")
    done[[0, 7, 9]] = True
    _check(specq.beam_select(x, s, n=n, done=done, pad=V - 2), x, s, n, done, V - 2)
    # only exact ties: every index is that of the definition where the rows begin alike; rows that begin at other places of 16 bytes
    # add the same terms up in another order, so that their totals meet to the bound of lse only, within which beams have no order
    y, flat = x[2:3].repeat(B * K, 1), torch.full_like(s, -3.0)
    got = specq.beam_select(y, flat, n=n)
    _check(got, y, flat, n)
    if V * x.element_size() % 16 == 0:
        _, rp, rt = O.beam_select(y.float().cpu().numpy(), flat.cpu().numpy(), n)
        assert (got[1].cpu().numpy() == rp).all() and (got[2].cpu().numpy() == rt).all()
    # fewer candidates than places
    y[:] = -torch.inf
    y[11, V - 3] = 0.0
    done[:] = False
    done[[3, 20]] = True
    flat[:, 30] = -1.0
    _check(specq.beam_select(y, flat, n=n, done=done, pad=4), y, flat, n, done, 4)
