"""The block-scaled cache's operators together: some ticks of tree-speculative serving with every check on.
Outputs are averages of values of size about 3 (normal draws quantised); fp16 output and fp16 p bound the
difference from fp32 attention over the same cache by 2^-11 (3 + 3 * max|v|), max|v| < 6."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("rows,layers,nodes", [(5, 2, 21), (3, 1, 64), (8, 2, 4)])
def test_ticks(cuda, dtype, rows, layers, nodes):
    from specq import tree_serve
    r = tree_serve.run(steps=12, rows=rows, layers=layers, nodes=nodes, seed=rows, check=True, dtype=dtype)
    assert r["status"] == 0 and r["missing_pages"] == 0
    assert r["forks"] == 2 and r["ended"] >= 1
    assert r["max_abs_error"] <= 2.0 ** -11 * (3 + 3 * 6)


def test_draw_tree_is_a_tree():
    import random
    from specq import tree_serve
    rng = random.Random(0)
    for n in (1, 2, 21, 64):
        depth, mask, path = tree_serve.draw_tree(rng, n)
        assert len(depth) == len(mask) == n and depth[0] == 0
        assert path == sorted(path) and path[0] == 0 and [depth[j] for j in path] == list(range(len(path)))
        for j in range(n):
            assert bin(mask[j]).count("1") == depth[j] + 1 and mask[j] >> j == 1
