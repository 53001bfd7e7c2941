"""Scores of -inf in xs_tree_attend8: a token of such a score has weight 0, and a row that has no
other gets out 0 and lse -inf, whatever the queries' bits below bf16's."""
import math

import numpy as np
import pytest
import torch

from tests.test_gpu_cache8 import agree, filled, look, step

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
INF = math.inf
# exact in bf16; in float16 with a remainder above and below the nearest bf16 value
QUERIES = [1.0, 1.0 + 2.0**-9, 1.0 + 2.0**-7 - 2.0**-9]


@pytest.fixture(scope="module")
def ctx():
    from xwen_amd import tree
    return tree.CacheContext(max_seqs=8, max_nodes=64, q_heads=32, kv_heads=2, head_dim=256, capacity=4096)


def chain(n):
    return [[-1] + list(range(n - 1))] * 5


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("nodes,g", [(1, 1), (5, 3), (12, 4), (24, 4), (50, 4)])
@pytest.mark.parametrize("value", QUERIES)
def test_fresh_keys_that_hold_minus_infinity(ctx, value, nodes, g, d, dtype):
    """Tiles of 16 rows, of 32 whose keys two waves share, of 32, and eight waves of them.  One such
    key beside others, all of a row's, all but a cache's, and each other node's."""
    rng = np.random.default_rng(nodes * d)
    c = filled([70, 0, 700, 0, 3], 2, d)
    s = step(rng, c, nodes, 2 * g, dtype, parent=chain(nodes))
    s["q"][..., 0] = value
    s["fk"][0, nodes // 2, :, 0] = -INF
    s["fk"][1, :, :, 0] = -INF
    s["fk"][2, :, :, 0] = -INF
    s["fk"][3, ::2, :, 0] = -INF
    got = look(ctx, c, s)
    agree(c, s, got)
    assert bool((got.out[1] == 0).all()) and bool((got.lse[1] == -INF).all())
    assert not bool(torch.isnan(got.out).any())


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("nodes,g", [(1, 1), (5, 3), (12, 4), (24, 4), (50, 4)])
@pytest.mark.parametrize("value", QUERIES)
def test_queries_that_hold_an_infinity(ctx, value, nodes, g, dtype):
    """-inf against keys above 0, +inf against keys below: every score of the row is -inf; and +inf
    against keys above 0, which makes the row NaN."""
    rng = np.random.default_rng(nodes)
    c = filled([0, 0, 0, 0, 0], 2, 128)
    s = step(rng, c, nodes, 2 * g, dtype, parent=chain(nodes))
    s["q"][..., 0] = 1.0
    s["fk"][..., 0] = value
    i = nodes // 2
    s["q"][0, i, :, 0] = -INF
    s["fk"][1, :, :, 0] = -value
    s["q"][1, i, :, 0] = INF
    s["q"][2, i, :, 0] = INF
    got = look(ctx, c, s)
    agree(c, s, got)
    assert bool((got.out[:2, i] == 0).all()) and bool((got.lse[:2, i] == -INF).all())
    assert bool(torch.isnan(got.out[2, i]).all())
