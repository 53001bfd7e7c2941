"""xs_cache_commit's weights where scores are large: exp(scale q.k - lse) from one difference."""
import math

import numpy as np
import pytest
import torch

from tests.test_gpu_tree_attend import BF, HF, blank, case, context, run
from tests.treeref import F32

pytestmark = pytest.mark.gpu

LOWEST = torch.finfo(BF).min


@pytest.fixture(scope="module")
def ctx():
    return context()


def i32(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


def chain_case(rng, lens, nodes, m, hq, h, d, dtype):
    """A chain of nodes, the first m accepted; scores are column 0's product alone."""
    c = case(rng, lens, nodes, hq, h, d, dtype, cap=max(lens) + nodes, parent=[list(range(-1, nodes - 1))] * len(lens))
    c["q"][:] = 0.0
    c["path"], c["m"] = [list(range(nodes))] * len(lens), [m] * len(lens)
    return c


def committed(ctx, c, lse, mass, scale=None):
    from xwen_amd import tree
    new = torch.full_like(mass, -5.0)
    got = tree.cache_commit(ctx, c["k"], c["v"], i32(c["lens"]), c["fk"], c["fv"], i32(c["path"]), i32(c["m"]), q=c["q"], lse=lse,
                            mass=mass, new_mass=new, scale=scale)
    assert got.seq_status.tolist() == [0] * len(c["lens"])
    return new


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("nodes,m,hq,h,d", [(1, 1, 1, 1, 64), (6, 5, 4, 2, 72), (24, 20, 8, 2, 128), (40, 30, 8, 2, 64)])
def test_large_scores_lose_nothing(ctx, nodes, m, hq, h, d, dtype):
    """Products that are whole numbers, a scale of 1/4 and lse given in halves: every exponent is
    y = scale q.k - lse exactly.  A term is off by the roundings of log2(e) and of y times it, and
    exp2's last place: (2 |y| + 2) F32 of it; the sum of n terms by n F32 more.  A term below f32's
    least normal value may come out as 0, which is off by less than 2^-126."""
    rng = np.random.default_rng(nodes + d)
    c = chain_case(rng, [70, 200, 0], nodes, m, hq, h, d, dtype)
    b, G = 3, hq // h
    c["q"][..., 0] = 48.0
    k0 = torch.from_numpy(rng.integers(70, 90, (b, c["k"].shape[1], h)).astype(np.float32)).cuda()
    f0 = torch.from_numpy(rng.integers(70, 90, (b, nodes, h)).astype(np.float32)).cuda()
    c["k"][..., 0], c["fk"][..., 0] = k0.to(dtype), f0.to(dtype)
    lse = torch.from_numpy(1080.0 + 0.5 * rng.integers(0, 40, (b, nodes, hq)).astype(np.float32)).cuda()
    mass = torch.zeros((b, h, c["k"].shape[1]), device="cuda")
    got = committed(ctx, c, lse, mass, scale=0.25).double().cpu()
    for x, n in enumerate(c["lens"]):
        keys = torch.cat([k0[x, :n], f0[x, :m]]).double().cpu()             # [slots, kv heads]
        y = 12.0 * keys[:, :, None, None] - lse[x, :m].double().cpu().view(m, h, G).permute(1, 2, 0)[None]
        sees = torch.arange(m)[None] >= torch.arange(n + m)[:, None] - n     # [slots, ranks]
        term = y.exp() * sees[:, None, None]
        want = term.sum((2, 3)).T
        tol = (term * (2 * y.abs() + 2 + m * G) * F32 * 1.01 + 2.0**-126).sum((2, 3)).T
        off = (got[x, :, :n + m] - want).abs()
        assert bool((off <= tol).all()), float((off / tol).max())


@pytest.mark.parametrize("value", [-1e6, -1e7, -1e8, -1e9, LOWEST, 1e9])
@pytest.mark.parametrize("nodes,hq,h,d", [(1, 4, 2, 128), (7, 4, 2, 72), (40, 8, 2, 80)])
def test_one_huge_score_for_all_stays_in_bounds(ctx, nodes, hq, h, d, value):
    """lse as an f32 says nothing about such a row's weights (each 1 / n), but that none is above 1:
    whatever the rounding of the two huge terms leaves, no slot gains more than one a row."""
    rng = np.random.default_rng(d)
    m = max(1, nodes - 2)
    c = chain_case(rng, [300, 33, 0], nodes, m, hq, h, d, BF)
    c["q"][..., 0] = 1.0
    c["k"][..., 0] = c["fk"][..., 0] = value
    lse = run(ctx, c, out=blank(c)).lse
    mass = torch.rand((3, h, c["k"].shape[1]), device="cuda")
    got = committed(ctx, c, lse, mass).double().cpu()
    rows, old = m * hq // h, mass.double().cpu()
    for b, n in enumerate(c["lens"]):
        top = old[b, :, :n] + rows
        assert bool((got[b, :, :n] >= old[b, :, :n]).all()) and bool((got[b, :, :n] <= top * (1 + (rows + 2) * F32)).all())
        fresh = got[b, :, n:n + m]
        assert bool((fresh >= 0).all()) and bool((fresh <= rows * (1 + (rows + 2) * F32)).all())


def test_a_path_that_is_no_chain_keeps_its_weights(ctx):
    """A node that the row's lse does not count may weigh more than 1: exp(scale q.k - lse) as it is."""
    rng = np.random.default_rng(3)
    c = chain_case(rng, [40], 4, 4, 2, 1, 64, BF)
    c["parent"] = torch.tensor([[-1, 0, 0, 0]], dtype=torch.int32)
    c["q"][..., 0] = 1.0
    c["k"][..., 0] = 0.0
    c["fk"][..., 0] = torch.tensor([0.0, 64.0, 0.0, 0.0], device="cuda")[None, :, None]
    lse = run(ctx, c, scale=0.25, out=blank(c)).lse
    got = committed(ctx, c, lse, torch.zeros((1, 1, c["k"].shape[1]), device="cuda"), scale=0.25)
    ln = lse.double().cpu()[0]
    want = sum(float((16.0 - ln[i]).exp().sum()) for i in (1, 2, 3))  # nodes 2 and 3 do not see node 1
    assert want > 1e5 and abs(float(got[0, 0, 41]) - want) <= 60 * F32 * want
