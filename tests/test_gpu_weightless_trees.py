"""Values that are not finite reach the rows that give them weight and no others: masked slots and
nodes whose values hold infinities and NaN, in xs_tree_attend and xs_tree_attend8."""
import math

import numpy as np
import pytest
import torch

from tests import treeref
from tests.test_gpu_cache8 import empty_cache, filled, look, put, step
from tests.test_gpu_tree_attend import blank, case, run
from tests.test_gpu_weightless_values import BF, HF, INF, LOWS, agree, definition, spoil

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from xwen_amd import tree
    return tree.CacheContext(max_seqs=8, max_nodes=64, q_heads=32, kv_heads=4, head_dim=256, capacity=8192)


def sight(parent, n, length):
    """Of the nodes [n, length + n]: the cache's slots, and what treeref.sees gives."""
    m = torch.zeros((n, length + n), dtype=torch.bool)
    for i, c in enumerate(treeref.sees(parent, n)):
        if c is not None:
            m[i, :length] = True
            m[i, [length + j for j in c]] = True
    return m.cuda()


def check_trees(got, q, k, v, lens, fk, fv, parent, used):
    """k, v: what the caches hold, by sequence [slots, heads, size]."""
    scale = float(np.float32(1 / math.sqrt(q.shape[-1])))
    HQ, H = q.shape[2], fk.shape[2]
    for b, n in enumerate(used):
        seen = sight(parent[b].tolist(), n, lens[b])
        for h in range(0, HQ, max(1, HQ // 4)):
            o = h // (HQ // H)
            keys = torch.cat([k[b][:lens[b], o].double(), fk[b, :n, o].double()])
            values = torch.cat([v[b][:lens[b], o].double(), fv[b, :n, o].double()])
            agree(got.out[b, :n, h], got.lse[b, :n, h], definition(q[b, :n, h], keys, values, seen, scale), (b, h))


SHAPES = [(1, 1), (5, 3), (10, 3), (12, 4), (24, 4), (50, 4)]  # nodes, query heads of a kv head
LENS = [0, 45, 700, 5000]


def masked_nodes(c, name, low, g):
    """Every third node masked, its values spoilt; node 2's infinite value counts."""
    n = c["q"].shape[1]
    c["q"][..., 0] = 1.0
    c["fk"][..., 0] = 0.0
    for b in range(len(LENS)):
        for i in range(0, n, 3):
            c["fk"][b, i, :, 0] = low
            spoil(c["fv"][b], [i], g)
        if n > 2:
            c["fv"][b, 2, :, 13] = INF


@pytest.mark.parametrize("dtype,low", LOWS)
@pytest.mark.parametrize("d", [64, 72, 128, 256])
@pytest.mark.parametrize("nodes,group", SHAPES)
def test_trees_over_16_bits(ctx, nodes, group, d, dtype, low):
    rng = np.random.default_rng(nodes * d)
    g = torch.Generator().manual_seed(nodes + d)
    c = case(rng, LENS, nodes, 2 * group, 2, d, dtype)
    masked_nodes(c, "v", low, g)
    c["k"][..., 0] = 0.0
    for b, n in enumerate(LENS):
        at = sorted({i for i in (0, 1, 31, 32, 40, 100, 333, 640, 699, 2000, 3333, 4990, 4999) if i < n})
        c["k"][b, at, :, 0] = low
        spoil(c["v"][b], at, g)
    c["v"][2, 350, :, 8], c["v"][3, 4100, :, 9] = -INF, math.nan  # these have weight
    got = run(ctx, c, out=blank(c))
    assert got.seq_status.tolist() == [0] * 4
    check_trees(got, c["q"], c["k"], c["v"], LENS, c["fk"], c["fv"], c["parent"], c["used"])


@pytest.mark.parametrize("dtype,low", LOWS)
@pytest.mark.parametrize("d", [64, 80, 128, 256])
@pytest.mark.parametrize("nodes,group", SHAPES)
def test_trees_over_8_bits(ctx, nodes, group, d, dtype, low):
    """(A key of -inf cannot be held in 8 bits: the cache's masked keys hold a finite one.)"""
    rng = np.random.default_rng(nodes * d)
    g = torch.Generator().manual_seed(nodes + d)
    c = empty_cache([0] * 4, 2, d, 5024)
    rows = [(torch.randn((4, 5000, 2, d), generator=g)).to(dtype).cuda() for _ in "kv"]
    rows[0][..., 0] = 0.0
    for b, n in enumerate(LENS):
        at = sorted({i for i in (0, 1, 31, 32, 40, 100, 333, 640, 699, 2000, 3333, 4990, 4999) if i < n})
        rows[0][b, at, :, 0] = low if low > -INF else -60000.0
        spoil(rows[1][b], at, g)
        if dtype == BF and n:
            rows[1][b, at[-1], :, 1] = torch.finfo(BF).max  # held as an infinity
    rows[1][2, 350, :, 8], rows[1][3, 4100, :, 9] = -INF, math.nan  # these have weight
    got = put(ctx, c, *rows, n_path=torch.tensor(LENS, dtype=torch.int32).cuda())
    assert got.seq_status.tolist() == [0] * 4 and got.new_len.tolist() == LENS
    c["len"] = got.new_len
    s = step(rng, c, nodes, 2 * group, dtype)
    masked_nodes(s, "fv", low, g)
    got = look(ctx, c, s)
    assert got.seq_status.tolist() == [0] * 4
    held = []
    for n in "kv":
        e = (c[n + "_exp"].int() - 127).repeat_interleave(32, 2)[:, :, :5024].transpose(1, 2)[..., None]
        x = c[n].double() * torch.exp2(e.double())
        held.append(torch.where(x.abs() >= 2.0**128, torch.copysign(torch.full_like(x, INF), x), x))
    check_trees(got, s["q"], *held, LENS, s["fk"], s["fv"], s["parent"], s["used"])


@pytest.mark.parametrize("nodes,group,d", [(5, 3, 64), (12, 4, 128), (24, 4, 128), (50, 4, 256)])
def test_rows_of_nan_beside(ctx, nodes, group, d):
    """A NaN query's row, and rows whose masked tokens' values are not finite, in one tile."""
    rng = np.random.default_rng(nodes)
    g = torch.Generator().manual_seed(nodes)
    c = case(rng, LENS, nodes, 2 * group, 2, d, BF)
    masked_nodes(c, "v", -INF, g)
    c["q"][:, nodes // 2, 1, 5] = math.nan
    got = run(ctx, c, out=blank(c))
    check_trees(got, c["q"], c["k"], c["v"], LENS, c["fk"], c["fv"], c["parent"], c["used"])


@pytest.mark.parametrize("nodes,group", [(1, 4), (12, 4), (50, 4)])
def test_a_graph_replays_with_values_that_come_and_go(ctx, nodes, group):
    """Captured with finite values; replayed with NaN and infinities in the cache, then without."""
    from xwen_amd import cache8, tree
    rng = np.random.default_rng(nodes)
    c = filled([4000, 70], 2, 128, seed=nodes)
    s = step(rng, c, nodes, 2 * group, BF)
    s["q"][..., 0], s["fk"][..., 0] = 1.0, 0.0
    clean = look(ctx, c, s)
    out = tree.Attended(*(torch.zeros_like(t) for t in (clean.out, clean.lse, clean.seq_status)))
    parent = s["parent"].cuda()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache8.tree_attend8(ctx, s["q"], c["k"], c["v"], c["k_exp"], c["v_exp"], c["len"], s["fk"], s["fv"], parent, out=out)
    fine = c["v"].view(torch.uint8).clone()
    for i in range(4):
        c["v"].view(torch.uint8).copy_(fine)
        s["fv"][:, 0, :, 3] = (math.nan, 1.0, -INF, 1.0)[i]
        if i % 2 == 0:
            c["v"].view(torch.uint8)[:, 33, :, 7] = 127
        out.out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        want = look(ctx, c, s)
        same = (out.out == want.out) | (out.out.isnan() & want.out.isnan())
        assert bool(same.all()) and torch.equal(out.lse, want.lse)
        assert bool(torch.isnan(out.out[0, 0, :, 7]).all()) == (i % 2 == 0) and bool(torch.isfinite(out.out[0, 0, :, 20]).all())
        torch.cuda.synchronize()
