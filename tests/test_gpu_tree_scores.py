"""xs_tree_attend where scores are huge: keys masked by a large finite value beside keys that are
not, rows whose every score is one huge value, and scores whose logarithm to base 2 overflows.

The tolerances count only what a row's result depends on.  Keys of weight 0 in 64 bits (scores far
below the row's maximum) count for nothing, so their magnitude allows no error; and equal scores
have equal weights, whatever their magnitude, so a mean of the values is held to the rounding of
its sum and of the output alone."""
import math

import numpy as np
import pytest
import torch

from tests import treeref
from tests.test_gpu_tree_attend import BF, HF, blank, case, context, run
from tests.treeref import F32, half_step

pytestmark = pytest.mark.gpu

LOWEST = torch.finfo(BF).min


@pytest.fixture(scope="module")
def ctx():
    return context()


def one_column(c, value):
    """Scores are column 0's product plus the others'; column 0 of q is 1, of the keys `value`."""
    for t in ("k", "fk"):
        c[t][..., 0] = value
    c["q"][..., 0] = 1.0


def agree_with_the_live(c, got, scale=None):
    """As tests/treeref.py, with the error of a score counted from the keys of weight above 0: a
    product of D elements that starts from minus the reference is a sum of D + 1 terms, each at most
    the largest sum of |q k| among those keys, so it is off by (D + 5) F32 times twice that."""
    scale = float(np.float32(1.0 / math.sqrt(c["q"].shape[-1]) if scale is None else scale))
    assert got.seq_status.tolist() == [0] * len(c["lens"])
    q, k, v, fk, fv = (c[t].double().cpu() for t in ("q", "k", "v", "fk", "fv"))
    out, lse = got.out.double().cpu(), got.lse.double().cpu()
    G, D, u = q.shape[2] // k.shape[2], q.shape[3], half_step(c["q"].dtype)
    for b, n in enumerate(c["lens"]):
        for i, chain in enumerate(treeref.sees(c["parent"][b].tolist(), c["used"][b])):
            if chain is None:
                continue
            for h in range(q.shape[2]):
                g = h // G
                keys, values = torch.cat([k[b, :n, g], fk[b, chain, g]]), torch.cat([v[b, :n, g], fv[b, chain, g]])
                s = keys @ q[b, i, h] * scale
                p = torch.softmax(s, 0)
                live = p > 0
                want, around = p[live] @ values[live], p[live] @ values[live].abs()
                off = 2 * (D + 5) * F32 * float((keys[live].abs() @ q[b, i, h].abs()).max()) * abs(scale)
                off += 8 * F32 * (1 + float(s[live].abs().max()))
                tol = u * want.abs() * 1.01 + around * (u * 1.01 + 2 * off + 2 * (len(s) + 8) * F32)
                assert bool(((out[b, i, h] - want).abs() <= tol).all()), (b, i, h)
                full = float(torch.logsumexp(s, 0))
                assert abs(float(lse[b, i, h]) - full) <= off + (len(s) + 8) * F32 + 4 * F32 * abs(full), (b, i, h)


def agree_with_the_mean(c, got, value, scale=None):
    """Every score is `value` times the scale: the mean of the values that the row sees."""
    scale = float(np.float32(1.0 / math.sqrt(c["q"].shape[-1]) if scale is None else scale))
    v, fv, u = c["v"].double().cpu(), c["fv"].double().cpu(), half_step(c["q"].dtype)
    out, lse = got.out.double().cpu(), got.lse.double().cpu()
    G = c["q"].shape[2] // v.shape[2]
    for b, n in enumerate(c["lens"]):
        for i, chain in enumerate(treeref.sees(c["parent"][b].tolist(), c["used"][b])):
            if chain is None:
                continue
            values = torch.cat([v[b, :n], fv[b, chain]]).repeat_interleave(G, 1)
            many = len(values)
            want, around = values.mean(0), values.abs().mean(0)
            tol = u * want.abs() * 1.01 + around * (many + 8) * F32
            assert bool(((out[b, i] - want).abs() <= tol).all()), (b, i, float(((out[b, i] - want).abs() / tol).max()))
            full = value * scale + math.log(many)
            if abs(full) < torch.finfo(torch.float32).max:
                assert bool(((lse[b, i] - full).abs() <= 4 * F32 * (1 + abs(full))).all())


# one, two and four row tiles of a wave, and several waves that share the keys (float16 holds the
# masks as -inf)
SHAPES = [(3, 8, 2, 128, BF), (3, 4, 2, 72, BF), (8, 4, 1, 128, BF), (8, 4, 1, 200, BF), (6, 4, 1, 256, BF), (12, 4, 1, 64, BF),
          (12, 4, 1, 128, HF), (24, 4, 1, 128, BF), (40, 8, 2, 128, BF), (40, 8, 2, 72, BF), (20, 4, 1, 256, BF), (20, 4, 1, 136, HF)]


@pytest.mark.parametrize("mask", [-1e6, -1e7, -1e8, -1e9, LOWEST])
@pytest.mark.parametrize("nodes,hq,h,d,dtype", SHAPES)
def test_masked_slots_before_others(ctx, nodes, hq, h, d, dtype, mask):
    """A wave's first blocks hold masked keys only, later ones none, some or all."""
    rng = np.random.default_rng(nodes + d)
    c = case(rng, [500, 300, 161, 64, 0], nodes, hq, h, d, dtype, used=[nodes, nodes - 1, nodes, 1, nodes])
    one_column(c, 0.0)
    for b, n in enumerate((256, 130, 160, 64, 0)):
        c["k"][b, :n, :, 0] = mask
    c["k"][0, 300:340, :, 0] = mask
    c["k"][1, ::3, :, 0] = mask
    agree_with_the_live(c, run(ctx, c, out=blank(c)))


@pytest.mark.parametrize("nodes,hq", [(2, 4), (40, 8)])
def test_masked_slots_fill_whole_splits(ctx, nodes, hq):
    """Long enough for several workgroups a row: the first of them see masked keys only."""
    rng = np.random.default_rng(21)
    c = case(rng, [6000], nodes, hq, 1, 80, BF)
    one_column(c, 0.0)
    c["k"][0, :4000, :, 0] = -1e9
    c["k"][0, 5000:, :, 0] = LOWEST
    agree_with_the_live(c, run(ctx, c, out=blank(c)))


@pytest.mark.parametrize("nodes", [4, 40])
def test_masked_slots_and_a_negative_scale(ctx, nodes):
    rng = np.random.default_rng(22)
    c = case(rng, [500, 200], nodes, 8, 2, 64, BF)
    one_column(c, 0.0)
    c["k"][:, :150, :, 0] = 1e9
    agree_with_the_live(c, run(ctx, c, scale=-0.11, out=blank(c)), scale=-0.11)


@pytest.mark.parametrize("nodes", [4, 40])
def test_scores_that_climb_from_far_below(ctx, nodes):
    """Masks of ever smaller magnitude, block by block; the whole cache masked before the tree."""
    rng = np.random.default_rng(23)
    c = case(rng, [700, 500], nodes, 8, 2, 96, BF)
    one_column(c, 0.0)
    for b in range(6):
        c["k"][0, 100 * b:100 * (b + 1), :, 0] = -10.0 ** (9 - b)
    c["k"][1, :, :, 0] = -1e9
    agree_with_the_live(c, run(ctx, c, out=blank(c)))


@pytest.mark.parametrize("value", [-1e7, -1e8, -1e9, LOWEST, 1e9, -LOWEST])
@pytest.mark.parametrize("nodes,hq,h", [(5, 4, 2), (40, 8, 2)])
@pytest.mark.parametrize("d", [48, 64, 72, 80, 88, 128, 192, 240, 256])
def test_one_huge_score_for_all(ctx, d, nodes, hq, h, value):
    rng = np.random.default_rng(d)
    c = case(rng, [300, 33, 700], nodes, hq, h, d, BF)
    c["q"][:] = 0.0
    one_column(c, value)
    agree_with_the_mean(c, run(ctx, c, out=blank(c)), float(torch.tensor(value).to(BF)))


@pytest.mark.parametrize("value", [torch.finfo(HF).min, torch.finfo(HF).max])
@pytest.mark.parametrize("nodes", [5, 40])
def test_one_huge_score_for_all_f16(ctx, nodes, value):
    rng = np.random.default_rng(24)
    c = case(rng, [300, 33, 700], nodes, 8, 2, 72, HF)
    c["q"][:] = 0.0
    one_column(c, value)
    agree_with_the_mean(c, run(ctx, c, out=blank(c)), value)


@pytest.mark.parametrize("scale", [0.72, 1.0, -0.9, 4.0])
@pytest.mark.parametrize("nodes", [5, 40])
def test_scores_past_the_base_2_range(ctx, nodes, scale):
    """The lowest value times the scale is an f32; times log2(e) it is not."""
    rng = np.random.default_rng(25)
    c = case(rng, [300, 33, 3000], nodes, 8, 2, 64, BF)
    c["q"][:] = 0.0
    one_column(c, LOWEST)
    agree_with_the_mean(c, run(ctx, c, scale=scale, out=blank(c)), LOWEST, scale=scale)


@pytest.mark.parametrize("lens", [[50, 0, 300], [6000]])
@pytest.mark.parametrize("nodes", [5, 40])
def test_empty_rows_that_see_odd_values(ctx, nodes, lens):
    """Every score is -inf: out is 0 and lse -inf, also where the values seen are NaN or infinite."""
    rng = np.random.default_rng(26)
    c = case(rng, lens, nodes, 8, 2, 64, BF)
    one_column(c, -math.inf)
    c["fv"][:, 0, :, 3] = math.nan
    c["fv"][:, 2, :, 7] = math.inf
    c["v"][:, 7, :, 5] = math.nan
    got = run(ctx, c, out=blank(c))
    assert bool((got.out == 0.0).all()) and bool((got.lse == -math.inf).all())


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("nodes,lens", [(5, [70, 300, 1000]), (40, [70, 300, 1000]), (9, [7000])])
def test_values_at_the_end_of_the_type(ctx, nodes, lens, dtype):
    """A mean of finite values is finite: rounded weights over their exact sum may pass the largest
    value by half a step of the type, which must not become an infinity.  (bf16's largest over 2^20:
    sums of weights times values are f32, of weights up to 2^8.)"""
    rng = np.random.default_rng(27)
    c = case(rng, lens, nodes, 8, 2, 64, dtype, spread=2.0)
    top = torch.finfo(dtype).max * (1.0 if dtype == HF else 2.0**-20)
    for t in ("v", "fv"):
        c[t][..., ::2], c[t][..., 1::2] = top, -top
    got = run(ctx, c, out=blank(c)).out.double().cpu()
    want = torch.tensor([top, -top], dtype=torch.float64).repeat(32)
    for b, n in enumerate(c["lens"]):
        for i, chain in enumerate(treeref.sees(c["parent"][b].tolist(), c["used"][b])):
            # a rounded weight and the rounded output, and the sums
            assert bool(((got[b, i] - want).abs() <= top * (2.02 * half_step(dtype) + (n + 64) * F32)).all())
