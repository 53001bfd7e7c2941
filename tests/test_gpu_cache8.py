"""xs_cache_append8 and xs_tree_attend8 on the device against their definitions in 64 bits
(tests/promptref.py, tests/treeref.py)."""
import math

import numpy as np
import pytest
import torch

from tests import promptref, treeref
from tests.test_gpu_tree_attend import random_tree

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
F8 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def ctx():
    from xwen_amd import tree
    return tree.CacheContext(max_seqs=64, max_nodes=64, q_heads=32, kv_heads=16, head_dim=256, capacity=8192)


def empty_cache(lens, h, d, cap, layout="slot", seed=0):
    """Caches whose bytes are noise (no NaN) and whose exponents are small, `lens` slots in use."""
    g = torch.Generator().manual_seed(seed + cap)
    b = len(lens)
    shape = {"slot": (b, cap, h, d), "head": (b, h, cap, d), "seq_last": (cap, b, h, d)}[layout]
    back = {"slot": (0, 1, 2, 3), "head": (0, 2, 1, 3), "seq_last": (1, 0, 2, 3)}[layout]
    c = {}
    for n in "kv":
        byte = torch.randint(0, 255, shape, generator=g).to(torch.uint8)
        byte[(byte & 127) == 127] = 0
        c[n] = byte.cuda().view(F8).permute(back)
        c[n + "_exp"] = (torch.randint(-9, -4, (b, h, (cap + 31) // 32), generator=g) + 127).to(torch.uint8).cuda()
    c["len"] = torch.tensor(lens, dtype=torch.int32).cuda()
    c["ref"] = promptref.Cache(c["k"], c["v"], c["k_exp"], c["v_exp"], lens)
    return c


def put(ctx, c, fk, fv, **kw):
    from xwen_amd import cache8
    return cache8.cache_append8(ctx, c["k"], c["v"], c["k_exp"], c["v_exp"], c["len"], fk, fv, **kw)


def same(c, got, lens, status=None):
    assert got.new_len.tolist() == lens and got.seq_status.tolist() == (status or [0] * len(lens))
    c["ref"].check(c["k"], c["v"], c["k_exp"], c["v_exp"])


def fresh(g, *shape, dtype=BF, spread=1.0):
    return [(torch.randn(shape, generator=g) * spread).to(dtype).cuda() for _ in "kv"]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d", [16, 48, 64, 80, 128, 144, 256])
def test_append_prompts(ctx, d, dtype):
    """Packed prompts after what is there, block edges and partly used blocks among them."""
    g = torch.Generator().manual_seed(d)
    lens, new = [0, 31, 32, 40, 5, 63], [70, 1, 33, 0, 27, 129]
    c = empty_cache(lens, 3, d, 250, layout="head" if d == 80 else "slot")
    start = np.concatenate([[0], np.cumsum(new)])
    fk, fv = fresh(g, int(start[-1]), 3, d, dtype=dtype, spread=3.0)
    got = put(ctx, c, fk, fv, start=torch.tensor(start, dtype=torch.int32).cuda())
    for b, (i, j) in enumerate(zip(start, start[1:])):
        c["ref"].append(b, fk[i:j], fv[i:j])
    same(c, got, [a + b for a, b in zip(lens, new)])


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("spread", [1e-3, 1.0, 60.0])
def test_append_steps(ctx, spread, dtype):
    """A path's rows at a time, so that blocks fill over several calls and scales grow."""
    rng = np.random.default_rng(5)
    g = torch.Generator().manual_seed(5)
    lens = [0, 3, 30, 33]
    c = empty_cache(lens, 2, 64, 100, layout="seq_last")
    for step in range(6):
        fk, fv = fresh(g, 4, 9, 2, 64, dtype=dtype, spread=spread * 2.0**(step % 3 * 2))
        n = rng.integers(0, 10, 4)
        path = np.full((4, 9), -1, np.int32)
        for b in range(4):
            path[b, :n[b]] = rng.integers(0, 9, n[b])
        got = put(ctx, c, fk, fv, path=torch.from_numpy(path).cuda(), n_path=torch.tensor(n, dtype=torch.int32).cuda())
        for b in range(4):
            c["ref"].append(b, fk[b, path[b, :n[b]].tolist()], fv[b, path[b, :n[b]].tolist()])
        lens = [a + int(m) for a, m in zip(lens, n)]
        same(c, got, lens)
        c["len"] = got.new_len


def test_append_without_a_path(ctx):
    g = torch.Generator().manual_seed(1)
    c = empty_cache([0, 20], 2, 32, 64)
    fk, fv = fresh(g, 2, 7, 2, 32)
    c["len"] = put(ctx, c, fk, fv).new_len
    for b in range(2):
        c["ref"].append(b, fk[b], fv[b])
    got = put(ctx, c, fk, fv, n_path=torch.tensor([3, 0], dtype=torch.int32).cuda())
    c["ref"].append(0, fk[0, :3], fv[0, :3])
    same(c, got, [10, 27])


def test_append_values_at_the_borders(ctx):
    """Zeros, the least and the largest of a type, halves between two e4m3 values, 448 and its
    neighbours, and what is not finite."""
    for dtype in (BF, HF):
        big = torch.finfo(dtype).max
        tiny = 2.0**-24 if dtype == HF else 2.0**-133
        x = torch.zeros((1, 160, 1, 16))
        x[0, 32:64] = torch.tensor([448.0, 447.0, 1.0625, 1.1875, 1.3125, 0.0029296875, 2.0**-9, 2.0**-10, 1.5 * 2**-9, -1.0625, 17, 19, 2.0**-6,
                                    15 * 2.0**-9, 0.0, -0.0])
        x[0, 64:96] = 450.0
        x[0, 65] = 225.0
        x[0, 96:128] = big
        x[0, 97] = tiny
        x[0, 128:160] = tiny
        x[0, 130, 0, 1], x[0, 131, 0, 2], x[0, 132, 0, 3] = math.nan, math.inf, -math.inf
        fk = x.to(dtype).cuda()
        c = empty_cache([0], 1, 16, 160)
        got = put(ctx, c, fk, fk.flip(1))
        c["ref"].append(0, fk[0], fk.flip(1)[0])
        same(c, got, [160])


def test_append_failures(ctx):
    g = torch.Generator().manual_seed(2)
    fk, fv = fresh(g, 7, 4, 2, 64)
    lens = [10, 62, -1, 65, 10, 10, 60]
    c = empty_cache([0] * 7, 2, 64, 64)
    c["ref"].lens = [0] * 7
    c["len"] = torch.tensor(lens, dtype=torch.int32).cuda()
    path = torch.zeros((7, 4), dtype=torch.int32)
    path[4, 2], path[5, 3] = 4, -1
    n = torch.tensor([5, 3, 1, 0, 3, 3, 4], dtype=torch.int32)
    before = {f: c[f].clone() for f in ("k", "v", "k_exp", "v_exp")}
    got = put(ctx, c, fk, fv, path=path.cuda(), n_path=n.cuda())
    assert got.seq_status.tolist() == [7, 10, 7, 7, 7, 0, 0]
    assert got.new_len.tolist() == [10, 62, -1, 65, 10, 13, 64]
    for f, t in before.items():
        now = c[f]
        assert torch.equal(now[:5].contiguous().view(torch.uint8), t[:5].contiguous().view(torch.uint8)), f
    # starts: past the rows, backwards, below 0, more than `rows`; two sequences may share rows
    c = empty_cache([0] * 5, 2, 64, 64)
    flat = fk.flatten(0, 1), fv.flatten(0, 1)
    got = put(ctx, c, *flat, start=torch.tensor([0, 5, 3, 28, 29, -1], dtype=torch.int32).cuda())
    assert got.seq_status.tolist() == [0, 7, 0, 7, 7]
    got = put(ctx, c, *flat, start=torch.tensor([0, 5, 6, 20, 28, 28], dtype=torch.int32).cuda(), rows=6)
    assert got.seq_status.tolist() == [0, 0, 7, 7, 0]


def test_append_leaves_the_rest(ctx):
    """Bytes past the new length, other blocks' scales, and rows between the strides."""
    g = torch.Generator().manual_seed(3)
    wide = torch.randint(0, 100, (2, 64, 2, 48), generator=g).to(torch.uint8).cuda()
    c = empty_cache([33, 2], 2, 32, 64)
    c["k"] = wide.view(F8)[:, :, :, :32]
    c["v"] = wide.clone().view(F8)[:, :, :, :32]
    c["ref"] = promptref.Cache(c["k"], c["v"], c["k_exp"], c["v_exp"], [33, 2])
    exps = c["k_exp"].clone()
    fk, fv = fresh(g, 2, 5, 2, 32)
    before = wide.clone()
    got = put(ctx, c, fk, fv)
    for b in range(2):
        c["ref"].append(b, fk[b], fv[b])
    same(c, got, [38, 7])
    assert torch.equal(wide[..., 32:], before[..., 32:]) and torch.equal(c["k_exp"][0, :, 0], exps[0, :, 0])
    assert torch.equal(c["k_exp"][1, :, 1], exps[1, :, 1])


# ---------------------------------------------------------------------------
# Attention


def filled(lens, h, d, cap=None, layout="slot", seed=0, spread=1.0):
    """A cache of normal values, quantised by the definition."""
    c = empty_cache([0] * len(lens), h, d, cap or max(lens) + 5, layout=layout, seed=seed)
    g = torch.Generator().manual_seed(seed + 1)
    ref = c["ref"]
    for b, n in enumerate(lens):
        nb = (n + 31) // 32
        for i, (name, s) in enumerate((("k", spread), ("v", 1.0))):
            x = torch.randn((nb * 32, h, d), generator=g, dtype=torch.float64) * s
            top = x.view(nb, 32, h, d).abs().amax((1, 3)) if nb else torch.zeros((0, h), dtype=torch.float64)
            e = torch.ceil(torch.log2(top / 448)).int()
            y = promptref.nearest_e4m3(x * torch.exp2(-e.double()).repeat_interleave(32, 0)[:, :, None])[:n]
            c[name][b, :n] = y.float().to(F8).cuda()
            c[name + "_exp"][b, :, :nb] = (e.T + 127).to(torch.uint8).cuda()
    c["len"] = torch.tensor(lens, dtype=torch.int32).cuda()
    c["ref"] = promptref.Cache(c["k"], c["v"], c["k_exp"], c["v_exp"], lens)
    return c


def step(rng, c, nodes, hq, dtype, used=None, parent=None, spread=1.0):
    b, cap, h, d = c["k"].shape
    g = torch.Generator().manual_seed(int(rng.integers(1 << 30)))
    fk, fv = fresh(g, b, nodes, h, d, dtype=dtype)
    if parent is None:
        parent = [random_tree(rng, nodes, roots=True) for _ in range(b)]
    return dict(q=(torch.randn((b, nodes, hq, d), generator=g) * spread).to(dtype).cuda(), fk=fk, fv=fv,
                parent=torch.tensor(parent, dtype=torch.int32), used=used or [nodes] * b)


def look(ctx, c, s, scale=None, max_len=0, fill=7.0):
    from xwen_amd import cache8, tree
    b, n, hq, d = s["q"].shape
    out = tree.Attended(out=torch.full((b, n, hq, d), fill, dtype=s["q"].dtype, device="cuda"),
                        lse=torch.full((b, n, hq), fill, device="cuda"), seq_status=torch.full((b,), -1, dtype=torch.int32, device="cuda"))
    return cache8.tree_attend8(ctx, s["q"], c["k"], c["v"], c["k_exp"], c["v_exp"], c["len"], s["fk"], s["fv"], s["parent"].cuda(),
                               n_nodes=torch.tensor(s["used"], dtype=torch.int32).cuda(), scale=scale, max_len=max_len, out=out)


def agree(c, s, got, scale=None):
    scale = float(np.float32(1.0 / math.sqrt(s["q"].shape[-1]) if scale is None else scale))
    assert got.seq_status.tolist() == [0] * len(c["ref"].lens)
    k, v = c["ref"].values()
    want = treeref.attend(s["q"], k, v, c["ref"].lens, s["fk"], s["fv"], s["parent"], s["used"], scale)
    promptref.agree(got.out, got.lse, want, left=7.0)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d", [16, 64, 80, 128, 144, 256])
def test_attend_head_sizes(ctx, d, dtype):
    rng = np.random.default_rng(d)
    c = filled([0, 1, 33, 130, 517], 2, d)
    s = step(rng, c, 9, 8, dtype, used=[9, 1, 8, 0, 5])
    agree(c, s, look(ctx, c, s))


@pytest.mark.parametrize("hq,h", [(1, 1), (3, 3), (4, 1), (7, 1), (10, 2), (16, 1), (24, 8), (32, 1), (32, 16)])
def test_attend_head_layouts(ctx, hq, h):
    rng = np.random.default_rng(hq * 64 + h)
    c = filled([70, 5], h, 64)
    s = step(rng, c, 4, hq, BF)
    agree(c, s, look(ctx, c, s))


@pytest.mark.parametrize("nodes", [1, 2, 15, 16, 17, 31, 33, 48, 63, 64])
@pytest.mark.parametrize("g,dtype", [(1, BF), (4, HF), (5, BF)])
def test_attend_tree_sizes(ctx, nodes, g, dtype):
    rng = np.random.default_rng(nodes * 8 + g)
    c = filled([300, 0], 2, 64)
    s = step(rng, c, nodes, 2 * g, dtype, used=[nodes, max(1, nodes - 2)])
    agree(c, s, look(ctx, c, s))


@pytest.mark.parametrize("nodes,dtype", [(1, BF), (6, HF)])
def test_attend_lengths(ctx, nodes, dtype):
    rng = np.random.default_rng(nodes)
    lens = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 512, 513, 1023, 1025, 2047, 2500]
    c = filled(lens, 2, 128)
    s = step(rng, c, nodes, 4, dtype)
    agree(c, s, look(ctx, c, s))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("nodes,hq,h,d", [(1, 8, 2, 128), (40, 8, 2, 128), (64, 16, 2, 64), (20, 16, 2, 256)])
def test_attend_long(ctx, nodes, hq, h, d, dtype):
    """Long enough for several workgroups a row, with large scores."""
    rng = np.random.default_rng(nodes)
    c = filled([8000, 3001], h, d, spread=1.7, layout="head")
    s = step(rng, c, nodes, hq, dtype, spread=1.7)
    agree(c, s, look(ctx, c, s))
    agree(c, s, look(ctx, c, s, max_len=8000))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("nodes,g,d", [(43, 3, 128), (64, 4, 80), (52, 5, 96), (64, 6, 112), (64, 8, 128), (64, 4, 64)])
def test_attend_many_rows(ctx, nodes, g, d, dtype):
    """129 to 512 rows of a head, odd and even numbers of 128 of them, with an infinity that one row sees."""
    rng = np.random.default_rng(nodes * g + d)
    c = filled([2600, 0, 63, 700], 2, d)
    s = step(rng, c, nodes, 2 * g, dtype, used=[nodes, nodes, nodes - 1, nodes // 2])
    s["fv"][:, nodes - 1, :, ::2] = math.inf
    agree(c, s, look(ctx, c, s))


@pytest.mark.parametrize("nodes", [1, 5, 20])
@pytest.mark.parametrize("seqs,h", [(70, 1), (64, 16), (300, 1)])
def test_attend_many_sequences(seqs, h, nodes):
    """More than a wave of them, as many as the device has places, and too many to be split; long and
    short ones, empty and failing ones among them."""
    from xwen_amd import tree
    big = tree.CacheContext(max_seqs=seqs, max_nodes=nodes, q_heads=4 * h, kv_heads=h, head_dim=64, capacity=1600)
    rng = np.random.default_rng(seqs + nodes)
    lens = rng.integers(0, 40, seqs).tolist()
    lens[3], lens[seqs // 2], lens[-1] = 1500, 700, 600
    c = filled(lens, h, 64, cap=1600)
    used = rng.integers(0, nodes + 1, seqs).tolist()
    used[3], used[seqs // 2], used[-1] = nodes, nodes, 1
    s = step(rng, c, nodes, 4 * h, BF, used=used)
    agree(c, s, look(big, c, s))
    got, bad = look(big, c, s), seqs // 2 - 1
    c["len"][bad], c["len"][5] = -1, 1601
    again = look(big, c, s)
    assert [i for i, x in enumerate(again.seq_status.tolist()) if x] == sorted([5, bad])
    # the others' shares may be cut elsewhere now: two roundings of a mean of values below 4 in
    # bf16 (2^-8 of it at most each), and of its weights (as much again, averaged)
    keep = [i for i in range(seqs) if i not in (5, bad)]
    assert bool((again.out[5] == 7).all()) and bool(((again.out[keep].float() - got.out[keep].float()).abs() <= 2.0**-5).all())


@pytest.mark.parametrize("dtype", [BF, HF])
def test_attend_scales_of_any_size(ctx, dtype):
    """Blocks whose values differ by many powers of two (past f16's range), keys' and values'."""
    rng = np.random.default_rng(9)
    c = filled([200, 64], 2, 64)
    e = torch.tensor([-9, 8, -20, 3, -60, 20, -7], dtype=torch.int32) + 127
    c["v_exp"][0] = e[:c["v_exp"].shape[2]].to(torch.uint8).cuda()
    c["k_exp"][0, :, :4] = (torch.tensor([-9, -14, -30, -8]) + 127).to(torch.uint8).cuda()
    c["ref"] = promptref.Cache(c["k"], c["v"], c["k_exp"], c["v_exp"], [200, 64])
    s = step(rng, c, 5, 4, dtype)
    got = look(ctx, c, s)
    if dtype == HF:  # a mean past 65520, half a step beyond f16's end, is an infinity
        k, v = c["ref"].values()
        out, lse, tol, ltol = treeref.attend(s["q"], k, v, [200, 64], s["fk"], s["fv"], s["parent"], s["used"], float(np.float32(0.125)))
        o = got.out.double().cpu()
        near = (o - out).abs() <= tol
        past = (out.abs() + tol >= 65520) & (o == torch.copysign(torch.tensor(math.inf, dtype=torch.float64), out))
        assert bool((near | past).all()) and bool(past.any()) and not bool(past[1].any())
    else:
        agree(c, s, got)


def test_attend_what_is_not_seen(ctx):
    """NaN bytes past the length, in unused blocks and in other branches."""
    rng = np.random.default_rng(10)
    c = filled([45, 64], 2, 64)
    s = step(rng, c, 8, 4, BF, parent=[[-1, 0, 0, 1, 1, 2, 2, 0]] * 2)
    clean = look(ctx, c, s)
    for n in "kv":
        c[n].view(torch.uint8)[0, 45:] = 127
        c[n].view(torch.uint8)[1, 64:] = 255
    s["fk"][:, 6], s["fv"][:, 6] = math.nan, math.inf
    got = look(ctx, c, s)
    seen = [0, 1, 2, 3, 4, 5, 7]
    assert torch.equal(got.out[:, seen], clean.out[:, seen]) and torch.equal(got.lse[:, seen], clean.lse[:, seen])
    assert bool(torch.isnan(got.out[:, 6]).all())


@pytest.mark.parametrize("dtype", [BF, HF])
def test_attend_fresh_values_that_are_not_finite(ctx, dtype):
    rng = np.random.default_rng(11)
    c = filled([40], 1, 64)
    s = step(rng, c, 40, 2, dtype, parent=[[-1] + list(range(39))])
    s["fv"][0, 3, 0, 5], s["fv"][0, 35, 0, 6] = math.inf, math.nan
    got = look(ctx, c, s)
    agree(c, s, got)
    assert bool((got.out[0, 3:, :, 5] == math.inf).all()) and bool(torch.isfinite(got.out[0, :3]).all())


def test_attend_nan_in_the_cache(ctx):
    rng = np.random.default_rng(12)
    c = filled([100, 100], 2, 64)
    c["k"].view(torch.uint8)[0, 70, 1, 3] = 127
    c["v"].view(torch.uint8)[0, 20, 0, 9] = 255
    c["ref"] = promptref.Cache(c["k"], c["v"], c["k_exp"], c["v_exp"], [100, 100])
    s = step(rng, c, 3, 4, HF)
    agree(c, s, look(ctx, c, s))


def test_attend_rows_that_see_nothing(ctx):
    rng = np.random.default_rng(13)
    c = filled([50, 0], 2, 64)
    s = step(rng, c, 5, 4, BF, parent=[[-1, 1, 0, 9, -2], [-1, 0, -7, 2, 1]])
    got = look(ctx, c, s)
    agree(c, s, got)
    assert bool((got.lse[0, 1] == -math.inf).all()) and bool((got.out[0, 1] == 0).all())


@pytest.mark.parametrize("low", [-1e30, -3e37])
def test_attend_masked_by_a_huge_value(ctx, low):
    """Keys that a huge finite element masks, before others and all of a row's."""
    rng = np.random.default_rng(14)
    c = empty_cache([0, 0], 1, 64, 200)
    g = torch.Generator().manual_seed(4)
    fk, fv = fresh(g, 2, 200, 1, 64)
    fk[:, :, :, 0] = 0.0
    fk[:, :64, :, 0] = low
    fk[1, :, :, 0] = low
    got = put(ctx, c, fk, fv)
    for b in range(2):
        c["ref"].append(b, fk[b], fv[b])
    same(c, got, [200, 200])
    c["len"] = got.new_len
    s = step(rng, c, 3, 2, BF)
    s["q"][..., 0] = 1.0
    agree(c, s, look(ctx, c, s))


def test_attend_bad_sequences(ctx):
    rng = np.random.default_rng(15)
    c = filled([50, 60, 70, 80], 2, 64, cap=96)
    s = step(rng, c, 4, 4, BF, used=[4, 5, 4, -1])
    c["len"] = torch.tensor([50, 60, 97, 80], dtype=torch.int32).cuda()
    got = look(ctx, c, s)
    assert got.seq_status.tolist() == [0, 7, 7, 7] and bool((got.out[1:] == 7).all()) and bool((got.lse[1:] == 7).all())
    got = look(ctx, c, s, max_len=49)
    assert got.seq_status.tolist() == [7, 7, 7, 7]


@pytest.mark.parametrize("scale", [-0.2, 0.0, 2.0])
def test_attend_scales(ctx, scale):
    rng = np.random.default_rng(16)
    c = filled([90, 33], 2, 64)
    s = step(rng, c, 6, 4, HF)
    agree(c, s, look(ctx, c, s, scale=scale), scale=scale)


def test_attend_replays_in_a_graph(ctx):
    from xwen_amd import cache8, tree
    rng = np.random.default_rng(17)
    c = filled([4000, 900], 2, 128)
    s = step(rng, c, 5, 8, BF)
    want = look(ctx, c, s)
    out = tree.Attended(*(torch.zeros_like(t) for t in (want.out, want.lse, want.seq_status)))
    parent = s["parent"].cuda()

    def call():
        cache8.tree_attend8(ctx, s["q"], c["k"], c["v"], c["k_exp"], c["v_exp"], c["len"], s["fk"], s["fv"], parent, out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    for _ in range(3):
        out.out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.out, want.out) and torch.equal(out.lse, want.lse)
        assert torch.equal(look(ctx, c, s).out, want.out)


def test_refusals(ctx):
    from xwen_amd import _lib, cache8
    rng = np.random.default_rng(18)
    c = filled([40], 2, 64)
    s = step(rng, c, 3, 4, BF)
    p = s["parent"].cuda()
    args = [c["k"], c["v"], c["k_exp"], c["v_exp"], c["len"]]
    for bad in ([c["k"].view(torch.uint8), *args[1:]], [*args[:2], c["k_exp"][:, :, :1], c["v_exp"][:, :, :1], c["len"]],
                [*args[:2], c["k_exp"].int(), c["v_exp"], c["len"]], [*args[:4], c["len"].long()]):
        with pytest.raises(ValueError):
            cache8.tree_attend8(ctx, s["q"], *bad, s["fk"], s["fv"], p)
        with pytest.raises(ValueError):
            cache8.cache_append8(ctx, *bad, s["fk"], s["fv"])
    with pytest.raises(ValueError):
        cache8.tree_attend8(ctx, s["q"].half(), *args, s["fk"], s["fv"], p)
    with pytest.raises(ValueError):
        cache8.cache_append8(ctx, *args, s["fk"].float(), s["fv"].float())
    with pytest.raises(ValueError):
        cache8.cache_append8(ctx, *args, s["fk"][0], s["fv"][0], start=torch.zeros(2, dtype=torch.int32, device="cuda"), n_path=c["len"])
    with pytest.raises(_lib.XsError):
        cache8.tree_attend8(ctx, s["q"][:, :, :3].contiguous(), *args, s["fk"], s["fv"], p)
