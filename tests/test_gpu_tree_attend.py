"""xs_tree_attend on the device against the definition in 64 bits (tests/treeref.py)."""
import math

import numpy as np
import pytest
import torch

from tests import treeref
from xwen_amd import _lib

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def context(**kw):
    from xwen_amd import tree
    d = dict(max_seqs=40, max_nodes=64, q_heads=32, kv_heads=16, head_dim=256, capacity=8192)
    d.update(kw)
    return tree.CacheContext(**d)


@pytest.fixture(scope="module")
def ctx():
    return context()


def random_tree(rng, n, roots=False):
    p = [-1]
    for i in range(1, n):
        p.append(-1 if roots and rng.random() < 0.2 else int(rng.integers(max(0, i - 6), i)))
    return p


def case(rng, lens, nodes, hq, h, d, dtype, used=None, layout="slot", cap=None, parent=None, spread=1.0):
    g = torch.Generator().manual_seed(int(rng.integers(1 << 30)))
    b = len(lens)
    cap = cap or max(lens) + 5
    shape = {"slot": (b, cap, h, d), "head": (b, h, cap, d), "seq_last": (cap, b, h, d)}[layout]
    back = {"slot": (0, 1, 2, 3), "head": (0, 2, 1, 3), "seq_last": (1, 0, 2, 3)}[layout]

    def fill(*s):
        return (torch.randn(s, generator=g) * spread).to(dtype).cuda()
    k, v = fill(*shape).permute(back), torch.randn(shape, generator=g).to(dtype).cuda().permute(back)
    q = fill(b, nodes, hq, d)
    fk, fv = fill(b, nodes, h, d), torch.randn((b, nodes, h, d), generator=g).to(dtype).cuda()
    if parent is None:
        parent = [random_tree(rng, nodes, roots=True) for _ in range(b)]
    used = used or [nodes] * b
    return dict(q=q, k=k, v=v, lens=lens, fk=fk, fv=fv, parent=torch.tensor(parent, dtype=torch.int32), used=used)


def run(ctx, c, scale=None, max_len=0, ragged=True, out=None):
    from xwen_amd import tree
    length = torch.tensor(c["lens"], dtype=torch.int32).cuda()
    n = torch.tensor(c["used"], dtype=torch.int32).cuda() if ragged else None
    return tree.tree_attend(ctx, c["q"], c["k"], c["v"], length, c["fk"], c["fv"], c["parent"].cuda(), n_nodes=n,
                            scale=scale, max_len=max_len, out=out)


def blank(c, fill=7.0):
    from xwen_amd import tree
    b, n, hq, d = c["q"].shape
    return tree.Attended(out=torch.full((b, n, hq, d), fill, dtype=c["q"].dtype, device="cuda"),
                         lse=torch.full((b, n, hq), fill, device="cuda"),
                         seq_status=torch.full((b,), -1, dtype=torch.int32, device="cuda"))


def agree(c, got, scale=None, fill=7.0):
    scale = float(np.float32(1.0 / math.sqrt(c["q"].shape[-1]) if scale is None else scale))
    out, lse, tol, ltol = treeref.attend(c["q"], c["k"], c["v"], c["lens"], c["fk"], c["fv"], c["parent"], c["used"], scale)
    assert got.seq_status.tolist() == [0] * len(c["lens"])
    o, s = got.out.double().cpu(), got.lse.double().cpu()
    for b, n in enumerate(c["used"]):
        assert bool((o[b, n:] == fill).all()) and bool((s[b, n:] == fill).all())
        empty = lse[b, :n] == -math.inf
        assert bool((s[b, :n][empty] == -math.inf).all()) and bool((o[b, :n][empty] == 0.0).all())
        x, y = o[b, :n][~empty], out[b, :n][~empty]
        assert bool((torch.isnan(x) == torch.isnan(y)).all())
        fine = torch.isfinite(y)
        assert bool((x[~fine & ~torch.isnan(y)] == y[~fine & ~torch.isnan(y)]).all())
        off = (x - y).abs()[fine]
        assert bool((off <= tol[b, :n][~empty][fine]).all()), float((off / tol[b, :n][~empty][fine]).max())
        x, y = s[b, :n][~empty], lse[b, :n][~empty]
        assert bool((torch.isnan(x) == torch.isnan(y)).all())
        fine = torch.isfinite(y)
        assert bool(((x - y).abs()[fine] <= ltol[b, :n][~empty][fine]).all())


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d", [8, 64, 72, 80, 128, 136, 256])
def test_head_sizes(ctx, d, dtype):
    rng = np.random.default_rng(d)
    c = case(rng, [0, 1, 33, 130, 517], 9, 8, 4, d, dtype, used=[9, 1, 8, 0, 5])
    agree(c, run(ctx, c, out=blank(c)))


@pytest.mark.parametrize("hq,h", [(1, 1), (3, 3), (4, 1), (7, 1), (10, 2), (16, 1), (24, 8), (32, 1), (32, 16)])
def test_head_layouts(ctx, hq, h):
    rng = np.random.default_rng(hq * 64 + h)
    c = case(rng, [70, 5], 4, hq, h, 64, BF)
    agree(c, run(ctx, c, out=blank(c)))


@pytest.mark.parametrize("nodes", [1, 2, 3, 15, 16, 17, 31, 33, 48, 63, 64])
@pytest.mark.parametrize("g", [1, 4, 5])
def test_tree_sizes(ctx, nodes, g):
    rng = np.random.default_rng(nodes * 8 + g)
    c = case(rng, [100, 0], nodes, 2 * g, 2, 64, BF, used=[nodes, max(1, nodes - 2)])
    agree(c, run(ctx, c, out=blank(c)))


@pytest.mark.parametrize("nodes", [1, 6])
def test_lengths(ctx, nodes):
    rng = np.random.default_rng(nodes)
    lens = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 512, 513, 1023, 1025, 2047, 2500]
    c = case(rng, lens, nodes, 4, 2, 128, BF)
    agree(c, run(ctx, c, out=blank(c)))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("nodes,hq,h,d", [(1, 8, 2, 128), (40, 8, 2, 128), (64, 16, 2, 64), (20, 16, 2, 256)])
def test_long(ctx, nodes, hq, h, d, dtype):
    """Long enough for several workgroups a row, with large scores."""
    rng = np.random.default_rng(nodes)
    c = case(rng, [8000, 3001], nodes, hq, h, d, dtype, spread=1.7)
    agree(c, run(ctx, c, out=blank(c)))
    agree(c, run(ctx, c, max_len=8000, out=blank(c)))


@pytest.mark.parametrize("layout", ["head", "seq_last"])
def test_layouts(ctx, layout):
    rng = np.random.default_rng(3)
    c = case(rng, [65, 200, 31], 5, 6, 3, 64, HF, layout=layout)
    agree(c, run(ctx, c, out=blank(c)))


def test_padded_and_repeated_rows(ctx):
    """Strides with room between the rows, one key row for every node, one query for every head."""
    rng = np.random.default_rng(4)
    c = case(rng, [90, 41], 6, 4, 2, 64, BF)
    wide = torch.randn((2, 100, 2, 96), device="cuda").to(BF)
    c["k"], c["v"] = wide[:, :95, :, :64], wide[:, :95, :, 32:]
    c["fk"] = c["fk"][:, :1].expand(2, 6, 2, 64)
    c["fv"] = c["fv"][:, :1].expand(2, 6, 2, 64)
    c["q"] = c["q"][:, :, :1].expand(2, 6, 4, 64)
    agree(c, run(ctx, c, out=blank(c)))


def test_nothing_in_the_cache_and_no_node(ctx):
    rng = np.random.default_rng(5)
    c = case(rng, [0, 0, 12], 3, 2, 2, 64, BF, used=[1, 0, 0], cap=20)
    agree(c, run(ctx, c, out=blank(c)))
    c["used"] = [3, 3, 3]
    agree(c, run(ctx, c, ragged=False, out=blank(c)))


def test_broken_parents_see_nothing(ctx):
    """A parent that is the node itself, one above it, one past the tree and one below -1;
    what follows them sees nothing either."""
    rng = np.random.default_rng(6)
    parent = [[-1, 1, 0, 1, 2, 9, -2, 6, 5, 4], [5, 0, -1, 2, 3, 4, 4, 10**9, -10**9, 8]]
    c = case(rng, [40, 0], 10, 4, 2, 64, BF, parent=parent)
    agree(c, run(ctx, c, out=blank(c)))
    c["used"] = [3, 4]
    agree(c, run(ctx, c, out=blank(c)))


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("nodes,hq", [(7, 4), (60, 8)])
def test_what_is_not_seen_does_not_count(ctx, bad, nodes, hq):
    """NaN and infinities past the length, past the tree and in other branches."""
    rng = np.random.default_rng(7)
    c = case(rng, [33, 0, 300], nodes, hq, 2, 64, BF, used=[nodes, nodes - 2, nodes - 1], cap=320)
    for b, n in enumerate(c["lens"]):
        for t in ("k", "v"):
            c[t][b, n:] = bad
        for t in ("fk", "fv", "q"):
            c[t][b, c["used"][b]:] = bad
    c["fk"][0, 3, 1, 5] = bad
    c["fv"][0, 4, 0, 9] = bad
    c["fv"][2, 5, 1, 63] = bad
    c["fv"][2, 2, 1, 63] = -bad
    agree(c, run(ctx, c, out=blank(c)))


@pytest.mark.parametrize("nodes", [2, 30])
def test_extreme_scores(ctx, nodes):
    """Rows whose every score is -inf, scores of the type's ends, one +inf, one NaN."""
    rng = np.random.default_rng(8)
    c = case(rng, [50, 50, 50, 50, 900], nodes, 4, 4, 64, BF)
    for t in ("q", "k", "fk"):
        c[t][:, :, :, 0] = 0.0
    c["q"][:, :, :, 0] = 1.0
    c["k"][0, :, :, 0] = -math.inf
    c["fk"][0, :, :, 0] = -math.inf
    c["k"][1, :, :, 0] = torch.finfo(BF).min
    c["fk"][1, :, :, 0] = torch.finfo(BF).min
    c["k"][2, 7, 1, 0] = math.inf
    c["k"][3, 49, 2, 0] = math.nan
    c["k"][4, :899, :, 0] = -math.inf
    agree(c, run(ctx, c, scale=0.125, out=blank(c)), scale=0.125)


@pytest.mark.parametrize("nodes", [5, 48])
@pytest.mark.parametrize("scale", [0.0, -0.3, 4.0])
def test_scales(ctx, scale, nodes):
    rng = np.random.default_rng(9)
    c = case(rng, [320, 3], nodes, 4, 2, 64, HF)
    agree(c, run(ctx, c, scale=scale, out=blank(c)), scale=scale)


@pytest.mark.parametrize("d", [64, 72, 128, 136])
@pytest.mark.parametrize("nodes,hq,h", [(33, 2, 1), (64, 4, 2), (64, 4, 1), (64, 5, 1), (20, 16, 1), (64, 16, 1)])
def test_many_rows(ctx, nodes, hq, h, d):
    """More rows than a wave holds: tiles of several waves, some of them empty, at lengths
    about the blocks (32) and stages (64) in which the keys are read."""
    rng = np.random.default_rng(nodes + d)
    lens = [0, 31, 32, 63, 64, 65, 96, 127, 128, 129, 190, 257]
    c = case(rng, lens, nodes, hq, h, d, BF if d % 64 else HF, used=[max(0, nodes - (b % 4) * 7) for b in range(len(lens))])
    agree(c, run(ctx, c, out=blank(c)))


def test_extreme_scores_of_many_rows(ctx):
    """As test_extreme_scores, where four waves share the keys; the maximum grows late, in steps."""
    rng = np.random.default_rng(16)
    c = case(rng, [300, 300, 300, 300, 900], 40, 8, 2, 64, BF)
    for t in ("q", "k", "fk"):
        c[t][:, :, :, 0] = 0.0
    c["q"][:, :, :, 0] = 1.0
    c["k"][0, :, :, 0] = -math.inf
    c["fk"][0, :, :, 0] = -math.inf
    c["k"][1, :, :, 0] = torch.finfo(BF).min
    c["fk"][1, :, :, 0] = torch.finfo(BF).min
    c["k"][2, 7, 1, 0] = math.inf
    c["k"][3, 99, 0, 0] = math.nan
    c["k"][4, :899, :, 0] = (torch.arange(899, device="cuda") * 0.9)[:, None].to(BF)
    agree(c, run(ctx, c, scale=0.125, out=blank(c)), scale=0.125)


def test_offsets_past_32_bits(ctx):
    """A cache whose slots lie 2^22 elements apart: 700 of them span 2.9e9 elements."""
    rng = np.random.default_rng(10)
    c = case(rng, [700], 3, 4, 2, 64, BF, cap=704)
    room = torch.zeros(704 << 22, dtype=BF, device="cuda")
    for t in ("k", "v"):
        far = room.as_strided((1, 704, 2, 64), (8, 1 << 22, 64, 1), storage_offset=0 if t == "k" else 4096)
        far.copy_(c[t])
        c[t] = far
    agree(c, run(ctx, c, out=blank(c)))


def test_a_sequence_out_of_bounds_fails_alone(ctx):
    rng = np.random.default_rng(11)
    c = case(rng, [20, 20, 20, 20, 20], 4, 4, 2, 64, BF, cap=30)
    want = run(ctx, c, out=blank(c))
    c["lens"], c["used"] = [20, 31, -1, 20, 20], [4, 4, 4, 5, -1]
    got = run(ctx, c, out=blank(c))
    assert got.seq_status.tolist() == [0] + [_lib.ROW_BAD_PARAM] * 4
    assert torch.equal(got.out[0], want.out[0]) and torch.equal(got.lse[0], want.lse[0])
    assert bool((got.out[1:] == 7.0).all()) and bool((got.lse[1:] == 7.0).all())
    c["lens"], c["used"] = [20] * 5, [4] * 5
    assert run(ctx, c, max_len=19, out=blank(c)).seq_status.tolist() == [_lib.ROW_BAD_PARAM] * 5


def test_without_lse_and_without_sequences(ctx):
    rng = np.random.default_rng(12)
    c = case(rng, [77], 3, 4, 2, 64, BF)
    want = run(ctx, c, out=blank(c))
    got = blank(c)
    got.lse = None
    run(ctx, c, out=got)
    assert torch.equal(got.out, want.out)
    e = dict(c, q=c["q"][:0], k=c["k"][:0], v=c["v"][:0], fk=c["fk"][:0], fv=c["fv"][:0], parent=c["parent"][:0], lens=[], used=[])
    assert run(ctx, e).out.shape[0] == 0


def test_the_same_bits_every_time_and_in_any_batch(ctx):
    rng = np.random.default_rng(13)
    c = case(rng, [5000, 300, 7000], 12, 8, 2, 128, BF)
    first = run(ctx, c, out=blank(c))
    for _ in range(5):
        again = run(ctx, c, out=blank(c))
        assert torch.equal(first.out, again.out) and torch.equal(first.lse, again.lse)


def test_streams_and_graph_replays(ctx):
    """Another stream than the default; a captured call replayed with new inputs, with eager
    calls of the same context between the replays."""
    rng = np.random.default_rng(14)
    c = case(rng, [3000, 64], 10, 8, 2, 128, BF, cap=3100)
    want = run(ctx, c, out=blank(c))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(ctx, c, out=blank(c))
    side.synchronize()
    assert torch.equal(got.out, want.out)
    from xwen_amd import tree
    length = torch.tensor(c["lens"], dtype=torch.int32).cuda()
    parent, out = c["parent"].cuda(), blank(c)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        tree.tree_attend(ctx, c["q"], c["k"], c["v"], length, c["fk"], c["fv"], parent, out=out)
    for step in range(4):
        c["q"].copy_(torch.randn(c["q"].shape, device="cuda"))
        length.copy_(torch.tensor([3000 - 900 * step, 64 + step], dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        c["lens"] = length.tolist()
        eager = run(ctx, c, out=blank(c))
        assert torch.equal(out.out, eager.out) and torch.equal(out.lse, eager.lse)


def test_streams_in_turn_share_the_workspace(ctx):
    """One context's calls from two streams, one after the other without a wait of the caller's."""
    rng = np.random.default_rng(17)
    cs = [case(rng, [6000, 900], 8, 8, 2, 128, BF), case(rng, [7000, 1200], 8, 8, 2, 128, BF)]
    want = [run(ctx, c, out=blank(c)) for c in cs]
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(6):
        for j in range(2):
            with torch.cuda.stream(streams[j]):
                outs[j].append(run(ctx, cs[j], out=blank(cs[j])))
    torch.cuda.synchronize()
    for j in range(2):
        for got in outs[j]:
            assert torch.equal(got.out, want[j].out) and torch.equal(got.lse, want[j].lse)


@pytest.mark.parametrize("nodes", [1, 20])
def test_many_sequences(nodes):
    """2,000 sequences over one cache (their stride 0): every one the first one's result."""
    from xwen_amd import tree
    rng = np.random.default_rng(19)
    big = context(max_seqs=2000, max_nodes=nodes, q_heads=8, kv_heads=2, head_dim=64, capacity=128)
    c = case(rng, [100], nodes, 8, 2, 64, BF)
    want = run(big, c, out=blank(c))
    agree(c, want)
    n = 2000
    many = {t: c[t].expand(n, *c[t].shape[1:]) for t in ("q", "k", "v", "fk", "fv")}
    got = tree.tree_attend(big, many["q"], many["k"], many["v"], torch.full((n,), 100, dtype=torch.int32, device="cuda"),
                           many["fk"], many["fv"], c["parent"].cuda().expand(n, nodes).contiguous())
    assert bool((got.seq_status == 0).all())
    assert torch.equal(got.out, want.out.expand_as(got.out)) and torch.equal(got.lse, want.lse.expand_as(got.lse))
    big.close()


def test_strides_of_single_entries_do_not_matter(ctx):
    """One kv head, one node, one sequence, their strides any number."""
    rng = np.random.default_rng(18)
    c = case(rng, [50], 1, 4, 1, 64, BF)
    want = run(ctx, c, out=blank(c))
    for t in ("k", "v"):
        c[t] = c[t].as_strided(c[t].shape, (3, 64, 5, 1))
    for t in ("fk", "fv"):
        c[t] = c[t].as_strided(c[t].shape, (1, 7, 9, 1))
    c["q"] = c["q"].as_strided(c["q"].shape, (11, 13, 64, 1))
    got = run(ctx, c, out=blank(c))
    assert torch.equal(got.out, want.out) and torch.equal(got.lse, want.lse)


def test_two_contexts_at_once(ctx):
    rng = np.random.default_rng(15)
    other = context()
    cs = [case(rng, [6000], 8, 8, 2, 128, BF), case(rng, [7000], 8, 8, 2, 128, BF)]
    want = [run(ctx, c, out=blank(c)) for c in cs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = [[], []]
    for _ in range(5):
        for j, (x, s) in enumerate(zip((ctx, other), streams)):
            with torch.cuda.stream(s):
                outs[j].append(run(x, cs[j], out=blank(cs[j])))
    torch.cuda.synchronize()
    for j in range(2):
        for got in outs[j]:
            assert torch.equal(got.out, want[j].out) and torch.equal(got.lse, want[j].lse)
    other.close()
