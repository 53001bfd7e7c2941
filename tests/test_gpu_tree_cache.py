"""xs_cache_commit and xs_cache_evict on the device against their definitions
(tests/treeref.py), and a whole speculative step: attend, verify, commit, evict."""
import math

import numpy as np
import pytest
import torch

from tests import treeref
from tests.test_gpu_tree_attend import BF, HF, blank, case, context, random_tree, run
from xwen_amd import _lib

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    return context()


def i32(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


def chain(rng, parent, n):
    """A path down the tree, as long as it goes."""
    path = [0]
    while True:
        kids = [j for j in range(path[-1] + 1, n) if parent[j] == path[-1]]
        if not kids:
            return path
        path.append(int(rng.choice(kids)))


def commit_case(rng, lens, nodes, hq, h, d, dtype, **kw):
    """A case with its attention run, and a path for each sequence (cut to various lengths)."""
    parent = [random_tree(rng, nodes) for _ in lens]
    c = case(rng, lens, nodes, hq, h, d, dtype, parent=parent, cap=max(lens) + nodes, **kw)
    path = [chain(rng, p, nodes) for p in parent]
    c["m"] = [len(p) if b % 3 else max(0, len(p) - b) for b, p in enumerate(path)]
    c["path"] = [p + [-1] * (nodes - len(p)) for p in path]
    b, cap = len(lens), c["k"].shape[1]
    c["mass"] = torch.rand((b, h, cap)).cuda()
    c["pos"] = torch.randint(0, 10**6, (b, h, cap), dtype=torch.int32).cuda()
    c["next_pos"] = [n + 1000 * b for b, n in enumerate(lens)]
    return c


def commit(ctx, c, lse, in_place=False, weights=True, positions=True, scale=None, max_len=0):
    from xwen_amd import tree
    c["new_mass"] = c["mass"] if in_place else torch.full_like(c["mass"], -5.0)
    kw = {}
    if weights:
        kw.update(q=c["q"], lse=lse, mass=c["mass"], new_mass=c["new_mass"], scale=scale)
    if positions:
        kw.update(pos=c["pos"], next_pos=i32(c["next_pos"]))
    return tree.cache_commit(ctx, c["k"], c["v"], i32(c["lens"]), c["fk"], c["fv"], i32(c["path"]), i32(c["m"]),
                             max_len=max_len, **kw)


def check_commit(ctx, c, scale=None, **kw):
    lse = run(ctx, c, scale=scale, out=blank(c)).lse
    before = {t: c[t].clone() for t in ("k", "v", "mass", "pos")}
    got = commit(ctx, c, lse, scale=scale, **kw)
    f = float(np.float32(1.0 / math.sqrt(c["q"].shape[-1]) if scale is None else scale))
    want = treeref.commit_mass(c["q"], lse, before["k"], c["lens"], c["fk"], c["path"], c["m"], f, before["mass"])
    assert got.seq_status.tolist() == [0] * len(c["lens"])
    assert got.new_len.tolist() == [n + m for n, m in zip(c["lens"], c["m"])]
    positions = kw.get("positions", True)
    if positions:
        assert got.new_next_pos.tolist() == [n + m for n, m in zip(c["next_pos"], c["m"])]
    for b, (n, m) in enumerate(zip(c["lens"], c["m"])):
        nodes = c["path"][b][:m]
        for t, f in (("k", "fk"), ("v", "fv")):
            assert torch.equal(c[t][b, n:n + m], c[f][b, nodes])
            assert torch.equal(c[t][b, :n], before[t][b, :n]) and torch.equal(c[t][b, n + m:], before[t][b, n + m:])
        if positions:
            assert c["pos"][b, :, n:n + m].tolist() == [list(range(c["next_pos"][b], c["next_pos"][b] + m))] * c["pos"].shape[1]
            before["pos"][b, :, n:n + m] = c["pos"][b, :, n:n + m]
        if kw.get("weights", True):
            w, tol = want[b]
            off = (c["new_mass"][b, :, :n + m].double().cpu() - w).abs()
            assert bool((off <= tol).all()), float((off / tol).max())
            rest = before["mass"] if kw.get("in_place") else torch.full_like(c["mass"], -5.0)
            assert torch.equal(c["new_mass"][b, :, n + m:], rest[b, :, n + m:])
    assert torch.equal(c["pos"], before["pos"])


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d", [8, 72, 128, 256])
def test_commit_head_sizes(ctx, d, dtype):
    rng = np.random.default_rng(d)
    check_commit(ctx, commit_case(rng, [0, 1, 63, 64, 65, 400], 9, 8, 4, d, dtype))


@pytest.mark.parametrize("hq,h", [(1, 1), (3, 3), (7, 1), (10, 2), (24, 8), (32, 1)])
@pytest.mark.parametrize("layout", ["slot", "head"])
def test_commit_head_layouts(ctx, hq, h, layout):
    rng = np.random.default_rng(hq)
    check_commit(ctx, commit_case(rng, [130, 17, 0], 12, hq, h, 64, BF, layout=layout), in_place=True)


@pytest.mark.parametrize("nodes", [1, 2, 16, 33, 64])
def test_commit_path_lengths(ctx, nodes):
    """Chains: paths as long as the tree."""
    rng = np.random.default_rng(nodes)
    c = commit_case(rng, [100, 257, 3, 31], nodes, 8, 2, 64, BF)
    c["parent"] = torch.tensor([list(range(-1, nodes - 1))] * 4, dtype=torch.int32)
    c["path"], c["m"] = [list(range(nodes))] * 4, [nodes, max(0, nodes - 1), nodes, 0]
    check_commit(ctx, c)


def test_commit_many_rows_in_place(ctx):
    """More rows than a wave holds: further passes add to what the first wrote, here into mass itself."""
    rng = np.random.default_rng(9)
    c = commit_case(rng, [300, 1000], 64, 16, 2, 128, BF)
    c["parent"] = torch.tensor([list(range(-1, 63))] * 2, dtype=torch.int32)
    c["path"], c["m"] = [list(range(64))] * 2, [64, 41]
    check_commit(ctx, c, in_place=True)


def test_commit_a_node_twice(ctx):
    """A path may name a node again (nothing forbids it): it is appended and counted again."""
    rng = np.random.default_rng(10)
    c = commit_case(rng, [70, 5], 6, 4, 2, 64, BF)
    c["path"], c["m"] = [[0, 0, 2, 0, -1, -1], [3, 3, 3, 3, 3, 3]], [4, 6]
    check_commit(ctx, c)


@pytest.mark.parametrize("nodes,hq,h,d,dtype", [(1, 8, 2, 128, BF), (30, 16, 2, 256, HF), (64, 32, 8, 64, BF)])
def test_commit_long(ctx, nodes, hq, h, d, dtype):
    rng = np.random.default_rng(nodes)
    check_commit(ctx, commit_case(rng, [8000, 2999], nodes, hq, h, d, dtype), max_len=8000)


def test_commit_without_weights_or_positions(ctx):
    rng = np.random.default_rng(1)
    check_commit(ctx, commit_case(rng, [100, 5], 7, 4, 2, 64, BF), weights=False)
    check_commit(ctx, commit_case(rng, [100, 5], 7, 4, 2, 64, BF), positions=False)
    check_commit(ctx, commit_case(rng, [100, 5], 7, 4, 2, 64, BF), weights=False, positions=False)


def test_commit_ignores_empty_rows_and_unused_slots(ctx):
    """An empty row's lse is -inf: it adds nothing.  What lies past the length counts for nothing."""
    rng = np.random.default_rng(2)
    c = commit_case(rng, [50, 9], 5, 4, 2, 64, BF)
    c["path"], c["m"] = [[0, 3, 4, -1, -1], [1, 2, -1, -1, -1]], [3, 2]
    c["parent"] = torch.tensor([[-1, 0, 0, 9, 0], [-1, -1, 1, 0, 0]], dtype=torch.int32)
    for b, n in enumerate(c["lens"]):
        c["k"][b, n:], c["v"][b, n:] = math.nan, math.nan
        c["fk"][b, 1 + 2 * (b == 1)] = math.nan
    lse = run(ctx, c, out=blank(c)).lse
    assert bool((lse[0, 3] == -math.inf).all())
    before = c["mass"].clone()
    kb = c["k"].clone()
    commit(ctx, c, lse)
    for b, (w, tol) in enumerate(treeref.commit_mass(c["q"], lse, kb, c["lens"], c["fk"], c["path"], c["m"], 0.125, before)):
        n = w.shape[1]
        assert bool(((c["new_mass"][b, :, :n].double().cpu() - w).abs() <= tol).all())


def test_commit_fails_alone(ctx):
    """Bad lengths, paths and a full cache: nothing of the sequence is written, the others are."""
    rng = np.random.default_rng(3)
    c = commit_case(rng, [40] * 8, 6, 4, 2, 64, BF)
    lse = run(ctx, c, out=blank(c)).lse
    good = [0, 1, 2, -1, -1, -1]
    c["path"], c["m"] = [list(good) for _ in range(8)], [3] * 8
    c["lens"][1], c["lens"][2] = -1, 47
    c["m"][3], c["m"][4] = -1, 7
    c["path"][5][1], c["path"][6][2] = 6, -1
    c["lens"][7] = 44
    before = {t: c[t].clone() for t in ("k", "v", "pos")}
    got = commit(ctx, c, lse)
    P = _lib.ROW_BAD_PARAM
    assert got.seq_status.tolist() == [0, P, P, P, P, P, P, _lib.ROW_CACHE_FULL]
    assert got.new_len.tolist() == [43, -1, 47, 40, 40, 40, 40, 44]
    assert got.new_next_pos.tolist() == [c["next_pos"][0] + 3] + c["next_pos"][1:]
    for t in before:
        assert torch.equal(c[t][1:], before[t][1:])
    assert bool((c["new_mass"][1:] == -5.0).all())
    assert torch.equal(c["k"][0, 40:43], c["fk"][0, :3])
    # exactly full is fine
    c["lens"], c["m"], c["path"] = [43] * 8, [3] * 8, [good] * 8
    assert commit(ctx, c, lse).seq_status.tolist() == [0] * 8


def test_commit_offsets_past_32_bits(ctx):
    rng = np.random.default_rng(4)
    c = commit_case(rng, [700], 3, 4, 2, 64, BF)
    room = torch.zeros(710 << 22, dtype=BF, device="cuda")
    for t in ("k", "v"):
        far = room.as_strided((1, c["k"].shape[1], 2, 64), (8, 1 << 22, 64, 1), storage_offset=0 if t == "k" else 4096)
        far.copy_(c[t])
        c[t] = far
    check_commit(ctx, c)


def evict_case(rng, lens, h, d, cap, dtype=BF, layout="slot", ties=False):
    b = len(lens)
    shape = {"slot": (b, cap, h, d), "head": (b, h, cap, d)}[layout]
    back = {"slot": (0, 1, 2, 3), "head": (0, 2, 1, 3)}[layout]
    c = {t: torch.from_numpy(rng.standard_normal(shape, dtype=np.float32)).to(dtype).cuda().permute(back) for t in "kv"}
    mass = rng.random((b, h, cap), dtype=np.float32) ** 6 * 30
    if ties:
        mass = rng.integers(0, 4, (b, h, cap)).astype(np.float32)
    pos = np.stack([[rng.permutation(cap) for _ in range(h)] for _ in range(b)]).astype(np.int32)
    for x, n in enumerate(lens):
        for y in range(h):
            pos[x, y, :n] = rng.permutation(n)
    c.update(mass=mass, pos=pos, lens=lens, next_pos=list(lens))
    return c


def check_evict(ctx, c, keep, sinks=0, recent=0, in_place=False, max_len=0):
    from xwen_amd import tree
    mass, pos = torch.from_numpy(c["mass"]).cuda(), torch.from_numpy(c["pos"]).cuda()
    nm, np_ = (mass, pos) if in_place else (torch.full_like(mass, -5.0), torch.full_like(pos, -5))
    before = {t: c[t].clone() for t in "kv"}
    rest = {"mass": nm.clone(), "pos": np_.clone()}
    got = tree.cache_evict(ctx, c["k"], c["v"], i32(c["lens"]), mass, pos, i32(c["next_pos"]), keep, sinks=sinks,
                           recent=recent, new_mass=None if in_place else nm, new_pos=None if in_place else np_, max_len=max_len)
    assert got.seq_status.tolist() == [0] * len(c["lens"])
    assert got.new_len.tolist() == [min(n, keep) for n in c["lens"]]
    for b, n in enumerate(c["lens"]):
        left = min(n, keep)
        for h in range(mass.shape[1]):
            source = list(range(n)) if n <= keep else treeref.evict_sources(
                c["mass"][b, h], c["pos"][b, h], n, c["next_pos"][b], keep, sinks, recent)
            at = torch.tensor(source, dtype=torch.long).cuda()
            for t in "kv":
                assert torch.equal(c[t][b, :left, h], before[t][b, at, h]), (b, h)
            m = nm[b, h, :left].cpu().numpy()
            np.testing.assert_array_equal(m, c["mass"][b, h, source])
            np.testing.assert_array_equal(np_[b, h, :left].cpu().numpy(), c["pos"][b, h, source])
        for t in "kv":
            assert torch.equal(c[t][b, left:], before[t][b, left:])
        assert torch.equal(nm[b, :, left:].nan_to_num(9), rest["mass"][b, :, left:].nan_to_num(9))
        assert torch.equal(np_[b, :, left:], rest["pos"][b, :, left:])


@pytest.mark.parametrize("keep", [1, 2, 31, 64, 100, 255, 256, 299, 300, 4000])
def test_evict_budgets(ctx, keep):
    rng = np.random.default_rng(keep)
    check_evict(ctx, evict_case(rng, [300, 0, 1, 64, 257, keep, keep + 1, keep // 2], 3, 64, 4096), keep, in_place=keep % 2 == 0)


@pytest.mark.parametrize("d,dtype,layout", [(8, BF, "slot"), (72, HF, "head"), (128, BF, "head"), (256, HF, "slot")])
def test_evict_layouts(ctx, d, dtype, layout):
    rng = np.random.default_rng(d)
    check_evict(ctx, evict_case(rng, [700, 513, 90], 4, d, 704, dtype, layout), 400, sinks=4, recent=32)


@pytest.mark.parametrize("sinks,recent", [(0, 0), (4, 0), (0, 50), (10, 90), (0, 100), (100, 0)])
def test_evict_protects_the_first_and_the_last(ctx, sinks, recent):
    rng = np.random.default_rng(sinks)
    c = evict_case(rng, [101, 640, 150], 2, 64, 640)
    check_evict(ctx, c, 100, sinks=sinks, recent=recent, in_place=True)


def test_evict_ties(ctx):
    """Few different weights, all alike, all zero (of either sign): the lower position stays."""
    rng = np.random.default_rng(1)
    check_evict(ctx, evict_case(rng, [500, 399, 1000], 2, 64, 1000, ties=True), 200, recent=20)
    c = evict_case(rng, [500, 399, 1000], 2, 64, 1000)
    c["mass"][:] = 0.0
    c["mass"][:, :, ::3] = -0.0
    check_evict(ctx, c, 200, recent=20, in_place=True)
    c["pos"][0, 0, :500] = 7  # positions alike too: the lower slot stays
    c["pos"][1, 1, :399] = 10**9
    c["next_pos"][1] = 0
    check_evict(ctx, c, 200, sinks=8, in_place=True)


def test_evict_odd_weights(ctx):
    """NaN last, infinities, negative and subnormal weights; negative positions."""
    rng = np.random.default_rng(2)
    c = evict_case(rng, [900, 300], 3, 64, 900)
    m = c["mass"]
    m[:, 0, ::7] = math.nan
    m[:, 1, ::5] = math.inf
    m[:, 1, 1::5] = -math.inf
    m[:, 2] = rng.standard_normal(m[:, 2].shape).astype(np.float32) * np.float32(1e-44)
    m.view(np.uint32)[:, 0, 1::7] = 0xFFC00000  # a NaN with its sign set
    c["pos"][1] -= 150
    check_evict(ctx, c, 150, sinks=2, recent=5)
    c["mass"][:] = math.nan
    check_evict(ctx, c, 150, sinks=2, recent=5, in_place=True)


@pytest.mark.parametrize("keep", [100, 4097, 8100])
def test_evict_long(ctx, keep):
    rng = np.random.default_rng(keep)
    check_evict(ctx, evict_case(rng, [8192, 5000], 2, 64, 8192), keep, sinks=4, recent=64, max_len=8192)


def test_evict_fails_alone(ctx):
    from xwen_amd import tree
    rng = np.random.default_rng(3)
    c = evict_case(rng, [60, 60, 60], 2, 64, 64)
    mass, pos = torch.from_numpy(c["mass"]).cuda(), torch.from_numpy(c["pos"]).cuda()
    before = [t.clone() for t in (c["k"], c["v"], mass, pos)]
    got = tree.cache_evict(ctx, c["k"], c["v"], i32([65, -3, 60]), mass, pos, i32([60] * 3), 40)
    assert got.seq_status.tolist() == [_lib.ROW_BAD_PARAM, _lib.ROW_BAD_PARAM, 0] and got.new_len.tolist() == [65, -3, 40]
    for x, y in zip(before, (c["k"], c["v"], mass, pos)):
        assert torch.equal(x[:2], y[:2])


def test_commit_and_evict_under_capture(ctx):
    """A captured commit and evict, replayed on a cache put back each time, with eager work between."""
    from xwen_amd import tree
    rng = np.random.default_rng(5)
    c = commit_case(rng, [3000, 500], 8, 8, 2, 128, BF)
    lse = run(ctx, c, out=blank(c)).lse
    start = {t: c[t].clone() for t in ("k", "v", "pos", "mass")}
    held = {t: i32(c[t]) for t in ("lens", "path", "m", "next_pos")}
    done = tree.Committed(i32([0, 0]), i32([0, 0]), i32([0, 0]))
    cut = tree.Evicted(i32([0, 0]), i32([0, 0]))

    def step():
        tree.cache_commit(ctx, c["k"], c["v"], held["lens"], c["fk"], c["fv"], held["path"], held["m"], pos=c["pos"],
                          next_pos=held["next_pos"], q=c["q"], lse=lse, mass=c["mass"], out=done)
        tree.cache_evict(ctx, c["k"], c["v"], done.new_len, c["mass"], c["pos"], done.new_next_pos, 400, sinks=4,
                         recent=16, out=cut)

    step()
    want = [c[t].clone() for t in start] + [cut.new_len.clone()]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for _ in range(3):
        for t in start:
            c[t].copy_(start[t])
        cut.new_len.zero_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for x, y in zip(want, [c[t] for t in start] + [cut.new_len]):
            assert torch.equal(x, y)
        run(ctx, c, out=blank(c))


def test_a_speculative_step_over_a_bounded_cache(ctx):
    """Steps as a user makes them: attend, verify, commit, evict, over TreeCache, against the
    same in plain code.  The plain cache follows the device's committed paths."""
    from xwen_amd import sampler as xsm
    from xwen_amd import tree
    rng = np.random.default_rng(6)
    torch.manual_seed(6)
    B, N, HQ, H, D, V, keep = 3, 12, 8, 2, 64, 2000, 20
    cache = tree.TreeCache(ctx, B, H, D, keep, dtype=BF, sinks=2, recent=4)
    sampler = xsm.Context(max_rows=B * N, vocab=V)
    sampler.bind_current_stream()
    head = torch.randn((HQ * D, V), device="cuda") * 0.4
    plain = [[[] for _ in range(H)] for _ in range(B)]  # per head: [k, v, mass, pos] of each slot
    seen = [0] * B
    for step in range(12):
        parent = [random_tree(rng, N) for _ in range(B)]
        q, fk, fv = (torch.randn((B, N, h, D), device="cuda").to(BF) for h in (HQ, H, H))
        got = cache.attend(q, fk, fv, i32(parent))
        logits = got.out.float().reshape(B * N, -1) @ head
        best = logits.view(B, N, V).topk(2, -1).indices.cpu().numpy()
        tokens = np.zeros((B, N), np.int32)
        for b in range(B):
            for j in range(1, N):
                tokens[b, j] = best[b, parent[b][j], rng.integers(0, 2)]
        params = xsm.params_tensor(0.5, 20, 0.9, B * N, "cuda")
        u = torch.from_numpy((rng.integers(0, 1 << 23, B * N) * 2.0**-23).astype(np.float32)).cuda()
        v = xsm.verify_tree_batch(sampler, logits, B, N, params, u, i32(tokens), i32(parent))
        # the attention and the weights against the definition, over the cache as it stands
        for b in range(B):
            lens = len(plain[b][0])
            k = torch.zeros((1, max(lens, 1), H, D), dtype=BF)
            vv = torch.zeros_like(k)
            for h in range(H):
                for s, row in enumerate(plain[b][h]):
                    k[0, s, h], vv[0, s, h] = row[0], row[1]
            out, lse, tol, ltol = treeref.attend(q[b:b + 1], k, vv, [lens], fk[b:b + 1], fv[b:b + 1], [torch.tensor(parent[b])],
                                                 [N], float(np.float32(1 / math.sqrt(D))))
            assert bool(((got.out[b].double().cpu() - out[0]).abs() <= tol[0]).all())
            assert bool(((got.lse[b].double().cpu() - lse[0]).abs() <= ltol[0]).all())
            acc, path, com, st = treeref.walk(v.row_token.view(B, N)[b].tolist(), v.row_status.view(B, N)[b].tolist(),
                                              tokens[b], parent[b], N, 1 << 30, (), [0] * N)
            m = int(v.n_committed[b])
            assert v.path[b, :m].tolist() == path and v.committed[b, :m].tolist() == com and int(v.accepted[b]) == acc
            mass = torch.tensor([[row[2] for row in plain[b][h]] + [0.0] for h in range(H)], dtype=torch.float64)
            (w, _), = treeref.commit_mass(q[b:b + 1], got.lse[b:b + 1], k, [lens], fk[b:b + 1], [path], [m],
                                          float(np.float32(1 / math.sqrt(D))), mass[None])
            for h in range(H):
                rows = plain[b][h]
                for s in range(lens):
                    rows[s][2] = float(w[h, s])
                for r, i in enumerate(path):
                    rows.append([fk[b, i, h].cpu(), fv[b, i, h].cpu(), float(w[h, lens + r]), seen[b] + r])
            seen[b] += m
        cache.commit(q, got.lse, fk, fv, v.path, v.n_committed)
        tree.check(cache.commit_status)
        for b in range(B):
            n = len(plain[b][0])
            assert cache.length.tolist()[b] == n and cache.next_pos.tolist()[b] == seen[b]
            for h in range(H):
                dev = cache.mass[b, h, :n].cpu().numpy()
                np.testing.assert_allclose(dev, [r[2] for r in plain[b][h]], rtol=2e-5, atol=1e-6)
                for s in range(n):  # go on from the device's sums, so that near ties are cut alike
                    plain[b][h][s][2] = float(dev[s])
        cache.evict()
        tree.check(cache.evict_status)
        for b in range(B):
            n = len(plain[b][0])
            for h in range(H):
                rows = plain[b][h]
                if n > keep:
                    source = treeref.evict_sources(np.array([r[2] for r in rows], np.float32), [r[3] for r in rows], n, seen[b],
                                                   keep, 2, 4)
                    plain[b][h] = [rows[s] for s in source]
                    assert {0, 1, seen[b] - 1, seen[b] - 4} <= {r[3] for r in plain[b][h]}
                left = min(n, keep)
                assert cache.pos[b, h, :left].tolist() == [r[3] for r in plain[b][h]]
                assert torch.equal(cache.k[b, :left, h].cpu(), torch.stack([r[0] for r in plain[b][h]]))
                assert torch.equal(cache.v[b, :left, h].cpu(), torch.stack([r[1] for r in plain[b][h]]))
        assert cache.length.tolist() == [len(plain[b][0]) for b in range(B)]
    assert max(seen) > keep


@pytest.mark.parametrize("cap", [301, 302, 303, 304])
def test_evict_slots_off_the_16_byte_grid(ctx, cap):
    """Per-slot arrays whose rows start anywhere."""
    rng = np.random.default_rng(cap)
    c = evict_case(rng, [cap, cap - 7, 150], 3, 64, cap)
    check_evict(ctx, c, 140, sinks=3, recent=11, in_place=cap % 2 == 0)
    c = evict_case(rng, [cap, cap - 7, 150], 3, 64, cap, ties=True)
    check_evict(ctx, c, cap - 9, sinks=3, recent=11)


@pytest.mark.parametrize("n", [4096, 4097, 8193, 32_768, 32_769, 70_001])
def test_evict_lengths_at_the_kernels_bounds(n):
    """Where the slots of a head stop fitting the registers of its workgroup."""
    big = context(max_seqs=2, kv_heads=2, q_heads=2, head_dim=8, capacity=70_016, max_nodes=1)
    rng = np.random.default_rng(n)
    check_evict(big, evict_case(rng, [n, n // 2], 2, 8, (n + 7) // 8 * 8), n // 3, sinks=4, recent=64)
    c = evict_case(rng, [n, n // 2], 2, 8, (n + 7) // 8 * 8, ties=True)
    c["pos"][0, 0, :n] = 5  # equal in everything but the slot
    check_evict(big, c, n - 100, in_place=True)
    big.close()
