"""xs_verify_tree on the device: for chains it is xs_verify, for trees the walk of
tests/treeref.py over the rows that it sampled, which are xs_sample's."""
import numpy as np
import pytest
import torch

from tests import treeref, workloads
from tests.test_gpu_tree_attend import random_tree
from xwen_amd import _lib

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.as_tensor(np.asarray(x, np.int32)).cuda()


def setup(rng, seqs, nodes, vocab, sharp=True):
    from xwen_amd import sampler as xsm
    ctx = xsm.Context(max_rows=max(1, seqs * nodes), vocab=vocab)
    ctx.bind_current_stream()
    ld = (vocab + 3) // 4 * 4
    x = rng.standard_normal((seqs * nodes, ld), dtype=np.float32) * 2
    if sharp:
        x[np.arange(seqs * nodes), rng.integers(0, vocab, seqs * nodes)] = 16.0
        x[np.arange(seqs * nodes), rng.integers(0, vocab, seqs * nodes)] = 16.0
    u = (rng.integers(0, 1 << 23, seqs * nodes) * 2.0**-23).astype(np.float32)
    params = xsm.params_tensor(0.8, 20, 0.95, seqs * nodes, "cuda")
    return xsm, ctx, torch.from_numpy(x).cuda(), params, torch.from_numpy(u).cuda()


@pytest.mark.parametrize("nodes", [1, 2, 16, 63, 64])
def test_a_chain_is_xs_verify(nodes):
    rng = np.random.default_rng(nodes)
    seqs, V = 6, 5003
    xsm, ctx, x, params, u = setup(rng, seqs, nodes, V)
    tokens = np.zeros((seqs, nodes), np.int32)
    drawn = xsm.sample_batch(ctx, x, params, u, enc=V).token.view(seqs, nodes).cpu().numpy()
    tokens[:, 1:] = drawn[:, :-1]
    for b in range(seqs):  # a wrong draft at places of their own
        if b and nodes > 1:
            tokens[b, min(nodes - 1, 1 + (b * 7) % nodes)] = (drawn[b, 0] + 1) % V
    parent = np.tile(np.arange(-1, nodes - 1, dtype=np.int32), (seqs, 1))
    budget = i32([nodes, 3, 0, 100, 2, -1])
    done = np.zeros((seqs, nodes), np.uint8)
    done[3, nodes // 2] = 1
    shifted = np.zeros((seqs, nodes), np.uint8)  # xs_verify marks the draft's position, xs_verify_tree its node
    shifted[:, :-1] = done[:, 1:]
    for eog in ((), (int(drawn[4, 0]), int(drawn[0, nodes - 1]))):
        for kw in ({}, {"budget": budget}, {"done": True}):
            extra = {k: v for k, v in kw.items() if k == "budget"}
            t = xsm.verify_tree_batch(ctx, x, seqs, nodes, params, u, i32(tokens), i32(parent), eog=eog, enc=V,
                                      done_after=torch.from_numpy(done).cuda() if "done" in kw else None, **extra)
            w = xsm.verify_batch(ctx, x, seqs, nodes, params, u, i32(tokens[:, 1:]), eog=eog, enc=V,
                                 done_after=torch.from_numpy(shifted).cuda() if "done" in kw else None, **extra)
            for f in ("row_token", "row_status", "accepted", "committed", "n_committed", "seq_status"):
                assert torch.equal(getattr(t, f), getattr(w, f)), (f, eog, kw)
            n = t.n_committed.tolist()
            for b in range(seqs):
                assert t.path[b].tolist() == list(range(n[b])) + [-1] * (nodes - n[b])


@pytest.mark.parametrize("seed", range(12))
def test_random_trees(seed):
    rng = np.random.default_rng(seed)
    seqs, nodes, V = int(rng.integers(1, 12)), int(rng.integers(1, 65)), int(rng.choice([700, 5003, 20_011]))
    xsm, ctx, x, params, u = setup(rng, seqs, nodes, V)
    drawn = xsm.sample_batch(ctx, x, params, u, enc=V).token.view(seqs, nodes).cpu().numpy()
    parent = np.array([random_tree(rng, nodes) for _ in range(seqs)], np.int32)
    tokens = rng.integers(0, V, (seqs, nodes)).astype(np.int32)
    for b in range(seqs):
        for j in range(1, nodes):
            if rng.random() < 0.6:  # (siblings may carry one token: the lowest is taken)
                tokens[b, j] = drawn[b, parent[b, j]]
            if rng.random() < 0.05:
                parent[b, j] = rng.choice([-1, -2, j, j + 1, nodes, 10**9])
    n = rng.integers(0, nodes + 1, seqs).astype(np.int32)
    budget = rng.integers(0, 8, seqs).astype(np.int32)
    eog = [int(t) for t in rng.choice(drawn.ravel(), 2)]
    done = (rng.random((seqs, nodes)) < 0.05).astype(np.uint8)
    got = xsm.verify_tree_batch(ctx, x, seqs, nodes, params, u, i32(tokens), i32(parent), n_nodes=i32(n), budget=i32(budget),
                                eog=eog, enc=V, done_after=torch.from_numpy(done).cuda())
    assert torch.equal(got.row_token.view(seqs, nodes).cpu(), torch.from_numpy(drawn))
    for b in range(seqs):
        acc, path, com, st = treeref.walk(drawn[b], np.zeros(nodes), tokens[b], parent[b], n[b], budget[b], eog, done[b])
        pad = [-1] * (nodes - len(path))
        assert got.path[b].tolist() == path + pad and got.committed[b].tolist() == com + pad
        assert int(got.accepted[b]) == acc and int(got.n_committed[b]) == len(com) and int(got.seq_status[b]) == st


def test_row_errors_end_the_walk_only_where_it_goes():
    rng = np.random.default_rng(1)
    seqs, nodes, V = 4, 5, 3001
    xsm, ctx, x, params, u = setup(rng, seqs, nodes, V)
    drawn = xsm.sample_batch(ctx, x, params, u, enc=V).token.view(seqs, nodes).cpu().numpy()
    parent = np.tile(np.array([-1, 0, 0, 2, 3], np.int32), (seqs, 1))
    tokens = np.zeros((seqs, nodes), np.int32)
    tokens[:, 1], tokens[:, 2], tokens[:, 3], tokens[:, 4] = V, drawn[:, 0], drawn[:, 2], drawn[:, 3]
    x[1 * nodes + 3, 17] = float("nan")   # on the way: the walk stops there
    x[2 * nodes + 1, 17] = float("nan")   # another branch
    x[3 * nodes, 17] = float("nan")       # the root
    got = xsm.verify_tree_batch(ctx, x, seqs, nodes, params, u, i32(tokens), i32(parent), enc=V)
    assert got.seq_status.tolist() == [0, _lib.ROW_NAN, 0, _lib.ROW_NAN]
    assert got.n_committed.tolist() == [4, 2, 4, 0] and got.accepted.tolist() == [3, 2, 3, 0]
    assert got.path.tolist() == [[0, 2, 3, 4, -1], [0, 2, -1, -1, -1], [0, 2, 3, 4, -1], [-1] * 5]
    # a tree's size out of bounds fails the sequence alone
    got = xsm.verify_tree_batch(ctx, x[:2 * nodes], 2, nodes, params, u, i32(tokens[:2]), i32(parent[:2]), enc=V, n_nodes=i32([4, 6]))
    assert got.seq_status.tolist() == [0, _lib.ROW_BAD_PARAM] and got.n_committed.tolist() == [3, 0]


def test_call_level_errors_fail_every_row():
    """A short mask and narrow rows, as xs_verify reports them; a budget of 0 asks for no row."""
    rng = np.random.default_rng(2)
    xsm, ctx, x, params, u = setup(rng, 2, 3, 3001)
    tokens, parent = i32(np.zeros((2, 3))), i32([[-1, 0, 1]] * 2)
    words = torch.full((6, 10), -1, dtype=torch.int32, device="cuda")
    got = xsm.verify_tree_batch(ctx, x, 2, 3, params, u, tokens, parent, enc=3001, allowed=words, budget=i32([5, 0]))
    assert got.row_status.tolist() == [_lib.ROW_MASK_SHORT] * 6 and got.row_token.tolist() == [-1] * 6
    assert got.seq_status.tolist() == [_lib.ROW_MASK_SHORT, 0] and got.n_committed.tolist() == [0, 0]
    assert got.path.tolist() == [[-1] * 3] * 2 and got.committed.tolist() == [[-1] * 3] * 2


def test_masks_and_controls_per_node():
    """Each node's own mask and controls, as xs_sample takes them."""
    rng = np.random.default_rng(3)
    seqs, nodes, V = 3, 6, 3001
    xsm, ctx, x, params, u = setup(rng, seqs, nodes, V, sharp=False)
    allow = rng.random((seqs * nodes, V)) < 0.3
    words = torch.from_numpy(workloads.pack_mask(allow).view(np.int32)).cuda()
    per_row = [None if r % 3 else xsm.SampleControl(force=int(np.nonzero(allow[r])[0][0])) for r in range(seqs * nodes)]
    ctl = xsm.controls_tensor(per_row, x.device)
    want = xsm.sample_batch(ctx, x, params, u, enc=V, allowed=words, controls=ctl)
    drawn = want.token.view(seqs, nodes).cpu().numpy()
    parent = np.tile(np.array([-1, 0, 1, 1, 3, 4], np.int32), (seqs, 1))
    tokens = np.zeros((seqs, nodes), np.int32)
    for b in range(seqs):
        for j in range(1, nodes):
            tokens[b, j] = drawn[b, parent[b, j]]
    got = xsm.verify_tree_batch(ctx, x, seqs, nodes, params, u, i32(tokens), i32(parent), enc=V, allowed=words, controls=ctl)
    assert torch.equal(got.row_token, want.token)
    for b in range(seqs):
        acc, path, com, _ = treeref.walk(drawn[b], np.zeros(nodes), tokens[b], parent[b], nodes, 99, (), np.zeros(nodes))
        assert got.path[b].tolist()[:len(path)] == path and got.committed[b].tolist()[:len(com)] == com and len(path) >= 3


def test_replayed_graphs():
    rng = np.random.default_rng(4)
    seqs, nodes, V = 4, 10, 20_011
    xsm, ctx, x, params, u = setup(rng, seqs, nodes, V)
    parent = i32([random_tree(rng, nodes) for _ in range(seqs)])
    tokens = i32(np.zeros((seqs, nodes)))
    out = xsm.verify_tree_batch(ctx, x, seqs, nodes, params, u, tokens, parent, enc=V)
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        ctx.bind_stream(s)
        xsm.verify_tree_batch(ctx, x, seqs, nodes, params, u, tokens, parent, enc=V, out=out)
    ctx.bind_current_stream()
    for _ in range(3):
        x.copy_(torch.randn(x.shape, device="cuda") * 2)
        drawn = xsm.sample_batch(ctx, x, params, u, enc=V).token.view(seqs, nodes)
        tokens[:, 1:] = drawn.gather(1, parent[:, 1:].long().clamp(min=0))
        eager = xsm.verify_tree_batch(ctx, x, seqs, nodes, params, u, tokens, parent, enc=V)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for f in ("row_token", "path", "committed", "n_committed", "accepted", "seq_status"):
            assert torch.equal(getattr(out, f), getattr(eager, f)), f
        assert int(eager.accepted.max()) > 0


def test_no_sequences():
    rng = np.random.default_rng(5)
    xsm, ctx, x, params, u = setup(rng, 1, 2, 1000)
    z = torch.empty((0, 2), dtype=torch.int32, device="cuda")
    assert xsm.verify_tree_batch(ctx, x[:0], 0, 2, params, u, z, z, enc=1000).n_committed.numel() == 0
