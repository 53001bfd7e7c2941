"""The calls from a prompt to an 8-bit cache as they are used together: projections rotated,
prompts attended and appended, then steps of draft trees attended, verified and committed."""
import math

import numpy as np
import pytest
import torch

from tests import promptref, treeref

pytestmark = pytest.mark.gpu

B, HQ, H, D, N, V = 3, 8, 2, 128, 6, 512
PARENT = [-1, 0, 0, 1, 1, 2]
DEPTH = [0, 1, 1, 2, 2, 2]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_prompt_and_steps(dtype):
    from xwen_amd import cache8, prompt, tree
    from xwen_amd import sampler as xs
    g = torch.Generator().manual_seed(11)
    ctx = tree.CacheContext(max_seqs=B, max_nodes=N, q_heads=HQ, kv_heads=H, head_dim=D, capacity=300)
    sctx = xs.Context(max_rows=B * N, vocab=V)
    cache = cache8.Cache8(ctx, B, H, D, 300)
    freq = prompt.frequencies(64, 1e6, "cuda")
    w = [(1 + 0.2 * torch.randn(D, generator=g)).cuda() for _ in "qk"]
    scale = float(np.float32(1 / math.sqrt(D)))

    def project(rows):
        return torch.randn((rows, HQ + 2 * H, D), generator=g).to(dtype).cuda()

    def turned(x, pos):
        q, k = prompt.qk_rotate(ctx, x[:, :HQ], x[:, HQ:HQ + H], pos, inv_freq=freq, q_weight=w[0], k_weight=w[1])
        for t, y, wt in ((x[:, :HQ], q, w[0]), (x[:, HQ:HQ + H], k, w[1])):
            want, tol = promptref.rotate(t, wt, 1e-6, pos, freq, False)
            assert bool(((y.double().cpu() - want).abs() <= tol).all())
        return q, k, x[:, HQ + H:]

    lens = [100, 1, 64]
    start = np.concatenate([[0], np.cumsum(lens)])
    ref = promptref.Cache(cache.k, cache.v, cache.k_exp, cache.v_exp, [0] * B)
    q, k, v = turned(project(int(start[-1])), torch.cat([torch.arange(n) for n in lens]).int().cuda())
    # (k is a new tensor, v a slice of the projection: prompt() takes pairs of one layout)
    v = v.contiguous()
    a = cache.prompt(q, k, v, torch.tensor(start, dtype=torch.int32).cuda(), max_len=100)
    tree.check(a.seq_status)
    tree.check(cache.append_status)
    promptref.agree(a.out, a.lse, promptref.prompt(q, k, v, start.tolist(), scale))
    for b, (i, j) in enumerate(zip(start, start[1:])):
        ref.append(b, k[i:j], v[i:j])
    ref.check(cache.k, cache.v, cache.k_exp, cache.v_exp)

    parent = torch.tensor([PARENT] * B, dtype=torch.int32).cuda()
    for step in range(4):
        assert cache.length.tolist() == ref.lens
        pos = (cache.length[:, None] + torch.tensor(DEPTH, device="cuda")).int().flatten()
        q, k, v = turned(project(B * N), pos)
        q, k, v = q.view(B, N, HQ, D), k.view(B, N, H, D), v.contiguous().view(B, N, H, D)
        a = cache.attend(q, k, v, parent)
        tree.check(a.seq_status)
        kk, vv = ref.values()
        promptref.agree(a.out, a.lse, treeref.attend(q, kk, vv, ref.lens, k, v, torch.tensor([PARENT] * B), [N] * B, scale))
        # drafts that the greedy sampler takes: node 1, then 3 or 4; a whole path, a part, none
        logits = torch.zeros((B, N, V), device="cuda")
        tokens = torch.tensor([[9, 20, 21, 30, 31, 32]] * B, dtype=torch.int32)
        logits[0, 0, 20], logits[0, 1, 31], logits[0, 4, 77] = 9.0, 9.0, 9.0
        logits[1, 0, 21], logits[1, 2, 50] = 9.0, 9.0
        logits[2, 0, 400] = 9.0
        params = xs.params_tensor(0.0, 1, 1.0, B * N, "cuda")
        verdict = xs.verify_tree_batch(sctx, logits.view(B * N, V), B, N, params, torch.zeros(B * N, device="cuda"), tokens.cuda(), parent)
        assert verdict.n_committed.tolist() == [3, 2, 1]
        cache.commit(k, v, verdict.path, verdict.n_committed)
        tree.check(cache.append_status)
        for b, path in enumerate(([0, 1, 4], [0, 2], [0])):
            ref.append(b, k[b, path], v[b, path])
        ref.check(cache.k, cache.v, cache.k_exp, cache.v_exp)


def test_a_step_replays_in_a_graph():
    """attend and commit captured once, replayed with the buffers' new contents."""
    from xwen_amd import cache8, tree
    g = torch.Generator().manual_seed(12)
    ctx = tree.CacheContext(max_seqs=2, max_nodes=4, q_heads=4, kv_heads=2, head_dim=64, capacity=100)
    caches = [cache8.Cache8(ctx, 2, 2, 64, 100) for _ in range(2)]
    start = torch.tensor([0, 30, 41], dtype=torch.int32).cuda()
    qkv = [torch.randn((41, h, 64), generator=g).bfloat16().cuda() for h in (4, 2, 2)]
    for c in caches:
        c.prompt(*qkv, start)
    q, k, v = (torch.zeros((2, 4, h, 64), dtype=torch.bfloat16, device="cuda") for h in (4, 2, 2))
    parent = torch.tensor([[-1, 0, 1, 2]] * 2, dtype=torch.int32).cuda()
    path = torch.tensor([[0, 1, 2, 3]] * 2, dtype=torch.int32).cuda()
    n = torch.tensor([3, 1], dtype=torch.int32).cuda()
    out = tree.Attended(torch.zeros_like(q), torch.zeros((2, 4, 4), device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda"))

    def step(c, out):
        a = c.attend(q, k, v, parent, out=out)
        c.commit(k, v, path, n)
        return a
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(caches[0], out)
    for i in range(4):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        want = step(caches[1], None)
        assert torch.equal(out.out, want.out) and torch.equal(out.lse, want.lse)
        for a, b in zip(*((c.k.view(torch.uint8), c.v.view(torch.uint8), c.k_exp, c.v_exp, c.length) for c in caches)):
            assert torch.equal(a, b)
    assert caches[0].length.tolist() == [42, 15]
