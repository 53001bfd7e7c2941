"""The prompt's and the 8-bit cache's calls where offsets pass 32 bits, at the largest strides, and
on streams that change between the calls."""
import math

import numpy as np
import pytest
import torch

from tests import promptref, treeref
from tests.test_gpu_cache8 import filled, look, step

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def ctx():
    from xwen_amd import tree
    return tree.CacheContext(max_seqs=4, max_nodes=64, q_heads=32, kv_heads=16, head_dim=256, capacity=8192)


def test_prompt_rows_past_32_bits(ctx):
    """2 MiB from token to token: the last of 2,200 tokens lie 4.6 GB in."""
    from xwen_amd import prompt
    g = torch.Generator().manual_seed(1)
    n, stride = 2200, 1 << 20
    room = torch.empty(n * stride + 4096, dtype=BF, device="cuda")
    parts = [torch.randn((n, h, 64), generator=g).to(BF).cuda() for h in (2, 1, 1)]
    views = []
    for i, t in enumerate(parts):
        v = room.as_strided(t.shape, (stride, 64, 1), i * 1024)
        v.copy_(t)
        views.append(v)
    out = prompt.PromptAttended(out=room.as_strided((n, 2, 64), (stride, 64, 1), 2560), lse=torch.zeros((n, 2), device="cuda"),
                                seq_status=torch.zeros(1, dtype=torch.int32, device="cuda"))
    start = torch.tensor([0, n], dtype=torch.int32).cuda()
    prompt.prompt_attend(ctx, *views, start, out=out)
    want = prompt.prompt_attend(ctx, *parts, start)
    assert out.seq_status.tolist() == [0] and torch.equal(out.out, want.out) and torch.equal(out.lse, want.lse)
    promptref.agree(want.out, want.lse, promptref.prompt_wide(*parts, [0, n], float(np.float32(0.125))))
    pos = torch.arange(n, dtype=torch.int32).cuda()
    freq = prompt.frequencies(64, 1e4, "cuda")
    a = prompt.qk_rotate(ctx, parts[0], parts[1], pos, inv_freq=freq)
    b = prompt.qk_rotate(ctx, views[0], views[1], pos, inv_freq=freq, q_out=views[0], k_out=views[1])
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_cache_slots_past_32_bits(ctx):
    """A mebibyte from slot to slot: the last of 4,400 lie 4.6 GB in; the same cache packed."""
    from xwen_amd import cache8
    cap, stride = 4400, 1 << 20
    room = torch.empty(cap * stride + 4096, dtype=torch.uint8, device="cuda")
    far = {n: room.as_strided((1, cap, 2, 64), (stride, stride, 64, 1), i * 1024).view(torch.float8_e4m3fn) for i, n in enumerate("kv")}
    near = filled([4390], 2, 64, cap=cap)
    exps = {n: near[n + "_exp"].clone() for n in "kv"}
    for n in "kv":
        far[n].view(torch.uint8).copy_(near[n].view(torch.uint8))
    rng = np.random.default_rng(1)
    for nodes in (1, 12, 40):
        s = step(rng, near, nodes, 4, BF)
        want = look(ctx, near, s)
        got = look(ctx, {**near, **far}, s)
        assert torch.equal(got.out, want.out) and torch.equal(got.lse, want.lse)
    g = torch.Generator().manual_seed(2)
    fk, fv = (torch.randn((1, 10, 2, 64), generator=g).to(HF).cuda() * 4 for _ in "kv")
    a = cache8.cache_append8(ctx, near["k"], near["v"], near["k_exp"], near["v_exp"], near["len"], fk, fv)
    b = cache8.cache_append8(ctx, far["k"], far["v"], exps["k"], exps["v"], near["len"], fk, fv)
    assert a.new_len.tolist() == b.new_len.tolist() == [4400]
    for n in "kv":
        assert torch.equal(near[n].view(torch.uint8), far[n].view(torch.uint8)) and torch.equal(near[n + "_exp"], exps[n])


def test_long_fresh_rows_past_32_bits(ctx):
    """Rows of a packed prompt that lie 4.6 GB in, appended."""
    from xwen_amd import cache8
    n, stride = 2200, 1 << 20
    room = torch.empty(n * stride + 4096, dtype=BF, device="cuda")
    g = torch.Generator().manual_seed(3)
    packed = [torch.randn((n, 1, 64), generator=g).to(BF).cuda() for _ in "kv"]
    spread = []
    for i, t in enumerate(packed):
        v = room.as_strided(t.shape, (stride, 64, 1), i * 1024)
        v.copy_(t)
        spread.append(v)
    caches = [cache8.Cache8(ctx, 1, 1, 64, n) for _ in range(2)]
    start = torch.tensor([0, n], dtype=torch.int32).cuda()
    for c, rows in zip(caches, (packed, spread)):
        cache8.cache_append8(ctx, c.k, c.v, c.k_exp, c.v_exp, c.length, *rows, start=start)
    for f in ("k", "v", "k_exp", "v_exp"):
        assert torch.equal(*(getattr(c, f).view(torch.uint8) for c in caches)), f


def test_streams_that_change_between_the_calls(ctx):
    """A step's calls on streams in turn: the context orders them, their workspace is shared."""
    rng = np.random.default_rng(4)
    c = filled([4000, 1500], 2, 128)
    steps = [step(rng, c, n, 8, BF) for n in (1, 30, 4, 64)]
    want = [look(ctx, c, s) for s in steps]
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for i, s in enumerate(steps * 3):
        with torch.cuda.stream(streams[i % 3]):
            got.append(look(ctx, c, s))
    torch.cuda.synchronize()
    for i, x in enumerate(got):
        assert torch.equal(x.out, want[i % 4].out) and torch.equal(x.lse, want[i % 4].lse), i


def test_captured_calls_on_forked_streams(ctx):
    """Two trees' attention in one capture that forks: replayed with eager calls between."""
    rng = np.random.default_rng(5)
    from xwen_amd import cache8, tree
    c = filled([4000, 1500], 2, 128)
    steps = [step(rng, c, n, 8, BF) for n in (2, 30)]
    want = [look(ctx, c, s) for s in steps]
    outs = [tree.Attended(*(torch.zeros_like(t) for t in (w.out, w.lse, w.seq_status))) for w in want]
    parents = [s["parent"].cuda() for s in steps]
    side = torch.cuda.Stream()

    def call(i):
        s = steps[i]
        cache8.tree_attend8(ctx, s["q"], c["k"], c["v"], c["k_exp"], c["v_exp"], c["len"], s["fk"], s["fv"], parents[i], out=outs[i])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        call(0)
        with torch.cuda.stream(side):
            call(1)
        main.wait_stream(side)
    for _ in range(4):
        for o in outs:
            o.out.zero_()
        g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o.out, w.out) and torch.equal(o.lse, w.lse)
        assert torch.equal(look(ctx, c, steps[0]).out, want[0].out)
        torch.cuda.synchronize()


def test_one_sequence_twice(ctx):
    """The same rows under two sequences of an append, and one cache read by two sequences."""
    from xwen_amd import cache8
    g = torch.Generator().manual_seed(6)
    rows = [torch.randn((50, 2, 64), generator=g).to(BF).cuda() for _ in "kv"]
    c = cache8.Cache8(ctx, 2, 2, 64, 64)
    one = cache8.cache_append8(ctx, c.k, c.v, c.k_exp, c.v_exp, c.length, *(t.unsqueeze(0).expand(2, 50, 2, 64) for t in rows))
    assert one.new_len.tolist() == [50, 50]
    assert torch.equal(c.k.view(torch.uint8)[0], c.k.view(torch.uint8)[1]) and torch.equal(c.k_exp[0], c.k_exp[1])
    q = torch.randn((1, 3, 4, 64), generator=g).to(BF).cuda().expand(2, 3, 4, 64)
    fk = torch.randn((2, 3, 2, 64), generator=g).to(BF).cuda()
    parent = torch.tensor([[-1, 0, 1]] * 2, dtype=torch.int32).cuda()
    fk = fk[:1].expand(2, 3, 2, 64)
    a = cache8.tree_attend8(ctx, q, c.k[:1].expand(2, 64, 2, 64), c.v[:1].expand(2, 64, 2, 64), c.k_exp, c.v_exp, one.new_len, fk, fk, parent)
    assert torch.equal(a.out[0], a.out[1])
    k, v = promptref.Cache(c.k, c.v, c.k_exp, c.v_exp, [50, 50]).values()
    want = treeref.attend(q, k, v, [50, 50], fk, fk, parent.cpu(), [3, 3], float(np.float32(1 / math.sqrt(64))))
    promptref.agree(a.out, a.lse, want)
