"""One cache context on the forked streams of a captured step: its calls share a workspace, so the
graph has to run them one after the other."""
import numpy as np
import pytest
import torch

from tests.test_gpu_tree_attend import BF, blank, case, context, run

pytestmark = pytest.mark.gpu


def test_forks_of_a_captured_step():
    """Two layers' attention on two streams of one graph, long enough to be split and joined,
    replayed with new queries and eager calls between."""
    from xwen_amd import tree
    ctx = context()
    rng = np.random.default_rng(1)
    cs = [case(rng, [7000, 3000], 8, 8, 2, 128, BF), case(rng, [6000, 500], 8, 8, 2, 128, BF)]
    held = [dict(length=torch.tensor(c["lens"], dtype=torch.int32).cuda(), parent=c["parent"].cuda(), out=blank(c)) for c in cs]

    def attend(j):
        c, h = cs[j], held[j]
        tree.tree_attend(ctx, c["q"], c["k"], c["v"], h["length"], c["fk"], c["fv"], h["parent"], out=h["out"])

    for j in range(2):
        attend(j)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        for _ in range(3):
            attend(0)
            with torch.cuda.stream(side):
                attend(1)
        main.wait_stream(side)
    for _ in range(4):
        for c in cs:
            c["q"].copy_(torch.randn(c["q"].shape, device="cuda"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for c, h in zip(cs, held):
            want = run(ctx, c, out=blank(c))
            assert torch.equal(h["out"].out, want.out) and torch.equal(h["out"].lse, want.lse)
    ctx.close()
