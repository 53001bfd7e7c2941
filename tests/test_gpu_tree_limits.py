"""The largest launches of the cache calls, and the first ones past them, which are refused."""
import pytest
import torch

from xwen_amd import _lib

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def test_attend_up_to_the_largest_launch():
    """2^24 (sequence, kv head) pairs are one too many for workgroups of 256; 256 fewer run.
    Every sequence sees the same two slots and one node."""
    from xwen_amd import tree
    seqs, heads = 65_536, 256
    ctx = tree.CacheContext(max_seqs=seqs, max_nodes=1, q_heads=heads, kv_heads=heads, head_dim=8, capacity=8)
    one = {n: torch.randn((1, s, heads, 8), device="cuda").to(BF) for n, s in (("q", 1), ("k", 8), ("v", 8), ("fk", 1), ("fv", 1))}

    def attend(n):
        t = {x: y.expand(n, *y.shape[1:]) for x, y in one.items()}
        return tree.tree_attend(ctx, t["q"], t["k"], t["v"], torch.full((n,), 2, dtype=torch.int32, device="cuda"), t["fk"], t["fv"],
                                torch.full((n, 1), -1, dtype=torch.int32, device="cuda"))
    want, most = attend(1), attend(seqs - 1)
    assert not bool(most.seq_status.any())
    assert torch.equal(most.out, want.out.expand_as(most.out)) and torch.equal(most.lse, want.lse.expand_as(most.lse))
    with pytest.raises(_lib.XsError, match="XS_ERR_CAPACITY"):
        attend(seqs)
    ctx.close()


def test_evict_up_to_the_largest_launch():
    """2^22 pairs for workgroups of 1,024."""
    from xwen_amd import tree
    seqs, heads = 65_536, 64
    ctx = tree.CacheContext(max_seqs=seqs, max_nodes=1, q_heads=heads, kv_heads=heads, head_dim=8, capacity=8)
    k, v = (torch.randn((seqs, 8, heads, 8), device="cuda").to(BF) for _ in "kv")
    mass = torch.tensor([3.0, 1.0, 2.0, 0.0, 5.0, 4.0, 0.5, 0.25], device="cuda").repeat(seqs, heads, 1)
    pos = torch.arange(8, dtype=torch.int32, device="cuda").repeat(seqs, heads, 1)
    length = torch.full((seqs,), 8, dtype=torch.int32, device="cuda")

    def evict(n):
        return tree.cache_evict(ctx, k[:n], v[:n], length[:n], mass[:n], pos[:n], length[:n], 4)
    start = k.clone()
    with pytest.raises(_lib.XsError, match="XS_ERR_CAPACITY"):
        evict(seqs)
    assert torch.equal(k, start)
    got = evict(seqs - 1)
    assert not bool(got.seq_status.any()) and bool((got.new_len == 4).all())
    # slots 4 and 5 (the heaviest) take the places of 1 and 3
    source = [0, 4, 2, 5]
    assert torch.equal(k[:-1, :4], start[:-1, source]) and torch.equal(k[-1], start[-1])
    assert bool((pos[:-1, :, :4] == torch.tensor(source, dtype=torch.int32, device="cuda")).all())
    ctx.close()


def test_a_context_that_cannot_be_made_leaves_no_error():
    """Sizes that no memory holds and a device that is not there: refused, and what follows runs."""
    from xwen_amd import tree
    for bad in (dict(max_seqs=65_536, q_heads=4096, kv_heads=4096, capacity=1 << 28), dict(device=torch.cuda.device_count())):
        with pytest.raises(_lib.XsError, match="XS_ERR_HIP"):
            tree.CacheContext(**{**dict(max_seqs=1, max_nodes=1, q_heads=1, kv_heads=1, head_dim=64, capacity=64), **bad})
        assert float(torch.ones(5, device="cuda").sum()) == 5.0
        ctx = tree.CacheContext(max_seqs=1, max_nodes=1, q_heads=1, kv_heads=1, head_dim=64, capacity=64)
        t = torch.ones((1, 64, 1, 64), device="cuda", dtype=BF)
        n = torch.ones(1, dtype=torch.int32, device="cuda")
        got = tree.tree_attend(ctx, t[:, :1], t, t, n, t[:, :1], t[:, :1], -n.view(1, 1))
        tree.check(got.seq_status)
        assert bool((got.out == 1.0).all())
        ctx.close()
