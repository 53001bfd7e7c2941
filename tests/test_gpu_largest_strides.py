"""The largest strides that the calls take, over whole stages of keys and parts of one, against packed
copies: 2^24 elements from token to token of a prompt, 2^25 bytes from slot to slot of an 8-bit cache."""
import numpy as np
import pytest
import torch

from tests.test_gpu_cache8 import filled, look, step
from tests.test_gpu_prompt import blank, case
from xwen_amd import _lib

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
PROMPT, CACHE = 1 << 24, 1 << 25


@pytest.fixture(scope="module")
def ctx():
    from xwen_amd import tree
    return tree.CacheContext(max_seqs=1, max_nodes=64, q_heads=64, kv_heads=2, head_dim=256, capacity=1024)


@pytest.mark.parametrize("n", [65, 100])
@pytest.mark.parametrize("d,hq,h,dtype", [(64, 4, 2, BF), (64, 1024, 1, HF), (128, 4, 2, HF), (128, 1024, 1, BF), (80, 3, 1, BF), (256, 4, 2, BF)])
def test_prompts(ctx, n, d, hq, h, dtype):
    """Tiles of 64 and of 128 rows (1,024 query heads)."""
    from xwen_amd import prompt
    c = case([n], hq, h, d, dtype)
    start = torch.tensor([0, n], dtype=torch.int32).cuda()
    want = prompt.prompt_attend(ctx, c["q"], c["k"], c["v"], start, out=blank(c))
    room = torch.empty(n * PROMPT, dtype=dtype, device="cuda")
    far = []
    for i, name in enumerate("kv"):
        t = room.as_strided(c[name].shape, (PROMPT, d, 1), i * 8192)
        t.copy_(c[name])
        far.append(t)
    got = prompt.prompt_attend(ctx, c["q"], *far, start, out=blank(c))
    assert torch.equal(got.out, want.out) and torch.equal(got.lse, want.lse)
    over = room.as_strided((2, h, d), (PROMPT + 8, d, 1))
    with pytest.raises(_lib.XsError):
        prompt.prompt_attend(ctx, c["q"][:2], over, over, torch.tensor([0, 2], dtype=torch.int32).cuda())


@pytest.mark.parametrize("n", [65, 100])
@pytest.mark.parametrize("d,dtype", [(64, HF), (128, BF), (80, BF), (256, BF)])
def test_caches(ctx, n, d, dtype):
    """Single rows, rows that two waves share, tiles of 128 and of 256; then rows appended."""
    from xwen_amd import cache8
    near = filled([n], 2, d, cap=n + 4)
    room = torch.empty((n + 4) * CACHE, dtype=torch.uint8, device="cuda")
    far = {}
    for i, name in enumerate("kv"):
        far[name] = room.as_strided((1, n + 4, 2, d), (CACHE, CACHE, d, 1), i * 8192).view(torch.float8_e4m3fn)
        far[name].view(torch.uint8).copy_(near[name].view(torch.uint8))
        far[name + "_exp"] = near[name + "_exp"].clone()
    rng = np.random.default_rng(n)
    for nodes, group in ((1, 1), (5, 4), (20, 4), (64, 4)):
        s = step(rng, near, nodes, 2 * group, dtype)
        want, got = look(ctx, near, s), look(ctx, {**near, **far}, s)
        assert torch.equal(got.out, want.out) and torch.equal(got.lse, want.lse)
    rows = [torch.randn((1, 4, 2, d), generator=torch.Generator().manual_seed(n)).to(dtype).cuda() * 9 for _ in "kv"]
    for c in (near, far):
        cache8.cache_append8(ctx, c["k"], c["v"], c["k_exp"], c["v_exp"], near["len"], *rows)
    for name in "kv":
        assert torch.equal(near[name].view(torch.uint8), far[name].view(torch.uint8)) and torch.equal(near[name + "_exp"], far[name + "_exp"])
    wide = room.as_strided((1, 2, 2, d), (CACHE + 16, CACHE + 16, d, 1)).view(torch.float8_e4m3fn)
    with pytest.raises(_lib.XsError):
        look(ctx, {**near, "k": wide, "v": wide, "len": torch.ones_like(near["len"])}, s)
