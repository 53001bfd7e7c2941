"""xs_qk_rotate on the device against the definition in 64 bits (tests/promptref.py)."""
import pytest
import torch

from tests import promptref

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def ctx():
    from xwen_amd import tree
    return tree.CacheContext(max_seqs=1, max_nodes=1, q_heads=1, kv_heads=1, head_dim=8, capacity=1)


def case(tokens, hq, h, d, dtype, rot, seed=0, norm=True, far=False, packed=False):
    from xwen_amd import prompt
    g = torch.Generator().manual_seed(seed + tokens)
    x = (torch.randn((tokens, hq + h + 2, d), generator=g) * 2).to(dtype).cuda()
    q, k = (x[:, :hq], x[:, hq:hq + h]) if packed else (x[:, :hq].contiguous(), x[:, hq:hq + h].contiguous())
    high = 2**31 - 1 if far else 200_000
    pos = torch.randint(-high if far else 0, high, (tokens,), generator=g).int()
    pos[0] = 2**31 - 1 if far else 0
    w = [(1 + 0.3 * torch.randn(d, generator=g)).cuda() if norm else None for _ in "qk"]
    return dict(q=q, k=k, pos=pos.cuda() if rot else None, inv_freq=prompt.frequencies(rot, 1e4, "cuda") if rot else None, w=w)


def run(ctx, c, neighbours=False, eps=1e-6, **kw):
    from xwen_amd import prompt
    return prompt.qk_rotate(ctx, c["q"], c["k"], c["pos"], inv_freq=c["inv_freq"], neighbours=neighbours, q_weight=c["w"][0],
                            k_weight=c["w"][1], eps=eps, **kw)


def agree(c, got, neighbours=False, eps=1e-6, src=None):
    for x, w, y in zip(src or (c["q"], c["k"]), c["w"], got):
        if x is None:
            assert y is None
            continue
        want, tol = promptref.rotate(x, w, eps, c["pos"], c["inv_freq"], neighbours)
        off = (y.double().cpu() - want).abs() / tol
        assert float(off.max()) <= 1.0, float(off.max())


@pytest.mark.parametrize("neighbours", [False, True])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d,rot", [(16, 16), (64, 64), (64, 32), (72, 48), (80, 80), (96, 96), (128, 128), (136, 64), (256, 64), (256, 256)])
def test_head_sizes(ctx, d, rot, dtype, neighbours):
    c = case(37, 6, 2, d, dtype, rot)
    agree(c, run(ctx, c, neighbours), neighbours)


def test_small_heads_and_odd_rotations(ctx):
    c = case(9, 3, 1, 8, HF, 8)
    agree(c, run(ctx, c, True), True)
    c = case(9, 3, 1, 8, BF, 0)
    agree(c, run(ctx, c))
    c = case(9, 3, 1, 24, BF, 16)
    agree(c, run(ctx, c))
    c = case(9, 3, 1, 24, BF, 24)
    agree(c, run(ctx, c, True), True)


@pytest.mark.parametrize("tokens", [1, 2, 3, 31, 33, 257, 2000, 5000])
@pytest.mark.parametrize("hq,h", [(16, 2), (1, 1), (7, 1), (32, 8)])
def test_tokens(ctx, tokens, hq, h):
    c = case(tokens, hq, h, 128, BF, 128, packed=tokens % 2 == 1)
    agree(c, run(ctx, c))


@pytest.mark.parametrize("tokens", [3, 6000])
def test_one_side_only(ctx, tokens):
    c = case(tokens, 5, 3, 256, HF, 256)
    for c1 in ({**c, "k": None}, {**c, "q": None}):
        agree(c1, run(ctx, c1))
    c1 = {**case(70000, 1, 1, 256, BF, 256), "k": None}  # one head a token: as many angles as elements
    agree(c1, run(ctx, c1))


@pytest.mark.parametrize("norm", [False, True])
def test_far_and_negative_positions(ctx, norm):
    c = case(300, 4, 2, 128, HF, 128, norm=norm, far=True)
    agree(c, run(ctx, c))


def test_no_norm_no_rotation_is_a_copy(ctx):
    c = case(40, 4, 2, 80, BF, 0, norm=False, packed=True)
    q, k = run(ctx, c)
    assert torch.equal(q, c["q"]) and torch.equal(k, c["k"])


def test_zero_rows_and_eps(ctx):
    c = case(8, 2, 1, 64, BF, 64)
    c["q"][3] = 0
    agree(c, run(ctx, c, eps=1e-2), eps=1e-2)
    c["k"][2, 0] = 0
    q, k = run(ctx, c, eps=0.0)
    assert bool(torch.isnan(k[2, 0]).all()) and bool(torch.isfinite(k[1]).all())  # 0 / 0


def test_a_token_that_is_not_finite_stays_its_own(ctx):
    c = case(20, 4, 2, 128, BF, 128)
    clean = [t.clone() for t in run(ctx, c)]
    c["q"][5, 1, 7] = float("nan")
    c["k"][6, 0, 3] = float("inf")
    q, k = run(ctx, c)
    for got, was, at in ((q, clean[0], (5, 1)), (k, clean[1], (6, 0))):
        other = torch.ones(got.shape[:2], dtype=torch.bool)
        other[at] = False
        assert torch.equal(got[other.cuda()], was[other.cuda()]) and not bool(torch.isfinite(got[at]).all())


@pytest.mark.parametrize("neighbours", [False, True])
def test_in_place_and_into_strided_outputs(ctx, neighbours):
    c = case(130, 6, 2, 80, HF, 64, packed=True)
    src = (c["q"].clone(), c["k"].clone())
    wide = torch.full((130, 2, 96), 7.0, dtype=HF, device="cuda")
    got = run(ctx, c, neighbours, q_out=c["q"], k_out=wide[:, :, :80])
    assert got[0].data_ptr() == c["q"].data_ptr()
    agree(c, got, neighbours, src=src)
    assert bool((wide[:, :, 80:] == 7).all())


def test_same_results_wherever_a_head_lies(ctx):
    """A token's results do not depend on the others of the call."""
    c = case(4000, 32, 8, 128, BF, 128)
    q, k = run(ctx, c)
    one = {**c, "q": c["q"][777:778], "k": c["k"][777:778], "pos": c["pos"][777:778]}
    a, b = run(ctx, one)
    assert torch.equal(a[0], q[777]) and torch.equal(b[0], k[777])


def test_a_graph_replays(ctx):
    c = case(50, 4, 2, 128, BF, 128)
    want = [t.clone() for t in run(ctx, c)]
    out = [torch.zeros_like(t) for t in want]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        run(ctx, c, q_out=out[0], k_out=out[1])
    for _ in range(3):
        for t in out:
            t.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
        again = run(ctx, c)
        assert torch.equal(again[0], want[0])


def test_refusals(ctx):
    from xwen_amd import _lib, prompt
    c = case(10, 4, 2, 64, BF, 64)
    f = prompt.qk_rotate
    for kw in (dict(pos=c["pos"]), dict(pos=c["pos"].long(), inv_freq=c["inv_freq"]), dict(q_weight=c["w"][0]),
               dict(q_weight=c["w"][0].half(), k_weight=c["w"][1]), dict(pos=c["pos"][:9], inv_freq=c["inv_freq"])):
        with pytest.raises(ValueError):
            f(ctx, c["q"], c["k"], **kw)
    with pytest.raises(ValueError):
        f(ctx, c["q"], c["k"].half())
    with pytest.raises(ValueError):
        f(ctx, None, None)
    with pytest.raises(ValueError):
        f(ctx, c["q"].cpu(), c["k"].cpu())
    with pytest.raises(_lib.XsError):
        f(ctx, c["q"], c["k"], c["pos"], inv_freq=c["inv_freq"][:12])  # 24 elements as halves
    with pytest.raises(_lib.XsError):
        f(ctx, c["q"][:, :, 4:60], c["k"][:, :, 4:60])  # off the 16-byte grid
