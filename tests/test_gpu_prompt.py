"""xs_prompt_attend on the device against the definition in 64 bits (tests/promptref.py)."""
import math

import numpy as np
import pytest
import torch

from tests import promptref

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def ctx():
    from xwen_amd import tree
    return tree.CacheContext(max_seqs=1, max_nodes=1, q_heads=1, kv_heads=1, head_dim=8, capacity=1)


def case(lens, hq, h, d, dtype, seed=0, packed=False, spread=1.0, front=0, back=0):
    g = torch.Generator().manual_seed(seed + sum(lens) + d)
    T = front + sum(lens) + back
    x = torch.randn((T, hq + 2 * h, d), generator=g)
    x[:, :hq + h] *= spread
    x = x.to(dtype).cuda()
    parts = x[:, :hq], x[:, hq:hq + h], x[:, hq + h:]
    q, k, v = parts if packed else (t.contiguous() for t in parts)
    return dict(q=q, k=k, v=v, start=(front + np.concatenate([[0], np.cumsum(lens)])).tolist())


def blank(c, fill=7.0, seqs=None):
    from xwen_amd import prompt
    T, HQ, D = c["q"].shape
    return prompt.PromptAttended(out=torch.full((T, HQ, D), fill, dtype=c["q"].dtype, device="cuda"),
                                 lse=torch.full((T, HQ), fill, device="cuda"),
                                 seq_status=torch.full((len(c["start"]) - 1,), -1, dtype=torch.int32, device="cuda"))


def run(ctx, c, scale=None, out=None):
    from xwen_amd import prompt
    start = torch.tensor(c["start"], dtype=torch.int32).cuda()
    return prompt.prompt_attend(ctx, c["q"], c["k"], c["v"], start, scale=scale, out=out or blank(c))


def agree(c, got, scale=None):
    scale = float(np.float32(1.0 / math.sqrt(c["q"].shape[-1]) if scale is None else scale))
    assert got.seq_status.tolist() == [0] * (len(c["start"]) - 1)
    promptref.agree(got.out, got.lse, promptref.prompt(c["q"], c["k"], c["v"], c["start"], scale), left=7.0)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d", [8, 16, 40, 64, 72, 80, 96, 104, 128, 136, 192, 256])
def test_head_sizes(ctx, d, dtype):
    c = case([0, 1, 33, 130, 200], 4, 2, d, dtype, packed=d % 16 == 0)
    agree(c, run(ctx, c))


@pytest.mark.parametrize("hq,h", [(1, 1), (3, 3), (4, 1), (7, 1), (10, 2), (16, 1), (24, 8), (48, 1), (130, 1)])
def test_head_layouts(ctx, hq, h):
    c = case([70, 5, 1], hq, h, 64, BF)
    agree(c, run(ctx, c))


@pytest.mark.parametrize("hq,h,d,dtype", [(2, 1, 128, BF), (3, 1, 64, HF), (1, 1, 256, BF), (2, 2, 96, HF)])
def test_lengths(ctx, hq, h, d, dtype):
    lens = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 191, 192, 193, 255, 256, 257, 320, 449]
    c = case(lens, hq, h, d, dtype, front=3, back=5)
    agree(c, run(ctx, c))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("hq,h,d", [(4, 1, 128), (2, 1, 256), (2, 2, 64), (6, 2, 80)])
def test_long_with_large_scores(ctx, hq, h, d, dtype):
    c = case([1500, 700], hq, h, d, dtype, spread=1.7)
    agree(c, run(ctx, c))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d", [64, 72, 96, 128])
def test_enough_rows_to_fill_the_device(ctx, d, dtype):
    """128 rows a workgroup: from 65,536 rows (tokens times q heads) on."""
    c = case([1700, 0, 1, 333, 70], 32, 4, d, dtype, packed=True, spread=1.5, front=1)
    got = run(ctx, c)
    assert got.seq_status.tolist() == [0] * 5
    promptref.agree(got.out, got.lse, promptref.prompt_wide(c["q"], c["k"], c["v"], c["start"], float(np.float32(1 / math.sqrt(d)))), left=7.0)


@pytest.mark.parametrize("dtype", [BF, HF])
def test_what_is_not_finite_with_many_rows(ctx, dtype):
    c = case([1000, 1100], 32, 2, 128, dtype)
    clean = run(ctx, c)
    c["v"][500, 0, 3], c["v"][501, 1, 4], c["k"][700, 0, 5] = math.inf, math.nan, math.nan
    got = run(ctx, c)
    assert torch.equal(got.out[:500], clean.out[:500]) and torch.equal(got.out[1000:], clean.out[1000:])
    assert bool((got.out[500:700, :16, 3] == math.inf).all()) and bool(torch.isnan(got.out[501:1000, 16:, 4]).all())
    assert bool(torch.isnan(got.out[700:1000, :16]).all()) and torch.equal(got.out[500:1000, 16:, 5:], clean.out[500:1000, 16:, 5:])


def test_many_sequences(ctx):
    """More than a wave of them, empty ones among them."""
    rng = np.random.default_rng(1)
    lens = rng.integers(0, 12, 300).tolist()
    lens[150], lens[63], lens[64], lens[299] = 100, 0, 40, 0
    c = case(lens, 2, 1, 64, BF, front=2)
    agree(c, run(ctx, c))


def test_exactly_a_wave_of_sequences(ctx):
    rng = np.random.default_rng(2)
    for n in (63, 64, 65):
        c = case(rng.integers(0, 70, n).tolist(), 2, 1, 64, HF)
        agree(c, run(ctx, c))


def test_every_sequence_is_its_own(ctx):
    """Bit for bit what a call of its own gives, whatever lies beside it."""
    c = case([300, 77, 129], 8, 2, 128, BF, packed=True)
    got = run(ctx, c)
    for a, b in zip(c["start"], c["start"][1:]):
        one = {n: c[n][a:b] for n in "qkv"} | {"start": [0, b - a]}
        alone = run(ctx, one)
        assert torch.equal(alone.out, got.out[a:b]) and torch.equal(alone.lse, got.lse[a:b])


def test_strided_and_repeated_rows(ctx):
    c = case([90, 41], 6, 2, 64, BF)
    wide = torch.randn((131, 2, 160), device="cuda").to(BF)
    c["k"], c["v"] = wide[:, :, :64], wide[:, :, 96:]
    c["q"] = c["q"][:, :1].expand(131, 6, 64)
    agree(c, run(ctx, c))
    c["k"], c["v"] = (torch.randn((131, 1, 64), device="cuda").to(BF).expand(131, 2, 64) for _ in "kv")
    agree(c, run(ctx, c))
    heads = [torch.randn((2, 131, 64), device="cuda").to(BF).transpose(0, 1) for _ in "kv"]  # heads outermost
    c["k"], c["v"] = heads
    out = blank(c)
    out.out = torch.full((6, 131, 64), 7.0, dtype=BF, device="cuda").transpose(0, 1)
    agree(c, run(ctx, c, out=out))


def test_sequences_that_fail(ctx):
    c = case([40, 30, 20, 10], 4, 2, 64, BF)
    T = 100
    # (start, which sequences hold)
    for start, good in (([0, 40, 70, 90, 101], [1, 1, 1, 0]), ([-1, 40, 70, 90, 100], [0, 1, 1, 1]),
                        ([0, 40, 30, 90, 100], [1, 0, 0, 1]), ([0, 60, 10, 55, 100], [1, 0, 0, 0]),
                        ([0, 100, 0, 100, 0], [1, 0, 0, 0]), ([T, T, T, T, T], [1, 1, 1, 1]), ([2**31 - 1, 0, 40, 90, -5], [0, 0, 0, 0]),
                        ([-2**31, 2**31 - 1, -2**31, 3, 9], [0, 0, 0, 0])):
        c["start"] = start
        got = run(ctx, c)
        assert (got.seq_status == 0).int().tolist() == good, (start, got.seq_status.tolist())
        assert set(got.seq_status.tolist()) <= {0, 7}
        spans = [(a, b) for a, b, ok in zip(start, start[1:], good) if ok]
        left = torch.ones(T, dtype=torch.bool)
        for a, b in spans:
            one = {n: c[n][a:b] for n in "qkv"} | {"start": [0, b - a]}
            if b > a:
                agree(one, type(got)(out=got.out[a:b], lse=got.lse[a:b], seq_status=got.seq_status[:1] * 0))
            left[a:b] = False
        assert bool((got.out[left.cuda()] == 7).all()) and bool((got.lse[left.cuda()] == 7).all()), start


def test_failing_sequences_among_many(ctx):
    lens = [5] * 200
    c = case(lens, 1, 1, 64, BF)
    start = list(c["start"])
    c["start"][100] = 3       # 99 ends before it starts, 100 begins inside earlier ones
    got = run(ctx, c)
    assert [i for i, s in enumerate(got.seq_status.tolist()) if s] == [99, 100]
    want = run(ctx, {**c, "start": start})
    assert torch.equal(got.out[:99 * 5], want.out[:99 * 5]) and torch.equal(got.out[101 * 5:], want.out[101 * 5:])
    assert bool((got.out[99 * 5:101 * 5] == 7).all())


def test_no_tokens(ctx):
    from xwen_amd import prompt
    x = torch.empty((0, 2, 64), dtype=BF, device="cuda")
    for start, want in (([0, 0, 0], [0, 0]), ([0, 1, 0], [7, 7]), ([0], [])):
        got = prompt.prompt_attend(ctx, x, x, x, torch.tensor(start, dtype=torch.int32).cuda())
        assert got.seq_status.tolist() == want and got.out.shape == (0, 2, 64)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_what_a_token_does_not_see_never_reaches_it(ctx, d, dtype):
    c = case([150, 90], 4, 2, d, dtype)
    clean = run(ctx, c)
    at = 70                      # from token 70 of the first sequence on
    for i, bad in enumerate((math.nan, math.inf, -math.inf)):
        c["v"][at + i, i % 2, 3 + i] = bad
        c["k"][at + 20 + i, 0, 5] = math.nan
    got = run(ctx, c)
    assert torch.equal(got.out[:at], clean.out[:at]) and torch.equal(got.lse[:at], clean.lse[:at])
    assert torch.equal(got.out[150:], clean.out[150:])
    agree(c, got)


def test_values_that_are_not_finite_reach_the_rows_that_see_them(ctx):
    c = case([200], 2, 1, 128, BF)
    c["v"][3, 0, 10] = math.inf
    c["v"][100, 0, 11] = -math.inf
    c["v"][199, 0, 12] = math.nan
    got = run(ctx, c)
    agree(c, got)
    assert bool((got.out[3:, :, 10] == math.inf).all()) and bool((got.out[100:, :, 11] == -math.inf).all())
    assert bool(torch.isfinite(got.out[:3]).all()) and bool(torch.isnan(got.out[199, :, 12]).all())


def test_scores_that_are_not_finite(ctx):
    c = case([100], 2, 1, 64, BF)
    c["q"][:] = c["q"].abs()
    c["k"][0:2, 0, 0] = -math.inf       # scores of -inf: tokens 0 and 1 see nothing else
    c["k"][50, 0, 1] = math.inf         # +inf: rows from 50 on are NaN
    got = run(ctx, c)
    agree(c, got)
    assert bool((got.lse[:2] == -math.inf).all()) and bool((got.out[:2] == 0).all())
    assert bool(torch.isfinite(got.out[2:50]).all()) and bool(torch.isnan(got.out[50:]).all())


@pytest.mark.parametrize("dtype,low", [(BF, -3.0e38), (BF, -1e30), (HF, -65504.0)])
def test_keys_masked_by_a_huge_value(ctx, dtype, low):
    """A key of one huge negative element, before others and after, and all of a row's."""
    c = case([160], 4, 2, 64, dtype)
    c["q"][:, :, 0] = 1.0
    c["k"][:, :, 0] = 0.0
    c["k"][:5, :, 0] = low
    c["k"][40:130, :, 0] = low
    agree(c, run(ctx, c))


def test_equal_huge_scores_weigh_alike(ctx):
    """Rows all of whose scores are one huge finite number: the mean of what they see."""
    c = case([140], 2, 1, 64, BF)
    c["q"][:], c["k"][:] = 0.0, 0.0
    c["q"][:, :, 0], c["k"][:, :, 0] = 2.0, -1.0e37
    got = run(ctx, c)
    v = c["v"].double().cpu()[:, 0]
    mean = v.cumsum(0) / torch.arange(1, 141)[:, None]
    size = v.abs().cumsum(0) / torch.arange(1, 141)[:, None]
    # each weight is 1 exactly; f32 sums, one rounding at the end (bf16's steps are 2^-7 of a
    # value from 1 to 2, so half a step 2^-8)
    off = (got.out.double().cpu() - mean[:, None]).abs()
    assert bool((off <= 2.0**-8 * mean.abs()[:, None] * 1.01 + size[:, None] * 150 * 2.0**-24).all())


@pytest.mark.parametrize("scale", [-0.2, 0.0, 3.0])
def test_scales(ctx, scale):
    c = case([100, 33], 4, 2, 64, HF)
    agree(c, run(ctx, c, scale=scale), scale=scale)


def test_values_at_the_end_of_f16(ctx):
    c = case([100], 2, 1, 64, HF)
    c["v"][:] = 65504.0
    got = run(ctx, c)
    assert bool((got.out == 65504.0).all())


def test_growing_scores_move_the_reference(ctx):
    """Every later key scores far above the ones before, tile after tile."""
    c = case([400], 2, 1, 64, BF)
    c["q"][:], c["k"][:] = 0.0, 0.0
    c["q"][:, :, 0] = 8.0
    c["k"][:, 0, 0] = torch.arange(400, device="cuda").to(BF)
    agree(c, run(ctx, c))
    c["k"][:, 0, 0] = -torch.arange(400, device="cuda").to(BF)
    agree(c, run(ctx, c))


def test_without_lse(ctx):
    c = case([50], 2, 1, 64, BF)
    want, out = run(ctx, c), blank(c)
    out.lse = None
    assert torch.equal(run(ctx, c, out=out).out, want.out)


def test_another_stream_and_a_graph(ctx):
    c = case([130, 60], 4, 2, 128, BF)
    want = run(ctx, c)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = run(ctx, c)
    s.synchronize()
    assert torch.equal(got.out, want.out)
    from xwen_amd import prompt
    out, start = blank(c), torch.tensor(c["start"], dtype=torch.int32).cuda()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        prompt.prompt_attend(ctx, c["q"], c["k"], c["v"], start, out=out)
    for i in range(3):
        out.out.zero_()
        out.lse.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.out, want.out) and torch.equal(out.lse, want.lse)
        assert torch.equal(run(ctx, c).out, want.out)
    start.copy_(torch.tensor([0, 60, 190]))  # other lengths, the same graph
    g.replay()
    torch.cuda.synchronize()
    agree({**c, "start": [0, 60, 190]}, out)


def test_refusals(ctx):
    from xwen_amd import _lib, prompt
    c = case([20], 4, 2, 64, BF)
    start = torch.tensor([0, 20], dtype=torch.int32).cuda()
    f = prompt.prompt_attend
    for q, k, v, s in ((c["q"].float(), c["k"], c["v"], start), (c["q"], c["k"].half(), c["v"], start), (c["q"], c["k"][:19], c["v"], start),
                       (c["q"], c["k"], c["v"], start.long()), (c["q"], c["k"], c["v"], start.cpu()), (c["q"], c["k"], c["v"], start[:0]),
                       (c["q"], c["k"], torch.empty((20, 2, 128), dtype=BF, device="cuda")[:, :, :64], start)):
        with pytest.raises(ValueError):
            f(ctx, q, k, v, s)
    with pytest.raises(_lib.XsError):
        f(ctx, c["q"][:, :3], c["k"], c["v"], start)  # 3 query heads for 2
    with pytest.raises(_lib.XsError):
        f(ctx, c["q"][:, :, :60].contiguous(), c["k"][:, :, :60].contiguous(), c["v"][:, :, :60].contiguous(), start)
