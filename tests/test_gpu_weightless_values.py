"""Values that are not finite reach the rows that give them weight and no others: tokens masked by a
score of -inf or of a type's end, whose values hold infinities and NaN, in xs_prompt_attend,
against the definition in 64 bits."""
import math

import numpy as np
import pytest
import torch

from tests.treeref import F32, half_step

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
INF = math.inf


@pytest.fixture(scope="module")
def ctx():
    from xwen_amd import tree
    return tree.CacheContext(max_seqs=1, max_nodes=1, q_heads=1, kv_heads=1, head_dim=8, capacity=1)


def definition(q, k, v, seen, scale):
    """(out, lse, out tolerance, lse tolerance), f64, of one head's rows q [rows, size] over k, v [keys,
    size], seen [rows, keys].  An element is what the finite values give, and infinite or NaN by the
    values that have weight.  The tolerances are treeref.attend's."""
    dtype = q.dtype
    q, k, v = q.double(), k.double(), v.double()
    D = q.shape[1]
    s = torch.where(seen, q @ k.T.contiguous() * scale, -INF)
    empty = (s == -INF).all(-1, keepdim=True)
    p = torch.where(empty, 0.0, s.softmax(-1))
    lse = s.logsumexp(-1, keepdim=True)
    fine = torch.where(torch.isfinite(v), v, 0.0)
    weight = (p > 0).double()
    plus, minus = (weight @ ((v == x) | v.isnan()).double() > 0 for x in (INF, -INF))
    y = p @ fine
    out = torch.where(plus & minus, math.nan, torch.where(plus, INF, torch.where(minus, -INF, y)))
    size = torch.where(p > 0, q.abs() @ k.abs().nan_to_num(0, 0, 0).T.contiguous(), 0.0).amax(-1, keepdim=True) * abs(scale)
    off = (D + 4) * F32 * size + 8 * F32 * (1 + torch.where(p > 0, s, 0.0).abs().amax(-1, keepdim=True))
    n = k.shape[0]
    u = half_step(dtype)
    tol = u * y.abs() * 1.01 + p @ fine.abs() * (u * 1.01 + 2 * off + 2 * (n + 8) * F32)
    if dtype == HF:  # the least half step of float16, where it stops being relative
        tol = tol + 2.0**-25 * (1 + n)
    return out, lse[:, 0], tol, (off + (n + 8) * F32 + 4 * F32 * lse.abs())[:, 0]


def agree(got_out, got_lse, want, where):
    out, lse, tol, ltol = want
    x, s = got_out.double(), got_lse.double()
    assert bool((s[lse == -INF] == -INF).all()) and bool((x[lse == -INF] == 0).all()), where
    same = (x == out) | (x.isnan() & out.isnan())
    fine = torch.isfinite(out)
    assert bool(same[~fine].all()), (where, (~same & ~fine).nonzero()[:5].tolist(), x[~same & ~fine][:5])
    assert bool(((x - out).abs() <= tol)[fine].all()), (where, ((x - out).abs() > tol).nonzero()[:5].tolist())
    fine = torch.isfinite(lse)
    assert bool(((s - lse).abs() <= ltol)[fine].all()), where


def spoil(v, at, g):
    """Infinities of both signs and NaN in the values [tokens, heads, size] of the tokens at."""
    D = v.shape[-1]
    for i, t in enumerate(at):
        for j, bad in enumerate((INF, -INF, math.nan)):
            v[t, :, int(torch.randint(0, D, (1,), generator=g))] = bad
        v[t, :, (3 * i) % D] = (INF, -INF)[i % 2]


LOWS = [(BF, -INF), (BF, -3.0e38), (HF, -INF), (HF, -65504.0)]


@pytest.mark.parametrize("dtype,low", LOWS)
@pytest.mark.parametrize("d,hq,h", [(40, 4, 2), (64, 4, 2), (64, 64, 1), (96, 3, 3), (128, 4, 2), (128, 64, 1), (256, 8, 2)])
def test_prompts(ctx, d, hq, h, dtype, low):
    """Masked tokens first, in the middle, and last of a sequence; some infinite values that count; 64
    query heads: tiles of 128 rows."""
    from xwen_amd import prompt
    g = torch.Generator().manual_seed(d + hq)
    lens = [700, 3, 0, 330]
    start = np.concatenate([[0], np.cumsum(lens)]).tolist()
    q, k, v = (torch.randn((start[-1], n, d), generator=g) for n in (hq, h, h))
    q[..., 0], k[..., 0] = 1.0, 0.0
    masked = torch.zeros(start[-1], dtype=torch.bool)
    for i in (0, 1, 2, 64, 65, 130, 200, 201, 333, 500, 640, 699, 700, 703, 710, 800, 900, 1000, 1032):
        masked[i] = True
    k[masked, :, 0] = low
    spoil(v, masked.nonzero()[:, 0].tolist(), g)
    v[400, :, 7], v[555, :, 9], v[950, :, 11] = INF, math.nan, -INF  # these have weight
    q, k, v = (t.to(dtype).cuda() for t in (q, k, v))
    got = prompt.prompt_attend(ctx, q, k, v, torch.tensor(start, dtype=torch.int32).cuda())
    scale = float(np.float32(1 / math.sqrt(d)))
    for i, j in zip(start, start[1:]):
        if i == j:
            continue
        seen = torch.ones((j - i, j - i), dtype=torch.bool, device="cuda").tril()
        for n in range(0, hq, max(1, hq // 4)):
            agree(got.out[i:j, n], got.lse[i:j, n], definition(q[i:j, n], k[i:j, n // (hq // h)], v[i:j, n // (hq // h)], seen, scale), (i, n))


@pytest.mark.parametrize("dtype", [BF, HF])
def test_a_light_weight_is_one(ctx, dtype):
    """A token of 2^-25 of the row's largest weight still carries its infinity, before and after it."""
    from xwen_amd import prompt
    q, k, v = (torch.zeros((200, 1, 64), dtype=dtype, device="cuda") for _ in "qkv")
    q[..., 0] = 8.0
    k[100, 0, 0] = 17.0  # a score of 17, where the others' are 0
    v[10, 0, 3], v[150, 0, 4] = INF, -INF
    got = prompt.prompt_attend(ctx, q, k, v, torch.tensor([0, 200], dtype=torch.int32).cuda())
    assert bool((got.out[10:, 0, 3] == INF).all()) and bool((got.out[150:, 0, 4] == -INF).all())
    assert bool((got.out[:10, 0, 3] == 0).all()) and bool((got.out[:150, 0, 4] == 0).all())
