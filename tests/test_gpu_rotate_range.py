"""xs_qk_rotate's norm where the squares of a head's elements pass f32's range, either way."""
import math

import pytest
import torch

from tests import promptref
from tests.test_gpu_rotate import ctx  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def normed(ctx, x, eps, w, rot=16):  # noqa: F811
    from xwen_amd import prompt
    pos = torch.arange(x.shape[0], dtype=torch.int32).cuda()
    freq = prompt.frequencies(rot, 1e4, "cuda")
    y, _ = prompt.qk_rotate(ctx, x, None, pos, inv_freq=freq, q_weight=w, eps=eps)
    want, tol = promptref.rotate(x, w, eps, pos, freq, False)
    return y, want, tol


@pytest.mark.parametrize("d", [16, 80, 256])
@pytest.mark.parametrize("power", [127, 100, 70, 64, 62, 59, 40, 0, -30, -39, -41, -62, -70, -100, -118])
def test_elements_of_any_size(ctx, power, d):  # noqa: F811
    """Heads of elements about 2^power (1/2 to 1 of it), one of them a lone large one."""
    g = torch.Generator().manual_seed(d + power)
    x = (torch.rand((9, 3, d), generator=g) / 2 + 0.5) * (torch.randint(0, 2, (9, 3, d), generator=g) * 2 - 1)
    x[4] *= 2.0**-8
    x[4, :, 3] *= 2.0**8
    x = (x * 2.0**power).to(BF).cuda()
    w = (1 + 0.3 * torch.randn(d, generator=g)).cuda()
    for eps in (0.0, 1e-6):
        y, want, tol = normed(ctx, x, eps, w)
        off = ((y.double().cpu() - want).abs() / tol).max()
        assert float(off) <= 1.0, (eps, float(off))


def test_subnormal_elements_and_small_eps(ctx):  # noqa: F811
    g = torch.Generator().manual_seed(3)
    x = (torch.randint(1, 60, (9, 2, 64), generator=g) * 2.0**-133).to(BF).cuda()
    w = torch.ones(64, device="cuda")
    for eps in (0.0, 2.0**-140, 2.0**-126, 2.0**-100):
        y, want, tol = normed(ctx, x, eps, w)
        assert bool(((y.double().cpu() - want).abs() <= tol).all()), eps


def test_ends_of_the_types(ctx):  # noqa: F811
    """A head of a type's largest, and one element of it beside zeros: +-1 and the root of size."""
    for dtype in (BF, HF):
        x = torch.zeros((2, 1, 64), dtype=dtype, device="cuda")
        x[0, 0] = torch.finfo(dtype).max
        x[1, 0, 5] = torch.finfo(dtype).min
        y, _, _ = normed(ctx, x, 0.0, torch.ones(64, device="cuda"), rot=0)
        assert bool((y[0] == 1).all()) and float(y[1, 0, 5]) == -8.0 and float(y[1].abs().sum()) == 8.0


def test_heads_beside_one_another(ctx):  # noqa: F811
    """Small, large and infinite heads of one wave leave the others' bits as they are."""
    g = torch.Generator().manual_seed(5)
    x = torch.randn((16, 4, 64), generator=g).to(BF).cuda()
    w = (1 + 0.3 * torch.randn(64, generator=g)).cuda()
    clean = normed(ctx, x, 1e-6, w)[0]
    x[3, 1] = 2.0**100
    x[5, 2, 7] = math.inf
    x[7, 0] = 2.0**-120
    y = normed(ctx, x, 1e-6, w)[0]
    keep = torch.ones((16, 4), dtype=torch.bool)
    keep[3, 1] = keep[5, 2] = keep[7, 0] = False
    assert torch.equal(y[keep.cuda()], clean[keep.cuda()])
    assert not bool(torch.isfinite(y[5, 2]).all()) and bool(torch.isfinite(y[3, 1]).all())
