"""xs_qk_rotate of one side, through the C ABI: the weight of a side without heads says nothing."""
import ctypes as C

import pytest
import torch

from tests import promptref
from tests.test_gpu_rotate import case, ctx  # noqa: F401 (a fixture)
from xwen_amd import _lib

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("side", ["q", "k"])
@pytest.mark.parametrize("own,other", [(False, True), (True, False), (True, True), (False, False)])
def test_the_other_sides_weight(ctx, side, own, other):  # noqa: F811
    c = case(30, 4, 4, 64, torch.bfloat16, 32)
    x, w = c["q"], c["w"][0]
    y = torch.full_like(x, 7.0)
    a = _lib.QkRotateArgs(dtype=_lib.BF16, head_dim=64, tokens=30, eps=1e-6, rot_dim=32, pairs=_lib.ROT_HALVES, pos=c["pos"].data_ptr(),
                          inv_freq=c["inv_freq"].data_ptr())
    setattr(a, "q_heads" if side == "q" else "kv_heads", 4)
    for name, t in ((side, x), (side + "_out", y)):
        setattr(a, name, t.data_ptr())
        setattr(a, name + "_token_stride", t.stride(0))
        setattr(a, name + "_head_stride", t.stride(1))
    if own:
        setattr(a, side + "_weight", w.data_ptr())
    if other:
        setattr(a, ("k" if side == "q" else "q") + "_weight", c["w"][1].data_ptr())
    ctx.bind_current_stream()
    assert ctx.lib.xs_qk_rotate(ctx.h, C.byref(a)) == _lib.XS_OK
    want, tol = promptref.rotate(x, w if own else None, 1e-6, c["pos"], c["inv_freq"], False)
    assert bool(((y.double().cpu() - want).abs() <= tol).all())
