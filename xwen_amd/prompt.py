"""A prompt's way to its attention, on the device: the host mirror of xs_qk_rotate and
xs_prompt_attend (include/xsamp.h).

A layer's projections give queries and keys; qk_rotate norms them per head and turns
them by their positions (of a prompt's tokens, or of a tree's nodes), prompt_attend is
the causal attention of whole prompts, packed one after the other.  What a cache stores
is qk_rotate's keys: cache8.Cache8.prompt appends them.

No counterpart among the reference's calls that this library replaces: its model's
forward does both (src/model.rs).  Calls run on torch's current stream and are
asynchronous; statuses are device tensors, raised by tree.check().
"""
from __future__ import annotations

import ctypes as C
import math
from dataclasses import dataclass

from . import _lib
from .sampler import _torch
from .tree import CacheContext, _dtype, _need, _tensor


def frequencies(rot_dim: int, base: float, device):
    """float32 [rot_dim / 2]: base ** (-2 i / rot_dim), qk_rotate's inv_freq."""
    torch = _torch()
    return (float(base) ** (-torch.arange(0, rot_dim, 2, dtype=torch.float64) / max(rot_dim, 1))).float().to(device)


def _two_strides(t):
    return [s if n > 1 else 0 for n, s in zip(t.shape[:2], t.stride()[:2])]


def _heads(ctx, a, name, t, shape, dtype):
    setattr(a, name, _tensor(ctx, t, name, shape, dtype, contiguous=False))
    ts, hs = _two_strides(t)
    setattr(a, name + "_token_stride", ts)
    setattr(a, name + "_head_stride", hs)


def qk_rotate(ctx: CacheContext, q, k, pos=None, *, inv_freq=None, neighbours: bool = False, q_weight=None, k_weight=None,
              eps: float = 1e-6, q_out=None, k_out=None):
    """One xs_qk_rotate call: (q_out, k_out).  q [tokens, q_heads, head_dim] and k [tokens,
    kv_heads, head_dim], bfloat16 or float16, any strides but 1 in the last dimension (a packed
    projection's slices); either may be None.  pos int32 [tokens] and inv_freq float32 [rot_dim
    / 2]: the first rot_dim elements of a head turn, as halves or as neighbours (None: no
    rotation).  q_weight, k_weight float32 [head_dim] (None: no norm).  q_out, k_out None: new
    tensors; q and k themselves: in place."""
    torch = _torch()
    some = q if q is not None else k
    _need(some is not None, "q and k are both None")
    T, _, D = some.shape
    a = _lib.QkRotateArgs()
    a.dtype, a.head_dim, a.tokens, a.eps = _dtype(some), D, T, eps
    a.pairs = _lib.ROT_NEIGHBOURS if neighbours else _lib.ROT_HALVES
    _need((pos is None) == (inv_freq is None), "pos and inv_freq go together")
    if pos is not None:
        a.rot_dim = 2 * inv_freq.numel()
        a.inv_freq = _tensor(ctx, inv_freq, "inv_freq", (inv_freq.numel(),), torch.float32)
        a.pos = _tensor(ctx, pos, "pos", (T,), torch.int32)
    if q is not None and k is not None:
        _need((q_weight is None) == (k_weight is None), "q_weight and k_weight go together")
    outs = []
    for name, heads, t, w, y in (("q", "q_heads", q, q_weight, q_out), ("k", "kv_heads", k, k_weight, k_out)):
        if t is None:
            outs.append(None)
            continue
        H = t.shape[1]
        setattr(a, heads, H)
        _heads(ctx, a, name, t, (T, H, D), some.dtype)
        if w is not None:
            setattr(a, name + "_weight", _tensor(ctx, w, name + "_weight", (D,), torch.float32))
        y = torch.empty((T, H, D), dtype=t.dtype, device=t.device) if y is None else y
        _heads(ctx, a, name + "_out", y, (T, H, D), some.dtype)
        outs.append(y)
    ctx.bind_current_stream()
    _lib.check(ctx.lib.xs_qk_rotate(ctx.h, C.byref(a)), "xs_qk_rotate")
    return tuple(outs)


@dataclass
class PromptAttended:
    out: object         # [tokens, q_heads, head_dim]
    lse: object         # float32 [tokens, q_heads], or None
    seq_status: object  # int32 [seqs]


def prompt_attend(ctx: CacheContext, q, k, v, start, *, scale: float | None = None,
                  out: PromptAttended | None = None) -> PromptAttended:
    """One xs_prompt_attend call.  q [tokens, q_heads, head_dim]; k, v [tokens, kv_heads,
    head_dim], bfloat16 or float16, any strides but 1 in the last dimension; start int32
    [seqs + 1]: sequence b's tokens are rows start[b] to start[b + 1].  Rows of no sequence of
    `out` are left as they were (unset in a new one)."""
    torch = _torch()
    T, HQ, D = q.shape
    H, B = k.shape[1], start.shape[0] - 1
    _need(B >= 0, "start is empty")
    a = _lib.PromptAttendArgs()
    a.dtype, a.head_dim, a.seqs, a.tokens, a.q_heads, a.kv_heads = _dtype(q), D, B, T, HQ, H
    _heads(ctx, a, "q", q, (T, HQ, D), q.dtype)
    a.k = _tensor(ctx, k, "k", (T, H, D), q.dtype, contiguous=False)
    a.v = _tensor(ctx, v, "v", (T, H, D), q.dtype, contiguous=False)
    _need(_two_strides(k) == _two_strides(v), "k and v have different strides")
    a.kv_token_stride, a.kv_head_stride = _two_strides(k)
    a.start = _tensor(ctx, start, "start", (B + 1,), torch.int32)
    a.scale = 1.0 / math.sqrt(D) if scale is None else scale
    if out is None:
        out = PromptAttended(out=torch.empty((T, HQ, D), dtype=q.dtype, device=q.device),
                             lse=torch.empty((T, HQ), dtype=torch.float32, device=q.device),
                             seq_status=torch.empty(B, dtype=torch.int32, device=q.device))
    _heads(ctx, a, "out", out.out, (T, HQ, D), q.dtype)
    a.lse = None if out.lse is None else _tensor(ctx, out.lse, "lse", (T, HQ), torch.float32)
    a.seq_status = _tensor(ctx, out.seq_status, "seq_status", (B,), torch.int32)
    ctx.bind_current_stream()
    _lib.check(ctx.lib.xs_prompt_attend(ctx.h, C.byref(a)), "xs_prompt_attend")
    return out
