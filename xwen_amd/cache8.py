"""A cache of keys and values held in 8 bits, on the device: the host mirror of
xs_cache_append8 and xs_tree_attend8 (include/xsamp.h).

Elements are e4m3 (torch.float8_e4m3fn) times a power of two that BLOCK slots of a head
share, its exponent + 127 in a uint8.  Cache8 holds one layer's buffers and makes the
calls of a sequence's life: prompt() attends a prompt to itself and appends it; per step
attend() is the draft tree's attention and commit() appends the accepted path.  It takes
half of tree.TreeCache's bytes and keeps every token (nothing is evicted).  A prompt sees
nothing of the cache: one that continues a sequence is not for prompt().

Calls run on torch's current stream and are asynchronous; statuses are device tensors,
raised by tree.check().
"""
from __future__ import annotations

import ctypes as C
import math
from dataclasses import dataclass

from . import _lib
from .prompt import PromptAttended, prompt_attend
from .sampler import _torch
from .tree import Attended, CacheContext, _dtype, _kv, _need, _queries, _strides, _tensor

BLOCK = _lib.CACHE8_BLOCK


def _kv8(ctx, kv, k, v, k_exp, v_exp):
    torch = _torch()
    B, cap, H, D = k.shape
    kv.k = _tensor(ctx, k, "k", k.shape, torch.float8_e4m3fn, contiguous=False)
    kv.v = _tensor(ctx, v, "v", k.shape, torch.float8_e4m3fn, contiguous=False)
    _need(_strides(k) == _strides(v), "k and v have different strides")
    kv.seq_stride, kv.slot_stride, kv.head_stride = _strides(k)
    blocks = k_exp.shape[-1]
    _need(blocks * BLOCK >= cap, f"k_exp has {blocks} blocks for {cap} slots")
    kv.k_exp = _tensor(ctx, k_exp, "k_exp", (B, H, blocks), torch.uint8)
    kv.v_exp = _tensor(ctx, v_exp, "v_exp", (B, H, blocks), torch.uint8)
    kv.exp_ld = blocks
    return B, cap, H, D


@dataclass
class Appended:
    new_len: object     # int32 [seqs]
    seq_status: object  # int32 [seqs]


def cache_append8(ctx: CacheContext, k, v, k_exp, v_exp, length, fresh_k, fresh_v, *, start=None, path=None, n_path=None,
                  rows: int = 0, out: Appended | None = None) -> Appended:
    """One xs_cache_append8 call.  k, v float8_e4m3fn [seqs, capacity, kv_heads, head_dim]; k_exp,
    v_exp uint8 [seqs, kv_heads, capacity / BLOCK rounded up]; length int32 [seqs].  The rows are
    those of fresh_k, fresh_v, bfloat16 or float16: [seqs, rows, kv_heads, head_dim], of which
    sequence b takes path[b, :n_path[b]] (int32; path None: the first n_path[b]; both None: all);
    or, with start (int32 [seqs + 1]), a packed [tokens, kv_heads, head_dim], of which it takes
    rows start[b] to start[b + 1], at most `rows` of them (0: any number)."""
    torch = _torch()
    a = _lib.CacheAppend8Args()
    B, cap, H, D = _kv8(ctx, a.cache, k, v, k_exp, v_exp)
    a.dtype, a.head_dim, a.seqs, a.kv_heads, a.capacity = _dtype(fresh_k), D, B, H, cap
    a.len = _tensor(ctx, length, "length", (B,), torch.int32)
    if start is not None:
        _need(path is None and n_path is None, "start goes without path and n_path")
        T = fresh_k.shape[0]
        _kv(ctx, a.fresh, fresh_k.unsqueeze(0), fresh_v.unsqueeze(0), (1, T, H, D), "fresh")
        a.tokens, a.rows = T, rows or T
        a.start = _tensor(ctx, start, "start", (B + 1,), torch.int32)
    else:
        N = fresh_k.shape[1]
        _kv(ctx, a.fresh, fresh_k, fresh_v, (B, N, H, D), "fresh")
        _need(rows in (0, N), "rows goes with start")
        a.rows = a.path_ld = N
        a.path = None if path is None else _tensor(ctx, path, "path", (B, N), torch.int32)
        a.n_path = None if n_path is None else _tensor(ctx, n_path, "n_path", (B,), torch.int32)
    if out is None:
        out = Appended(*(torch.empty(B, dtype=torch.int32, device=k.device) for _ in range(2)))
    a.new_len = _tensor(ctx, out.new_len, "new_len", (B,), torch.int32)
    a.seq_status = _tensor(ctx, out.seq_status, "seq_status", (B,), torch.int32)
    ctx.bind_current_stream()
    _lib.check(ctx.lib.xs_cache_append8(ctx.h, C.byref(a)), "xs_cache_append8")
    return out


def tree_attend8(ctx: CacheContext, q, k, v, k_exp, v_exp, length, fresh_k, fresh_v, parent, *, n_nodes=None,
                 scale: float | None = None, max_len: int = 0, out: Attended | None = None) -> Attended:
    """One xs_tree_attend8 call: tree.tree_attend over the cache of cache_append8."""
    torch = _torch()
    a = _lib.TreeAttend8Args()
    _, N, HQ, D = q.shape
    B, cap, H, _ = _kv8(ctx, a.cache, k, v, k_exp, v_exp)
    a.dtype, a.head_dim, a.seqs, a.nodes, a.q_heads, a.kv_heads = _dtype(q), D, B, N, HQ, H
    _need(k.shape[3] == D, f"the cache's head size is {k.shape[3]}, not {D}")
    _queries(ctx, a, q, (B, N, HQ, D), q.dtype)
    _kv(ctx, a.fresh, fresh_k, fresh_v, (B, N, H, D), "fresh")
    _need(fresh_k.dtype == q.dtype, "q and the fresh keys differ in type")
    a.capacity, a.max_len = cap, max_len
    a.len = _tensor(ctx, length, "length", (B,), torch.int32)
    a.parent = _tensor(ctx, parent, "parent", (B, N), torch.int32)
    a.n_nodes = None if n_nodes is None else _tensor(ctx, n_nodes, "n_nodes", (B,), torch.int32)
    a.scale = 1.0 / math.sqrt(D) if scale is None else scale
    if out is None:
        out = Attended(out=torch.empty((B, N, HQ, D), dtype=q.dtype, device=q.device),
                       lse=torch.empty((B, N, HQ), dtype=torch.float32, device=q.device),
                       seq_status=torch.empty(B, dtype=torch.int32, device=q.device))
    a.out = _tensor(ctx, out.out, "out", (B, N, HQ, D), q.dtype, contiguous=False)
    a.out_seq_stride, a.out_node_stride, a.out_head_stride = _strides(out.out)
    a.lse = None if out.lse is None else _tensor(ctx, out.lse, "lse", (B, N, HQ), torch.float32)
    a.seq_status = _tensor(ctx, out.seq_status, "seq_status", (B,), torch.int32)
    ctx.bind_current_stream()
    _lib.check(ctx.lib.xs_tree_attend8(ctx.h, C.byref(a)), "xs_tree_attend8")
    return out


class Cache8:
    """One layer's cache of committed tokens in 8 bits, of `capacity` slots a sequence."""

    def __init__(self, ctx: CacheContext, seqs: int, kv_heads: int, head_dim: int, capacity: int):
        torch = _torch()
        dev = torch.device("cuda", ctx.device)
        blocks = (capacity + BLOCK - 1) // BLOCK
        self.ctx = ctx
        self.k, self.v = (torch.zeros((seqs, capacity, kv_heads, head_dim), dtype=torch.float8_e4m3fn, device=dev) for _ in range(2))
        self.k_exp, self.v_exp = (torch.zeros((seqs, kv_heads, blocks), dtype=torch.uint8, device=dev) for _ in range(2))
        self.length, self._length = (torch.zeros(seqs, dtype=torch.int32, device=dev) for _ in range(2))
        self.append_status = torch.zeros(seqs, dtype=torch.int32, device=dev)

    def _append(self, fresh_k, fresh_v, **kw) -> None:
        cache_append8(self.ctx, self.k, self.v, self.k_exp, self.v_exp, self.length, fresh_k, fresh_v,
                      out=Appended(self._length, self.append_status), **kw)
        # the next call reads what this one wrote, in stream order (copied in
        # place, so that a captured step finds the same buffers when replayed)
        self.length.copy_(self._length)

    def prompt(self, q, k, v, start, *, scale: float | None = None, max_len: int = 0,
               out: PromptAttended | None = None) -> PromptAttended:
        """Prompts packed as prompt_attend takes them: their attention, each to itself (in 16
        bits), and their keys and values appended.  What a sequence's cache holds already is not
        attended to: a second turn, a shared prefix or a part of a prompt after the first gets
        the attention of a text of its own.  max_len: a bound on the prompts' lengths (0: none; it
        sizes the append's launch, and a longer prompt is attended but not appended:
        append_status)."""
        a = prompt_attend(self.ctx, q, k, v, start, scale=scale, out=out)
        self._append(k, v, start=start, rows=max_len)
        return a

    def attend(self, q, fresh_k, fresh_v, parent, **kw) -> Attended:
        return tree_attend8(self.ctx, q, self.k, self.v, self.k_exp, self.v_exp, self.length, fresh_k, fresh_v, parent, **kw)

    def commit(self, fresh_k, fresh_v, path, n_path) -> None:
        """The accepted path of a step, as a TreeVerdict gives it."""
        self._append(fresh_k, fresh_v, path=path, n_path=n_path)
