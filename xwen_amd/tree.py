"""A speculative step over a bounded cache, on the device: the host mirror of
xs_tree_attend, xs_cache_commit and xs_cache_evict (include/xsamp.h).

The drafts of a step are a tree of tokens (up to TREE_MAX nodes a sequence, node
0 the last committed token).  Per layer its nodes attend to the cache and to
their own ancestors (tree_attend); sampler.verify_tree_batch then samples every
node and walks down the tree; the accepted path is appended to each layer's cache
(cache_commit), with the attention weight it gave to every slot, and a cache over
its budget keeps the slots with the most (cache_evict).  TreeCache holds one
layer's buffers and makes the calls in that order.

No counterpart in the reference, which verifies one chain of drafts over a cache
of every token (src/generate.rs:2410-2461).  Calls run on torch's current stream
and are asynchronous; statuses are device tensors, raised by check().
"""
from __future__ import annotations

import ctypes as C
import math
from dataclasses import dataclass

from . import _lib
from .sampler import SampleError, _torch

TREE_MAX = _lib.TREE_MAX


class CacheContext:
    """An xs_cache_context: the workspace of the cache calls, sized for the
    largest of each dimension."""

    def __init__(self, *, max_seqs: int, max_nodes: int, q_heads: int, kv_heads: int, head_dim: int, capacity: int,
                 device: int = 0):
        self.lib = _lib.load()
        self.device = device
        self.h = None
        _torch().cuda.init()
        dims = _lib.CacheDims(max_seqs, max_nodes, q_heads, kv_heads, head_dim, capacity)
        h = C.c_void_p()
        _lib.check(self.lib.xs_cache_create(device, C.byref(dims), C.byref(h)), "xs_cache_create")
        self.h = h
        self._bound = None  # the stream's handle, and whether it recorded into a graph
        self._last = {False: None, True: None}  # the stream of the last call outside a graph, and in one

    def bind_stream(self, stream):
        """The stream of the calls from here on.  Their workspace is the context's: the new
        stream waits for the last call's, also where both are forks of one stream under capture.
        A capture does not wait for work outside it (torch.cuda.graph has the device run dry
        first), nor does that for a capture; replays, and calls beside them, are the caller's to
        keep apart."""
        inside = _capturing(stream)
        if self._bound == (stream.cuda_stream, inside):
            return
        last = self._last[inside]
        if last is not None and last.cuda_stream != stream.cuda_stream and (not inside or _capturing(last)):
            stream.wait_stream(last)
        _lib.check(self.lib.xs_cache_set_stream(self.h, C.c_void_p(stream.cuda_stream)), "xs_cache_set_stream")
        self._bound, self._last[inside] = (stream.cuda_stream, inside), stream

    def bind_current_stream(self):
        self.bind_stream(_torch().cuda.current_stream(self.device))

    def close(self):
        if getattr(self, "h", None):
            self.lib.xs_cache_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def _capturing(stream) -> bool:
    """Whether the stream records into a graph (the null stream never does)."""
    cuda = _torch().cuda
    if stream.cuda_stream == 0:
        return False
    if stream == cuda.current_stream():
        return cuda.is_current_stream_capturing()
    with cuda.stream(stream):
        return cuda.is_current_stream_capturing()


def check(seq_status) -> None:
    """Raise SampleError if any sequence of a call failed (waits for the call)."""
    st = seq_status.cpu().numpy()
    if st.any():
        raise SampleError(st)


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _tensor(ctx, t, name, shape, dtype, contiguous=True):
    _need(t.is_cuda and t.device.index == ctx.device, f"{name} is not on the context's device")
    _need(t.dtype == dtype, f"{name} is {t.dtype}, not {dtype}")
    _need(tuple(t.shape) == tuple(shape), f"{name} is {tuple(t.shape)}, not {tuple(shape)}")
    _need(t.is_contiguous() if contiguous else (t.numel() == 0 or t.stride(-1) == 1),
          f"{name} is not contiguous" + ("" if contiguous else " in its last dimension"))
    return t.data_ptr()


def _dtype(t):
    torch = _torch()
    kinds = {torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
    _need(t.dtype in kinds, f"keys, values and queries are bfloat16 or float16, not {t.dtype}")
    return kinds[t.dtype]


def _kv(ctx, kv, k, v, shape, name):
    kv.k = _tensor(ctx, k, name + "_k", shape, k.dtype, contiguous=False)
    kv.v = _tensor(ctx, v, name + "_v", shape, k.dtype, contiguous=False)
    _need(_strides(k) == _strides(v), f"{name}_k and {name}_v have different strides")
    kv.seq_stride, kv.slot_stride, kv.head_stride = _strides(k)


def _strides(t):
    """The first three strides; that of a dimension of one entry says nothing."""
    return [s if n > 1 else 0 for n, s in zip(t.shape[:3], t.stride()[:3])]


def _queries(ctx, a, q, shape, dtype):
    a.q = _tensor(ctx, q, "q", shape, dtype, contiguous=False)
    a.q_seq_stride, a.q_node_stride, a.q_head_stride = _strides(q)


@dataclass
class Attended:
    out: object         # [seqs, nodes, q_heads, head_dim]
    lse: object         # float32 [seqs, nodes, q_heads]
    seq_status: object  # int32 [seqs]


def tree_attend(ctx: CacheContext, q, cache_k, cache_v, length, fresh_k, fresh_v, parent, *, n_nodes=None,
                scale: float | None = None, max_len: int = 0, out: Attended | None = None) -> Attended:
    """One xs_tree_attend call.  q [seqs, nodes, q_heads, head_dim]; cache_k, cache_v
    [seqs, capacity, kv_heads, head_dim] and fresh_k, fresh_v [seqs, nodes, kv_heads,
    head_dim], bfloat16 or float16, any strides but 1 in the last dimension; length int32
    [seqs] the slots in use; parent int32 [seqs, nodes]; n_nodes int32 [seqs] or None;
    max_len a bound on every length (0: the capacity).  Rows past n_nodes of `out` are
    left as they were (unset in a new one)."""
    torch = _torch()
    B, N, HQ, D = q.shape
    cap, H = cache_k.shape[1:3]
    a = _lib.TreeAttendArgs()
    a.dtype, a.head_dim, a.seqs, a.nodes, a.q_heads, a.kv_heads = _dtype(q), D, B, N, HQ, H
    _queries(ctx, a, q, (B, N, HQ, D), q.dtype)
    _kv(ctx, a.cache, cache_k, cache_v, (B, cap, H, D), "cache")
    _kv(ctx, a.fresh, fresh_k, fresh_v, (B, N, H, D), "fresh")
    _need(cache_k.dtype == q.dtype and fresh_k.dtype == q.dtype, "q, the cache and the fresh keys differ in type")
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
    _lib.check(ctx.lib.xs_tree_attend(ctx.h, C.byref(a)), "xs_tree_attend")
    return out


@dataclass
class Committed:
    new_len: object        # int32 [seqs]
    new_next_pos: object   # int32 [seqs], or None
    seq_status: object     # int32 [seqs]


def cache_commit(ctx: CacheContext, cache_k, cache_v, length, fresh_k, fresh_v, path, n_path, *, pos=None, next_pos=None,
                 q=None, lse=None, scale: float | None = None, mass=None, new_mass=None, max_len: int = 0,
                 out: Committed | None = None) -> Committed:
    """One xs_cache_commit call: the cache takes the nodes path[:, :n_path] (int32 [seqs,
    nodes] and [seqs], a TreeVerdict's path and n_committed).  With pos (int32 [seqs, kv_heads,
    capacity]) and next_pos (int32 [seqs]) it keeps the slots' positions; with q and lse of the
    layer's tree_attend and mass (float32 [seqs, kv_heads, capacity]) it adds up the attention
    weight, into new_mass (None: into mass itself)."""
    torch = _torch()
    B, cap, H, D = cache_k.shape
    N = fresh_k.shape[1]
    a = _lib.CacheCommitArgs()
    a.dtype, a.head_dim, a.seqs, a.nodes, a.kv_heads, a.q_heads = _dtype(cache_k), D, B, N, H, H
    _kv(ctx, a.cache, cache_k, cache_v, (B, cap, H, D), "cache")
    _kv(ctx, a.fresh, fresh_k, fresh_v, (B, N, H, D), "fresh")
    _need(cache_k.dtype == fresh_k.dtype, "the cache and the fresh keys differ in type")
    a.capacity, a.max_len, a.slot_ld, a.path_ld = cap, max_len, cap, N
    a.len = _tensor(ctx, length, "length", (B,), torch.int32)
    a.path = _tensor(ctx, path, "path", (B, N), torch.int32)
    a.n_path = _tensor(ctx, n_path, "n_path", (B,), torch.int32)
    _need((pos is None) == (next_pos is None), "pos and next_pos go together")
    if out is None:
        out = Committed(*(torch.empty(B, dtype=torch.int32, device=cache_k.device) for _ in range(3)))
    a.new_len = _tensor(ctx, out.new_len, "new_len", (B,), torch.int32)
    a.seq_status = _tensor(ctx, out.seq_status, "seq_status", (B,), torch.int32)
    if pos is not None:
        a.pos = _tensor(ctx, pos, "pos", (B, H, cap), torch.int32)
        a.next_pos = _tensor(ctx, next_pos, "next_pos", (B,), torch.int32)
        a.new_next_pos = _tensor(ctx, out.new_next_pos, "new_next_pos", (B,), torch.int32)
    else:
        out.new_next_pos = None
    _need((mass is None) == (q is None) and (mass is None) == (lse is None), "q, lse and mass go together")
    if mass is not None:
        a.q_heads = q.shape[2]
        _queries(ctx, a, q, (B, N, a.q_heads, D), cache_k.dtype)
        a.lse = _tensor(ctx, lse, "lse", (B, N, a.q_heads), torch.float32)
        a.scale = 1.0 / math.sqrt(D) if scale is None else scale
        a.mass = _tensor(ctx, mass, "mass", (B, H, cap), torch.float32)
        a.new_mass = a.mass if new_mass is None else _tensor(ctx, new_mass, "new_mass", (B, H, cap), torch.float32)
    ctx.bind_current_stream()
    _lib.check(ctx.lib.xs_cache_commit(ctx.h, C.byref(a)), "xs_cache_commit")
    return out


@dataclass
class Evicted:
    new_len: object     # int32 [seqs]
    seq_status: object  # int32 [seqs]


def cache_evict(ctx: CacheContext, cache_k, cache_v, length, mass, pos, next_pos, keep: int, *, sinks: int = 0,
                recent: int = 0, new_mass=None, new_pos=None, max_len: int = 0, out: Evicted | None = None) -> Evicted:
    """One xs_cache_evict call: every sequence of more than `keep` slots keeps, per kv head,
    the slots of its first `sinks` and last `recent` positions and those with the most mass.
    mass, pos, next_pos as in cache_commit; new_mass and new_pos None: in place."""
    torch = _torch()
    B, cap, H, D = cache_k.shape
    a = _lib.CacheEvictArgs()
    a.dtype, a.head_dim, a.seqs, a.kv_heads = _dtype(cache_k), D, B, H
    _kv(ctx, a.cache, cache_k, cache_v, (B, cap, H, D), "cache")
    a.capacity, a.max_len, a.slot_ld = cap, max_len, cap
    a.len = _tensor(ctx, length, "length", (B,), torch.int32)
    a.mass = _tensor(ctx, mass, "mass", (B, H, cap), torch.float32)
    a.pos = _tensor(ctx, pos, "pos", (B, H, cap), torch.int32)
    a.new_mass = a.mass if new_mass is None else _tensor(ctx, new_mass, "new_mass", (B, H, cap), torch.float32)
    a.new_pos = a.pos if new_pos is None else _tensor(ctx, new_pos, "new_pos", (B, H, cap), torch.int32)
    a.next_pos = _tensor(ctx, next_pos, "next_pos", (B,), torch.int32)
    a.keep, a.sinks, a.recent = keep, sinks, recent
    if out is None:
        out = Evicted(*(torch.empty(B, dtype=torch.int32, device=cache_k.device) for _ in range(2)))
    a.new_len = _tensor(ctx, out.new_len, "new_len", (B,), torch.int32)
    a.seq_status = _tensor(ctx, out.seq_status, "seq_status", (B,), torch.int32)
    ctx.bind_current_stream()
    _lib.check(ctx.lib.xs_cache_evict(ctx.h, C.byref(a)), "xs_cache_evict")
    return out


class TreeCache:
    """One layer's cache of committed tokens and what the calls keep beside it.
    `keep` slots a kv head is its budget; it has room for `keep` plus TREE_MAX
    (or `capacity`) slots, so that evict() after every commit() never runs out."""

    def __init__(self, ctx: CacheContext, seqs: int, kv_heads: int, head_dim: int, keep: int, *, dtype, sinks: int = 4,
                 recent: int = 64, capacity: int = 0):
        torch = _torch()
        cap = capacity or keep + TREE_MAX
        dev = torch.device("cuda", ctx.device)
        self.ctx, self.keep, self.sinks, self.recent = ctx, keep, sinks, recent
        self.k, self.v = (torch.zeros((seqs, cap, kv_heads, head_dim), dtype=dtype, device=dev) for _ in range(2))
        self.mass = torch.zeros((seqs, kv_heads, cap), dtype=torch.float32, device=dev)
        self.pos = torch.zeros((seqs, kv_heads, cap), dtype=torch.int32, device=dev)
        self.length, self._length = (torch.zeros(seqs, dtype=torch.int32, device=dev) for _ in range(2))
        self.next_pos, self._next_pos = (torch.zeros(seqs, dtype=torch.int32, device=dev) for _ in range(2))
        self.commit_status, self.evict_status = (torch.zeros(seqs, dtype=torch.int32, device=dev) for _ in range(2))

    def attend(self, q, fresh_k, fresh_v, parent, **kw) -> Attended:
        return tree_attend(self.ctx, q, self.k, self.v, self.length, fresh_k, fresh_v, parent, **kw)

    def commit(self, q, lse, fresh_k, fresh_v, path, n_path, *, scale: float | None = None) -> None:
        """The accepted path of a step whose attend() took q, fresh_k and fresh_v and gave lse."""
        cache_commit(self.ctx, self.k, self.v, self.length, fresh_k, fresh_v, path, n_path, pos=self.pos,
                     next_pos=self.next_pos, q=q, lse=lse, scale=scale, mass=self.mass,
                     out=Committed(self._length, self._next_pos, self.commit_status))
        # the next call reads what this one wrote, in stream order (copied in
        # place, so that a captured step finds the same buffers when replayed)
        self.length.copy_(self._length)
        self.next_pos.copy_(self._next_pos)

    def evict(self) -> None:
        """Back to the budget."""
        cache_evict(self.ctx, self.k, self.v, self.length, self.mass, self.pos, self.next_pos, self.keep,
                    sinks=self.sinks, recent=self.recent, out=Evicted(self._length, self.evict_status))
        self.length.copy_(self._length)
