"""A speculative step over a bounded cache: the operators whose speed is watched.

A model that drafts a tree of tokens runs, per layer, attention of the tree's
nodes over the cache ("attend"); the head's logits then go through the tree's
verification ("verify"); the accepted path is appended to each layer's cache and
its attention weight added to the slots' totals ("commit"); a cache over its
budget drops the slots with the least weight ("evict").  A case is one call of
one of them, through the C ABI of include/xsamp.h, with the argument struct, the
context and the buffers that an engine keeps between steps.

Vocabulary 248,320 and the sampling options are the configurations that bench.py
and the tests name; the other sizes are generic.  With `own` false, run()
computes the same in elementary torch operations.
"""
from __future__ import annotations

import ctypes as C
import math

import numpy as np
import torch

own = False

V = 248_320
TREE_MAX = 64

DEFAULTS = dict(kind="attend", seqs=1, nodes=1, q_heads=32, kv_heads=8, dim=128, dtype="bf16", len=128, ragged=False,
                layout="slot", path=1, keep=0, sinks=4, recent=0, vocab=V, temperature=1.0, top_k=20, top_p=0.95)


def listed() -> list[dict]:
    return [
        # The smallest call: one new token of one user over a short context.
        dict(name="attend_one", seqs=1, nodes=1, q_heads=16, kv_heads=2, dim=256, len=100),
        # An odd model and odd lengths: 3 users, 7 nodes, head size 80, float16.
        dict(name="attend_odd", seqs=3, nodes=7, q_heads=12, kv_heads=4, dim=80, dtype="f16", len=1777, ragged=True,
             layout="head"),
        # Plain decoding of a serving batch, each sequence of another length.
        dict(name="attend_decode", seqs=32, nodes=1, len=8192, ragged=True),
        # One user's long document, a small draft tree.
        dict(name="attend_long", seqs=1, nodes=16, len=131_072, layout="head"),
        # The largest: full trees over long contexts, bound by the products.
        dict(name="attend_wide", seqs=8, nodes=64, len=32_768),
        # The smallest commit: one token after one token.
        dict(name="commit_one", seqs=1, nodes=1, q_heads=16, kv_heads=2, dim=256, len=100, kind="commit"),
        # A serving batch's accepted paths.
        dict(name="commit_batch", seqs=16, nodes=32, len=8192, ragged=True, kind="commit", path=5),
        # Long contexts, large heads.
        dict(name="commit_long", seqs=2, nodes=64, q_heads=16, kv_heads=2, dim=256, dtype="f16", len=65_536,
             layout="head", kind="commit", path=8),
        # A full cache after a step: a few slots over its budget.
        dict(name="evict_step", seqs=16, len=4128, keep=4096, recent=64, kind="evict"),
        # A prompt cut to its heaviest slots.
        dict(name="evict_prompt", seqs=4, len=32_768, keep=2048, recent=256, kind="evict", layout="head", ragged=True),
        # One user's small tree over a small, odd vocabulary.
        dict(name="verify_small", seqs=1, nodes=7, vocab=32_003, kind="verify", path=3),
        # A serving batch of trees, the thinking defaults.
        dict(name="verify_batch", seqs=8, nodes=26, kind="verify", path=4),
    ]


def draw(rng) -> dict:
    """One more case of those ranges."""
    def logint(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["attend", "attend", "attend", "commit", "commit", "evict", "evict", "verify"])
    if kind == "verify":
        nodes = rng.randint(1, 32)
        return dict(kind=kind, seqs=logint(1, max(1, 208 // nodes)), nodes=nodes, path=rng.randint(1, min(nodes, 6)),
                    vocab=V if rng.random() < 0.3 else logint(16_384, 262_144), top_k=rng.choice([5, 20, 40, 50, 100]),
                    temperature=rng.choice([0.6, 0.7, 1.0, 1.3]), top_p=rng.choice([0.8, 0.9, 0.95, 1.0]))
    q_heads, kv_heads = rng.choice([(32, 8), (16, 2), (12, 4), (8, 8), (10, 1), (28, 4), (24, 8)])
    dim = rng.choice([64, 80, 96, 128, 128, 256])
    c = dict(kind=kind, q_heads=q_heads, kv_heads=kv_heads, dim=dim, dtype=rng.choice(["bf16", "bf16", "f16"]),
             ragged=rng.random() < 0.6, layout=rng.choice(["slot", "head"]))
    # slots x kv heads x head size x sequences: at most a quarter of the largest listed case's
    most = 8 * 32_768 * 8 * 128 // 4
    c["len"] = logint(1, 65_536)
    c["seqs"] = min(logint(1, 32), max(1, most // (c["len"] * kv_heads * dim)))
    if kind == "evict":
        c["len"] = max(c["len"], 16)
        c["keep"] = rng.randint(max(8, c["len"] // 16), c["len"])
        c["recent"] = rng.randint(0, c["keep"] // 4)
        return c
    c["nodes"] = rng.choice([1, 1, rng.randint(2, 16), rng.randint(17, TREE_MAX)])
    c["path"] = rng.randint(1, min(c["nodes"], 8))
    return c


# ---------------------------------------------------------------------------
# Inputs


def _lengths(c):
    """Committed slots of each sequence: all alike, or spread from a few to all."""
    share = (1.0, 0.37, 0.81, 0.04, 0.63, 0.22, 0.93, 0.5) if c["ragged"] else (1.0,)
    return [max(1, round(c["len"] * share[b % len(share)])) for b in range(c["seqs"])]


def _used(c):
    """Nodes of each sequence's tree."""
    if c["kind"] == "verify" or not c["ragged"]:
        return [c["nodes"]] * c["seqs"]
    return [max(c["path"], c["nodes"] - (b % 3)) for b in range(c["seqs"])]


def _capacity(c):
    return (c["len"] + c["path"] + 63) // 64 * 64


def _tree(c, rng):
    """parent [seqs, nodes] and a path of c["path"] nodes down each tree."""
    parent = np.full((c["seqs"], c["nodes"]), -1, np.int32)
    path = np.full((c["seqs"], c["nodes"]), -1, np.int32)
    for b, n in enumerate(_used(c)):
        for i in range(1, n):
            parent[b, i] = rng.integers(max(0, i - 8), i)
        down = np.concatenate([[0], 1 + np.sort(rng.choice(n - 1, c["path"] - 1, replace=False))]) if n > 1 else [0]
        parent[b, down[1:]] = down[:-1]
        path[b, :c["path"]] = down
    return parent, path


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _inputs(case, seed):
    c = {**DEFAULTS, **case}
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    rng = np.random.default_rng(seed)
    B, N, D, H = c["seqs"], c["nodes"], c["dim"], c["kv_heads"]
    if c["kind"] == "verify":
        return _verify_inputs(c, g, rng)
    dt = torch.bfloat16 if c["dtype"] == "bf16" else torch.float16
    cap = _capacity(c)
    s = {"c": c, "len": torch.tensor(_lengths(c), dtype=torch.int32, device="cuda")}
    # keys gather round a direction of their head, the first slots far out along
    # it (the slots that every query looks at); [seqs, slots, heads, size] in either order
    way = _normal(g, H, D) * 0.5
    k, v = (torch.empty((B, cap, H, D) if c["layout"] == "slot" else (B, H, cap, D), dtype=dt, device="cuda") for _ in "kv")
    if c["layout"] == "head":
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    for b in range(B):
        kb = _normal(g, cap, H, D)
        kb[:4] += 4.0 * way
        k[b] = kb.to(dt)
        v[b] = _normal(g, cap, H, D).to(dt)
    s["k"], s["v"] = k, v
    if c["kind"] == "evict":
        # weights as they come: heavy-tailed, some slots with none; positions
        # out of order, as earlier evictions left them
        mass = torch.rand((B, H, cap), generator=g, device="cuda").pow(6) * 30.0
        s["mass"] = torch.where(torch.rand((B, H, cap), generator=g, device="cuda") < 0.05, 0.0, mass)
        s["pos"] = torch.rand((B, H, cap), generator=g, device="cuda").argsort(-1).int()
        for b, n in enumerate(_lengths(c)):
            s["pos"][b, :, :n] = torch.rand((H, n), generator=g, device="cuda").argsort(-1).int()
        s["next_pos"] = s["len"].clone()
        return s
    parent, path = _tree(c, rng)
    s["parent"] = torch.from_numpy(parent).cuda()
    s["n_nodes"] = torch.tensor(_used(c), dtype=torch.int32, device="cuda")
    s["q"] = (_normal(g, B, N, c["q_heads"], D) + way.repeat_interleave(c["q_heads"] // H, 0)).to(dt)
    s["fresh_k"], s["fresh_v"] = _normal(g, B, N, H, D).to(dt), _normal(g, B, N, H, D).to(dt)
    s["scale"] = 1.0 / math.sqrt(D)
    if c["kind"] == "commit":
        s["path"] = torch.from_numpy(path).cuda()
        s["n_path"] = torch.full((B,), c["path"], dtype=torch.int32, device="cuda")
        s["lse"] = _attend(s)[1]
        # a few earlier steps' worth of weight
        s["mass"] = torch.rand((B, H, cap), generator=g, device="cuda").pow(6) * (8.0 * c["path"] * c["q_heads"] / (H * c["len"]))
        s["pos"] = torch.arange(cap, dtype=torch.int32, device="cuda").repeat(B, H, 1)
        s["next_pos"] = s["len"] + 17
    return s


def _verify_inputs(c, g, rng):
    """Logits as a head leaves them (a bulk and 8 tall tokens a row); a node's
    token is one of its parent's tall ones."""
    B, N, enc = c["seqs"], c["nodes"], c["vocab"]
    ld = (enc + 3) // 4 * 4
    x = _normal(g, B * N, ld) * 3.0
    at = torch.randint(0, enc, (B * N, 8), generator=g, device="cuda")
    x.scatter_(1, at, torch.rand((B * N, 8), generator=g, device="cuda") * 6.0 + 8.0)
    parent, _ = _tree(c, rng)
    tall = x[:, :enc].topk(4, 1).indices.view(B, N, 4).cpu().numpy()
    tokens = np.zeros((B, N), np.int32)
    for b in range(B):
        for i in range(1, N):
            tokens[b, i] = tall[b, parent[b, i], rng.integers(0, 4)]
    return {"c": c, "x": x, "parent": torch.from_numpy(parent).cuda(), "tokens": torch.from_numpy(tokens).cuda(),
            "u": torch.from_numpy((rng.integers(0, 1 << 23, B * N) * 2.0**-23).astype(np.float32)).cuda()}


# ---------------------------------------------------------------------------
# The plain forms


def _ancestors(parent):
    """bool [seqs, nodes, nodes]: j is i or one of its ancestors."""
    n = parent.shape[1]
    up = (parent[:, :, None] == torch.arange(n, device=parent.device)).float()
    seen = torch.eye(n, device=parent.device).expand_as(up)
    for _ in range(max(1, n - 1).bit_length()):  # paths of up to 1, 3, 7, ... steps
        seen = seen + up @ seen
        up = up @ up
    return seen > 0


def _scores(s, q, k, scale):
    """f32 [seqs, kv heads, nodes, group, slots] of q [seqs, nodes, q heads, size] and k [seqs, slots, kv heads, size]."""
    B, N, HQ, D = q.shape
    H = k.shape[2]
    qf = q.float().view(B, N, H, HQ // H, D).permute(0, 2, 1, 3, 4).reshape(B, H, -1, D)
    kf = k.permute(0, 2, 3, 1).float().contiguous()
    return (qf @ kf * scale).view(B, H, N, HQ // H, -1)


def _attend(s):
    B, N, HQ, D = s["q"].shape
    H, top = s["k"].shape[2], s["c"]["len"]
    old = _scores(s, s["q"], s["k"][:, :top], s["scale"])
    old.masked_fill_((torch.arange(top, device="cuda") >= s["len"][:, None])[:, None, None, None], -math.inf)
    new = _scores(s, s["q"], s["fresh_k"], s["scale"])
    new.masked_fill_(~_ancestors(s["parent"])[:, None, :, None], -math.inf)
    m = torch.maximum(old.amax(-1), new.amax(-1))
    old, new = (old - m[..., None]).exp_(), (new - m[..., None]).exp_()
    total = old.sum(-1) + new.sum(-1)
    vo, vn = (v.permute(0, 2, 1, 3).float().contiguous() for v in (s["v"][:, :top], s["fresh_v"]))
    out = old.view(B, H, -1, top) @ vo + new.view(B, H, -1, N) @ vn
    out = out.view(B, H, N, HQ // H, D) / total[..., None]
    out = out.permute(0, 2, 1, 3, 4).reshape(B, N, HQ, D).to(s["q"].dtype)
    lse = (m + total.log()).permute(0, 2, 1, 3).reshape(B, N, HQ)
    used = (torch.arange(N, device="cuda") < s["n_nodes"][:, None])[..., None]
    return torch.where(used[..., None], out, 0.0), torch.where(used, lse, 0.0)


def _commit(s):
    B, N, HQ, D = s["q"].shape
    H, top, m = s["k"].shape[2], s["c"]["len"], s["c"]["path"]
    b = torch.arange(B, device="cuda")[:, None]
    path = s["path"][:, :m].long()
    q, lse = s["q"][b, path], s["lse"][b, path]  # [seqs, path, ...]
    rows = s["fresh_k"][b, path], s["fresh_v"][b, path]
    lse = lse.view(B, m, H, HQ // H).permute(0, 2, 1, 3)[..., None]
    old = (_scores(s, q, s["k"][:, :top], s["scale"]) - lse).exp_().sum((2, 3))
    new = (_scores(s, q, rows[0], s["scale"]) - lse).exp_()
    rank = torch.arange(m, device="cuda")
    new = (new * (rank[:, None] >= rank)[:, None]).sum((2, 3))
    out = {"new_mass": torch.zeros_like(s["mass"]), "pos": s["pos"], "k": s["k"], "v": s["v"]}
    out["new_mass"][:, :, :top] = torch.where(torch.arange(top, device="cuda") < s["len"][:, None, None], s["mass"][:, :, :top] + old, 0.0)
    at = s["len"][:, None].long() + rank
    out["new_mass"].transpose(1, 2)[b, at] = new.transpose(1, 2)
    s["k"][b, at], s["v"][b, at] = rows
    s["pos"].transpose(1, 2)[b, at] = (s["next_pos"][:, None] + rank).int()[..., None].expand(B, m, H)
    out["new_len"], out["new_next_pos"] = s["len"] + m, s["next_pos"] + m
    return out


def _evict(s):
    c = s["c"]
    keep, top = c["keep"], c["len"]
    slot = torch.arange(top, device="cuda")
    mass, pos, n = s["mass"][:, :, :top], s["pos"][:, :, :top], s["len"][:, None, None]
    held = (pos < c["sinks"]) | (pos >= s["next_pos"][:, None, None] - c["recent"])
    worth = torch.where(held, math.inf, mass).masked_fill(slot >= n, -math.inf)
    by_pos = pos.masked_fill(slot >= n, 2**31 - 1).sort(dim=-1, stable=True).indices
    order = by_pos.gather(-1, worth.gather(-1, by_pos).sort(dim=-1, descending=True, stable=True).indices)
    kept = torch.zeros_like(held).scatter_(-1, order[..., :keep], True) & (slot < n)
    free = ~kept & (slot < keep) & (n > keep)
    late = kept & (slot >= keep)
    to, frm = ((~f).to(torch.uint8).sort(dim=-1, stable=True).indices for f in (free, late))
    source = slot.expand_as(pos).clone()
    most = min(keep, top - keep)
    pair = slot[:most] < free.sum(-1, keepdim=True)
    source.scatter_(-1, to[..., :most], torch.where(pair, frm[..., :most], to[..., :most]))
    new_len = s["len"].clamp(max=keep)
    out = {"k": s["k"], "v": s["v"], "new_len": new_len}
    inside = slot[:keep] < new_len[:, None, None]
    source = source[..., :keep]
    for name in ("mass", "pos"):
        out["new_" + name] = torch.zeros_like(s[name])
        out["new_" + name][:, :, :keep] = torch.where(inside, s[name].gather(-1, source), 0)
    b, h, i = (source != slot[:keep]).nonzero(as_tuple=True)
    j = source[b, h, i]
    s["k"][b, i, h], s["v"][b, i, h] = s["k"][b, j, h], s["v"][b, j, h]
    return out


def _draw_rows(x, c, u):
    """One token a row: the k best of the softmax at the temperature, cut to the
    nucleus of top_p, drawn by u.  The sums over a handful of weights add one
    after the other in 32 bits, as the sampler's definition says."""
    z = x * np.float32(1.0 / c["temperature"]) if c["temperature"] != 1.0 else x
    top = z.max(1, keepdim=True).values
    total = (z - top).double().exp_().sum(1, keepdim=True).float()
    k = c["top_k"]
    val, ids = z.sort(dim=1, descending=True, stable=True)
    val, ids = val[:, :k + 28], ids[:, :k + 28]
    p = (val - top).double().exp().float() / total
    ids, first = ids.sort(1)
    p, first = p.gather(1, first).sort(dim=1, descending=True, stable=True)
    ids, w = ids.gather(1, first)[:, :k], list(p[:, :k].unbind(1))

    def add(values):
        run = [values[0]]
        for y in values[1:]:
            run.append(run[-1] + y)
        return run

    if c["top_p"] < 1.0:
        whole = add(w)[-1]
        w = [y / whole for y in w]
        so_far = add(w)
        w = w[:1] + [torch.where(so_far[i - 1] >= np.float32(c["top_p"]), 0.0, w[i]) for i in range(1, k)]
    steps = torch.stack(add(w), 1)
    at = (steps[:, :-1] <= (u * steps[:, -1])[:, None]).sum(1, keepdim=True)
    return ids.gather(1, at)[:, 0].int()


def _verify(s):
    c = s["c"]
    B, N = s["tokens"].shape
    token = _draw_rows(s["x"][:, :c["vocab"]], c, s["u"])
    drawn, b = token.view(B, N), torch.arange(B, device="cuda")
    node = torch.arange(N, device="cuda")
    cur = torch.zeros(B, dtype=torch.long, device="cuda")
    alive = torch.ones(B, dtype=torch.bool, device="cuda")
    path, committed = [], []
    for _ in range(N):
        t = drawn[b, cur]
        committed.append(torch.where(alive, t, -1))
        path.append(torch.where(alive, cur, -1))
        fits = (s["parent"] == cur[:, None]) & (s["tokens"] == t[:, None]) & (node > cur[:, None])
        alive = alive & fits.any(1)
        cur = torch.where(alive, fits.int().argmax(1), cur)
    path, committed = torch.stack(path, 1).int(), torch.stack(committed, 1).int()
    n = (committed >= 0).sum(1).int()
    return {"row_token": token, "row_status": torch.zeros_like(token), "path": path, "accepted": n - 1,
            "committed": committed, "n_committed": n, "seq_status": torch.zeros_like(n)}


# ---------------------------------------------------------------------------
# One call


def _tensor_ptr(a, **tensors):
    for f, t in tensors.items():
        setattr(a, f, t.data_ptr())


def _kv(kv, k, v):
    kv.k, kv.v = k.data_ptr(), v.data_ptr()
    kv.seq_stride, kv.slot_stride, kv.head_stride = k.stride()[:3]


def _call(s):
    """The argument struct, the context and the outputs an engine keeps."""
    from xwen_amd import _lib, tree
    from xwen_amd import sampler as xsm

    c = s["c"]
    B, N = c["seqs"], c["nodes"]
    lib = _lib.load()

    def new(*shape, dtype=torch.int32):
        return torch.zeros(shape, dtype=dtype, device="cuda")

    if c["kind"] == "verify":
        ctx = xsm.Context(max_rows=B * N, vocab=c["vocab"])
        ctx.bind_current_stream()
        a = _lib.VerifyTreeArgs()
        a.seqs, a.nodes, a.ld, a.width, a.enc = B, N, s["x"].shape[1], s["x"].shape[1], c["vocab"]
        s["params"] = xsm.params_tensor(c["temperature"], c["top_k"], c["top_p"], B * N, "cuda")
        _tensor_ptr(a, logits=s["x"], params=s["params"], uniforms=s["u"], tokens=s["tokens"], parent=s["parent"])
        out = {f: new(B * N) for f in ("row_token", "row_status")}
        out.update({f: new(B, N) for f in ("path", "committed")})
        out.update({f: new(B) for f in ("accepted", "n_committed", "seq_status")})
        _tensor_ptr(a, **out)
        return ctx, lib.xs_verify_tree, a, out
    ctx = tree.CacheContext(max_seqs=B, max_nodes=N, q_heads=c["q_heads"], kv_heads=c["kv_heads"], head_dim=c["dim"],
                            capacity=_capacity(c))
    ctx.bind_current_stream()
    a = {"attend": _lib.TreeAttendArgs, "commit": _lib.CacheCommitArgs, "evict": _lib.CacheEvictArgs}[c["kind"]]()
    a.dtype = _lib.BF16 if c["dtype"] == "bf16" else _lib.F16
    a.head_dim, a.seqs, a.kv_heads, a.capacity, a.max_len = c["dim"], B, c["kv_heads"], _capacity(c), c["len"]
    _kv(a.cache, s["k"], s["v"])
    status = new(B)
    _tensor_ptr(a, len=s["len"], seq_status=status)
    if c["kind"] == "evict":
        a.keep, a.sinks, a.recent, a.slot_ld = c["keep"], c["sinks"], c["recent"], _capacity(c)
        out = {"new_mass": torch.zeros_like(s["mass"]), "new_pos": torch.zeros_like(s["pos"]), "new_len": new(B)}
        _tensor_ptr(a, mass=s["mass"], pos=s["pos"], next_pos=s["next_pos"], **out)
        out.update(k=s["k"], v=s["v"])
        s["status"] = status
        return ctx, lib.xs_cache_evict, a, out
    a.nodes, a.q_heads, a.scale = N, c["q_heads"], s["scale"]
    _kv(a.fresh, s["fresh_k"], s["fresh_v"])
    _tensor_ptr(a, q=s["q"])
    a.q_seq_stride, a.q_node_stride, a.q_head_stride = s["q"].stride()[:3]
    s["status"] = status
    if c["kind"] == "attend":
        out = {"out": torch.zeros_like(s["q"]), "lse": new(B, N, c["q_heads"], dtype=torch.float32)}
        _tensor_ptr(a, parent=s["parent"], n_nodes=s["n_nodes"], **out)
        a.out_seq_stride, a.out_node_stride, a.out_head_stride = out["out"].stride()[:3]
        return ctx, lib.xs_tree_attend, a, out
    a.slot_ld, a.path_ld = _capacity(c), N
    out = {"new_mass": torch.zeros_like(s["mass"]), "pos": s["pos"], "new_len": new(B), "new_next_pos": new(B)}
    _tensor_ptr(a, path=s["path"], n_path=s["n_path"], lse=s["lse"], mass=s["mass"], next_pos=s["next_pos"], **out)
    out.update(k=s["k"], v=s["v"])
    return ctx, lib.xs_cache_commit, a, out


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        s["ctx"], s["call"], s["args"], s["out"] = _call(s)
        s["ref"] = C.byref(s["args"])
    return s


def run(state):
    if own:
        rc = state["call"](state["ctx"].h, state["ref"])
        if rc:
            raise RuntimeError(f"call failed: {rc}")
        return state["out"]
    kind = state["c"]["kind"]
    if kind == "attend":
        return dict(zip(("out", "lse"), _attend(state)))
    return {"commit": _commit, "evict": _evict, "verify": _verify}[kind](state)


def work(case):
    """Each input that the result needs read once, each output written once."""
    c = {**DEFAULTS, **case}
    B, N, H, HQ, D = c["seqs"], c["nodes"], c["kv_heads"], c["q_heads"], c["dim"]
    if c["kind"] == "verify":
        return {"bytes": B * N * (4.0 * c["vocab"] + 44.0), "flops": 4.0 * B * N * c["vocab"]}
    lens, used = _lengths(c), _used(c)
    if c["kind"] == "attend":
        b = sum(4.0 * (n + u) * H * D + u * HQ * (4.0 * D + 4.0) for n, u in zip(lens, used))
        return {"bytes": b, "flops": sum(4.0 * D * HQ * u * (n + 1) for n, u in zip(lens, used))}
    if c["kind"] == "commit":
        m = c["path"]
        b = sum((2.0 * D + 8.0) * H * n + m * (8.0 * H * D + 2.0 * HQ * D + 4.0 * HQ + 8.0 * H) for n in lens)
        return {"bytes": b, "flops": sum(2.0 * D * HQ * m * (n + 1) for n in lens)}
    b = 0.0
    for n in lens:
        left = min(n, c["keep"])
        moved = left * (n - left) / n  # a slot past the budget is kept as often as any other
        b += H * (8.0 * n + 8.0 * left + moved * 8.0 * D)
    return {"bytes": b, "flops": 2.0 * H * sum(lens)}


# ---------------------------------------------------------------------------
# The same in 64 bits


def exact(case, seed):
    """Computed numbers only: eviction moves what is there, verification answers
    with whole numbers."""
    c = {**DEFAULTS, **case}
    if c["kind"] in ("evict", "verify"):
        return None
    s = _inputs(case, seed)
    q, k, v = s["q"].double(), s["k"], s["v"]
    B, N, HQ, D = q.shape
    H = c["kv_heads"]
    G = HQ // H
    parent = s["parent"].tolist()
    if c["kind"] == "attend":
        out = torch.zeros((B, N, HQ, D), dtype=torch.float64, device="cuda")
        lse = torch.zeros((B, N, HQ), dtype=torch.float64, device="cuda")
    else:
        mass = torch.zeros(s["mass"].shape, dtype=torch.float64, device="cuda")
    for b, (n, used) in enumerate(zip(_lengths(c), _used(c))):
        sees = torch.zeros((used, used), dtype=torch.bool, device="cuda")
        for i in range(used):
            j = i
            while j >= 0:
                sees[i, j] = True
                j = parent[b][j]
        for h in range(H):
            heads = slice(h * G, (h + 1) * G)
            keys = torch.cat([k[b, :n, h], s["fresh_k"][b, :used, h]]).double()
            dots = torch.einsum("igd,sd->igs", q[b, :used, heads], keys) / math.sqrt(D)
            dots[:, :, n:].masked_fill_(~sees[:, None], -math.inf)
            if c["kind"] == "attend":
                values = torch.cat([v[b, :n, h], s["fresh_v"][b, :used, h]]).double()
                lse[b, :used, heads] = dots.logsumexp(-1)
                out[b, :used, heads] = dots.softmax(-1) @ values
            else:
                chain = s["path"][b, :c["path"]].long()
                weight = (dots[chain] - s["lse"][b, chain, heads].double()[..., None]).exp().sum((0, 1))
                mass[b, h, :n] = s["mass"][b, h, :n].double() + weight[:n]
                mass[b, h, n:n + c["path"]] = weight[n + chain]
    if c["kind"] == "attend":
        return {"out": out, "lse": lse}
    return {"new_mass": mass, "pos": None, "k": None, "v": None, "new_len": None, "new_next_pos": None}
