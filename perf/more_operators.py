"""From a prompt to a cache held in 8 bits: the operators whose speed is watched.

A layer's projections give queries and keys that are normed per head and turned
by their positions ("rotate"); a prompt's tokens attend to themselves ("prompt");
their keys and values, and later those of each step's accepted path, go into a
cache of e4m3 values with a power-of-two scale for every 32 slots of a head
("append"); a step's draft tree attends over that cache ("attend8").  A case is
one call of one of them, through the C ABI of include/xsamp.h, with the argument
struct, the context and the buffers that an engine keeps between steps.

The sizes are generic, as in perf/operators.py.  With `own` false, run()
computes the same in elementary torch operations.
"""
from __future__ import annotations

import ctypes as C
import math

import numpy as np
import torch

own = False

BLOCK = 32        # slots that share a scale
EXP_MIN = -100    # the least exponent of a scale
TREE_MAX = 64
EPS = 1e-6

DEFAULTS = dict(kind="attend8", seqs=1, nodes=1, q_heads=32, kv_heads=8, dim=128, dtype="bf16", len=128, ragged=False,
                layout="slot", path=1, rot=128, pairs="halves", norm=True)


def listed() -> list[dict]:
    return [
        # One new token of one user: large heads of which a quarter turns.
        dict(name="rotate_one", kind="rotate", seqs=1, len=1, q_heads=16, kv_heads=2, dim=256, rot=64),
        # A long prompt's queries and keys.
        dict(name="rotate_prompt", kind="rotate", seqs=1, len=16_384),
        # The smallest prompt: a short question.
        dict(name="prompt_one", kind="prompt", seqs=1, len=100, q_heads=16, kv_heads=2, dim=256),
        # An odd model and odd lengths: 3 users, head size 80, float16.
        dict(name="prompt_odd", kind="prompt", seqs=3, len=1777, q_heads=12, kv_heads=4, dim=80, dtype="f16", ragged=True),
        # A serving batch of prompts, packed, each of another length.
        dict(name="prompt_pack", kind="prompt", seqs=16, len=4096, ragged=True),
        # The largest: one user's long document.
        dict(name="prompt_long", kind="prompt", seqs=1, len=16_384),
        # A serving batch's accepted paths.
        dict(name="append_step", kind="append", seqs=16, nodes=32, len=8192, ragged=True, path=5),
        # Whole prompts into empty caches.
        dict(name="append_prompt", kind="append", seqs=4, nodes=0, len=8192, ragged=True),
        # One new token of one user over a short context.
        dict(name="attend8_one", seqs=1, nodes=1, q_heads=16, kv_heads=2, dim=256, len=100),
        # Plain decoding of a serving batch, each sequence of another length.
        dict(name="attend8_decode", seqs=32, nodes=1, len=8192, ragged=True),
        # One user's long document, a small draft tree.
        dict(name="attend8_long", seqs=1, nodes=16, len=131_072, layout="head"),
        # Full trees over long contexts, bound by the products.
        dict(name="attend8_wide", seqs=8, nodes=64, len=16_384),
    ]


def draw(rng) -> dict:
    """One more case of those ranges."""
    def logint(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["rotate", "prompt", "prompt", "append", "attend8", "attend8"])
    q_heads, kv_heads = rng.choice([(32, 8), (16, 2), (12, 4), (8, 8), (10, 1), (28, 4), (20, 4)])
    c = dict(kind=kind, q_heads=q_heads, kv_heads=kv_heads, dim=rng.choice([64, 80, 96, 128, 128, 256]),
             dtype=rng.choice(["bf16", "bf16", "f16"]), ragged=rng.random() < 0.6)
    if kind == "rotate":
        c["len"] = logint(1, 8192)
        c["seqs"] = min(logint(1, 8), max(1, 8192 // c["len"]))
        c["pairs"] = rng.choice(["halves", "halves", "neighbours"])
        c["rot"] = rng.choice([c["dim"], c["dim"], c["dim"] // 32 * 16])
        c["norm"] = rng.random() < 0.8
        return c
    if kind == "prompt":
        c["len"] = logint(1, 8192)
        # rows x keys x heads x head size: at most a third of the largest listed case's
        most = 16_384**2 * 32 * 128 // 3
        c["seqs"] = min(logint(1, 32), max(1, most // (c["len"]**2 * q_heads * c["dim"])))
        return c
    c["layout"] = rng.choice(["slot", "head"])
    # slots x kv heads x head size x sequences: at most half of a large listed case's
    most = 8 * 16_384 * 8 * 128 // 2
    if kind == "append" and rng.random() < 0.5:  # whole prompts
        c["nodes"], c["len"] = 0, logint(1, 16_384)
        c["seqs"] = min(logint(1, 32), max(1, most // (c["len"] * kv_heads * c["dim"])))
        return c
    c["len"] = logint(1, 65_536)
    c["seqs"] = min(logint(1, 32), max(1, most // (c["len"] * kv_heads * c["dim"])))
    c["nodes"] = rng.choice([1, 1, rng.randint(2, 16), rng.randint(17, TREE_MAX)])
    c["path"] = rng.randint(1, min(c["nodes"], 8))
    return c


# ---------------------------------------------------------------------------
# Inputs


def _lengths(c):
    """Tokens of each sequence: all alike, or spread from a few to all."""
    share = (1.0, 0.37, 0.81, 0.04, 0.63, 0.22, 0.93, 0.5) if c["ragged"] else (1.0,)
    return [max(1, round(c["len"] * share[b % len(share)])) for b in range(c["seqs"])]


def _used(c):
    """Nodes of each sequence's tree."""
    if not c["ragged"]:
        return [c["nodes"]] * c["seqs"]
    return [max(c["path"], c["nodes"] - (b % 3)) for b in range(c["seqs"])]


def _rows(c):
    """Rows that each sequence of an append takes: a path's, or the whole prompt."""
    return [c["path"]] * c["seqs"] if c["nodes"] else _lengths(c)


def _old(c):
    """Slots in use before an append."""
    return _lengths(c) if c["nodes"] else [0] * c["seqs"]


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


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _starts(lens):
    return _ints(np.concatenate([[0], np.cumsum(lens)]).tolist())


def _inputs(case, seed):
    c = {**DEFAULTS, **case}
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    rng = np.random.default_rng(seed)
    B, N, D, H, HQ = c["seqs"], c["nodes"], c["dim"], c["kv_heads"], c["q_heads"]
    dt = torch.bfloat16 if c["dtype"] == "bf16" else torch.float16
    lens = _lengths(c)
    s = {"c": c, "scale": 1.0 / math.sqrt(D)}
    # keys gather round a direction of their head, the first ones far out along
    # it (the tokens that every query looks at)
    way = _normal(g, H, D) * 0.5
    if c["kind"] in ("rotate", "prompt"):
        # one projection's output: a token's query heads, its key heads, its value heads
        T = sum(lens)
        x = _normal(g, T, HQ + 2 * H, D)
        s["start"] = _starts(lens)
        if c["kind"] == "rotate":
            # sequences in the middle of their texts
            first = rng.integers(0, 100_000, B)
            s["pos"] = _ints(np.concatenate([f + np.arange(n) for f, n in zip(first, lens)]).tolist())
            s["inv_freq"] = (1e6 ** (-torch.arange(0, c["rot"], 2, device="cuda", dtype=torch.float64) / c["rot"])).float()
            for w in ("q_weight", "k_weight"):
                s[w] = 1.0 + 0.2 * _normal(g, D) if c["norm"] else None
        else:
            x[:, :HQ] += way.repeat_interleave(HQ // H, 0)
            for i in s["start"][:-1].tolist():
                x[i:i + 4, HQ:HQ + H] += 4.0 * way
        x = x.to(dt)
        s["q"], s["k"], s["v"] = x[:, :HQ], x[:, HQ:HQ + H], x[:, HQ + H:]
        return s
    cap = _capacity(c)
    s["len"] = _ints(_old(c))
    shape = (B, cap, H, D) if c["layout"] == "slot" else (B, H, cap, D)
    k, v = (torch.empty(shape, dtype=torch.float8_e4m3fn, device="cuda") for _ in "kv")
    if c["layout"] == "head":
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    for name, t in (("k", k), ("v", v)):
        s[name], s[name + "_exp"] = t, torch.empty((B, H, cap // BLOCK), dtype=torch.uint8, device="cuda")
        for b in range(B):
            x = _normal(g, cap, H, D)
            if name == "k":
                x[:4] += 4.0 * way
            e = _exponents(x.view(-1, BLOCK, H, D).abs().amax((1, 3)))
            t[b] = torch.ldexp(x, -e.repeat_interleave(BLOCK, 0)[:, :, None]).to(torch.float8_e4m3fn)
            s[name + "_exp"][b] = (e.T + 127).to(torch.uint8)
    if c["kind"] == "append" and N == 0:
        T = sum(lens)
        s["start"] = _starts(lens)
        s["fresh_k"], s["fresh_v"] = (_normal(g, T, H, D).to(dt) for _ in "kv")
        return s
    parent, path = _tree(c, rng)
    s["fresh_k"], s["fresh_v"] = (_normal(g, B, N, H, D).to(dt) for _ in "kv")
    if c["kind"] == "append":
        s["path"], s["n_path"] = torch.from_numpy(path).cuda(), _ints([c["path"]] * B)
        return s
    s["parent"], s["n_nodes"] = torch.from_numpy(parent).cuda(), _ints(_used(c))
    s["q"] = (_normal(g, B, N, HQ, D) + way.repeat_interleave(HQ // H, 0)).to(dt)
    return s


# ---------------------------------------------------------------------------
# The plain forms


def _exponents(most):
    """The least exponent e with most <= 448 * 2^e (448: the largest e4m3), and EXP_MIN at least."""
    m, x = torch.frexp(most)
    e = x - 9 + (m > 0.875).int()
    return torch.where(most > 0, e, EXP_MIN).clamp(min=EXP_MIN).int()


def _rotate(s):
    c = s["c"]
    r = c["rot"]
    turn = s["pos"][:, None].double() * s["inv_freq"].double()
    cos, sin = turn.cos().float()[:, None], turn.sin().float()[:, None]
    out = {}
    for name in ("q", "k"):
        x = s[name].float()
        if s[name + "_weight"] is not None:
            x = x * (x.square().mean(-1, keepdim=True) + EPS).rsqrt() * s[name + "_weight"]
        if c["pairs"] == "halves":
            a, b = x[..., :r // 2], x[..., r // 2:r]
            y = torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., r:]], -1)
        else:
            a, b = x[..., 0:r:2], x[..., 1:r:2]
            y = torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), x[..., r:]], -1)
        out[name] = y.to(s[name].dtype)
    return out


def _prompt(s):
    c = s["c"]
    D, H, HQ = c["dim"], c["kv_heads"], c["q_heads"]
    G = HQ // H
    out = torch.empty((s["q"].shape[0], HQ, D), dtype=s["q"].dtype, device="cuda")
    lse = torch.empty((s["q"].shape[0], HQ), device="cuda")
    first = 0
    for n in _lengths(c):
        q = s["q"][first:first + n].float().view(n, H, G, D).permute(1, 2, 0, 3)
        k = s["k"][first:first + n].permute(1, 2, 0).float().contiguous()
        v = s["v"][first:first + n].permute(1, 0, 2).float().contiguous()
        step = max(64, (1 << 29) // (HQ * n))  # rows whose scores fill 2 GB
        for i in range(0, n, step):
            m = min(i + step, n)
            x = (q[:, :, i:m].reshape(H, -1, D) @ k[:, :, :m] * s["scale"]).view(H, G, m - i, m)
            x.masked_fill_(torch.arange(m, device="cuda") > torch.arange(i, m, device="cuda")[:, None], -math.inf)
            top = x.amax(-1, keepdim=True)
            x = (x - top).exp_()
            total = x.sum(-1, keepdim=True)
            y = (x.view(H, -1, m) @ v[:, :m]).view(H, G, m - i, D) / total
            out[first + i:first + m] = y.permute(2, 0, 1, 3).reshape(m - i, HQ, D).to(out.dtype)
            lse[first + i:first + m] = (top + total.log())[..., 0].permute(2, 0, 1).reshape(m - i, HQ)
        first += n
    return {"out": out, "lse": lse}


def _append(s):
    c = s["c"]
    H, D = c["kv_heads"], c["dim"]
    for b, (n, m) in enumerate(zip(_old(c), _rows(c))):
        at, end = n // BLOCK * BLOCK, (n + m + BLOCK - 1) // BLOCK * BLOCK
        i, j = at // BLOCK, end // BLOCK
        for name in ("k", "v"):
            cache, exps = s[name], s[name + "_exp"]
            rows = s["fresh_" + name]
            rows = rows[b, s["path"][b, :m].long()] if c["nodes"] else rows[s["start"][b]:s["start"][b] + m]
            x = torch.zeros((end - at, H, D), device="cuda")
            x[n - at:n - at + m] = rows.float()
            e = _exponents(x.view(-1, BLOCK, H, D).abs().amax((1, 3)))
            if n > at:  # the block that is partly in use keeps its scale or grows it
                old = exps[b, :, i].int() - 127
                e[0] = torch.maximum(e[0], old)
                x[:n - at] = torch.ldexp(cache[b, at:n].float(), old[:, None])
            x = torch.ldexp(x, -e.repeat_interleave(BLOCK, 0)[:, :, None]).to(torch.float8_e4m3fn)
            cache.view(torch.uint8)[b, at:n + m] = x.view(torch.uint8)[:n + m - at]
            exps[b, :, i:j] = (e.T + 127).to(torch.uint8)
    return {"k": s["k"], "v": s["v"], "k_exp": s["k_exp"], "v_exp": s["v_exp"], "new_len": s["len"] + _ints(_rows(c))}


def _ancestors(parent):
    """bool [seqs, nodes, nodes]: j is i or one of its ancestors."""
    n = parent.shape[1]
    up = (parent[:, :, None] == torch.arange(n, device=parent.device)).float()
    seen = torch.eye(n, device=parent.device).expand_as(up)
    for _ in range(max(1, n - 1).bit_length()):  # paths of up to 1, 3, 7, ... steps
        seen = seen + up @ seen
        up = up @ up
    return seen > 0


def _values(s, name, top):
    """f32 [seqs, kv heads, slots, size] of the cache's first slots."""
    x = s[name][:, :top].permute(0, 2, 1, 3).float()
    e = s[name + "_exp"][:, :, :(top + BLOCK - 1) // BLOCK].int() - 127
    return torch.ldexp(x, e.repeat_interleave(BLOCK, 2)[:, :, :top, None])


def _attend(s):
    c = s["c"]
    B, N, HQ, D = s["q"].shape
    H, top = c["kv_heads"], c["len"]
    G = HQ // H
    q = s["q"].float().view(B, N, H, G, D).permute(0, 2, 1, 3, 4).reshape(B, H, -1, D)

    def scores(keys):
        return (q @ keys.transpose(2, 3).contiguous() * s["scale"]).view(B, H, N, G, -1)

    old = scores(_values(s, "k", top))
    old.masked_fill_((torch.arange(top, device="cuda") >= s["len"][:, None])[:, None, None, None], -math.inf)
    new = scores(s["fresh_k"].permute(0, 2, 1, 3).float())
    new.masked_fill_(~_ancestors(s["parent"])[:, None, :, None], -math.inf)
    m = torch.maximum(old.amax(-1), new.amax(-1))
    old, new = (old - m[..., None]).exp_(), (new - m[..., None]).exp_()
    total = old.sum(-1) + new.sum(-1)
    out = old.view(B, H, -1, top) @ _values(s, "v", top)
    out += new.view(B, H, -1, N) @ s["fresh_v"].permute(0, 2, 1, 3).float().contiguous()
    out = out.view(B, H, N, G, D) / total[..., None]
    out = out.permute(0, 2, 1, 3, 4).reshape(B, N, HQ, D).to(s["q"].dtype)
    lse = (m + total.log()).permute(0, 2, 1, 3).reshape(B, N, HQ)
    used = (torch.arange(N, device="cuda") < s["n_nodes"][:, None])[..., None]
    return {"out": torch.where(used[..., None], out, 0.0), "lse": torch.where(used, lse, 0.0)}


# ---------------------------------------------------------------------------
# One call


def _fields(a, **tensors):
    for f, t in tensors.items():
        setattr(a, f, t.data_ptr())


def _fresh(kv, k, v, dims):
    kv.k, kv.v = k.data_ptr(), v.data_ptr()
    strides = k.stride()[:-1]
    kv.seq_stride, kv.slot_stride, kv.head_stride = strides if dims == 4 else (0, *strides)


def _cache(kv, s):
    kv.k, kv.v, kv.k_exp, kv.v_exp = (s[n].data_ptr() for n in ("k", "v", "k_exp", "v_exp"))
    kv.seq_stride, kv.slot_stride, kv.head_stride = s["k"].stride()[:3]
    kv.exp_ld = s["k_exp"].shape[2]


def _call(s):
    """The argument struct, the context and the outputs an engine keeps."""
    from xwen_amd import _lib, tree

    c = s["c"]
    lib = _lib.load()
    B, H, HQ, D, kind = c["seqs"], c["kv_heads"], c["q_heads"], c["dim"], c["kind"]
    ctx = tree.CacheContext(max_seqs=B, max_nodes=max(1, c["nodes"]), q_heads=HQ, kv_heads=H, head_dim=D, capacity=_capacity(c))
    ctx.bind_current_stream()
    a = {"rotate": _lib.QkRotateArgs, "prompt": _lib.PromptAttendArgs, "append": _lib.CacheAppend8Args,
         "attend8": _lib.TreeAttend8Args}[kind]()
    a.dtype = _lib.BF16 if c["dtype"] == "bf16" else _lib.F16
    a.head_dim, a.kv_heads = D, H
    status = torch.zeros(B, dtype=torch.int32, device="cuda")
    s["status"] = status
    if kind == "rotate":
        a.tokens, a.q_heads, a.rot_dim, a.eps = s["q"].shape[0], HQ, c["rot"], EPS
        a.pairs = _lib.ROT_HALVES if c["pairs"] == "halves" else _lib.ROT_NEIGHBOURS
        out = {n: torch.empty(s[n].shape, dtype=s[n].dtype, device="cuda") for n in ("q", "k")}
        _fields(a, q=s["q"], k=s["k"], inv_freq=s["inv_freq"], pos=s["pos"], q_out=out["q"], k_out=out["k"])
        if c["norm"]:
            _fields(a, q_weight=s["q_weight"], k_weight=s["k_weight"])
        for n in ("q", "k"):
            for to, t in ((n, s[n]), (n + "_out", out[n])):
                setattr(a, to + "_token_stride", t.stride(0))
                setattr(a, to + "_head_stride", t.stride(1))
        return ctx, lib.xs_qk_rotate, a, out
    if kind == "prompt":
        T = s["q"].shape[0]
        a.seqs, a.tokens, a.q_heads, a.scale = B, T, HQ, s["scale"]
        out = {"out": torch.empty(s["q"].shape, dtype=s["q"].dtype, device="cuda"), "lse": torch.empty((T, HQ), device="cuda")}
        _fields(a, q=s["q"], k=s["k"], v=s["v"], start=s["start"], seq_status=status, **out)
        a.q_token_stride, a.q_head_stride = s["q"].stride()[:2]
        a.kv_token_stride, a.kv_head_stride = s["k"].stride()[:2]
        a.out_token_stride, a.out_head_stride = out["out"].stride()[:2]
        return ctx, lib.xs_prompt_attend, a, out
    a.seqs, a.capacity = B, _capacity(c)
    _cache(a.cache, s)
    _fields(a, len=s["len"], seq_status=status)
    _fresh(a.fresh, s["fresh_k"], s["fresh_v"], s["fresh_k"].dim())
    if kind == "append":
        out = {"new_len": torch.zeros(B, dtype=torch.int32, device="cuda")}
        _fields(a, **out)
        if c["nodes"]:
            a.rows, a.path_ld = c["nodes"], c["nodes"]
            _fields(a, path=s["path"], n_path=s["n_path"])
        else:
            a.rows, a.tokens = c["len"], s["fresh_k"].shape[0]
            _fields(a, start=s["start"])
        out.update({n: s[n] for n in ("k", "v", "k_exp", "v_exp")})
        return ctx, lib.xs_cache_append8, a, out
    a.nodes, a.q_heads, a.scale, a.max_len = c["nodes"], HQ, s["scale"], c["len"]
    out = {"out": torch.zeros_like(s["q"]), "lse": torch.zeros((B, c["nodes"], HQ), device="cuda")}
    _fields(a, q=s["q"], parent=s["parent"], n_nodes=s["n_nodes"], **out)
    a.q_seq_stride, a.q_node_stride, a.q_head_stride = s["q"].stride()[:3]
    a.out_seq_stride, a.out_node_stride, a.out_head_stride = out["out"].stride()[:3]
    return ctx, lib.xs_tree_attend8, a, out


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
    return {"rotate": _rotate, "prompt": _prompt, "append": _append, "attend8": _attend}[state["c"]["kind"]](state)


def work(case):
    """Each input that the result needs read once, each output written once."""
    c = {**DEFAULTS, **case}
    N, H, HQ, D = c["nodes"], c["kv_heads"], c["q_heads"], c["dim"]
    lens = _lengths(c)
    if c["kind"] == "rotate":
        x = sum(lens) * (HQ + H) * D
        return {"bytes": 4.0 * x + 4.0 * sum(lens), "flops": 8.0 * x}
    if c["kind"] == "prompt":
        return {"bytes": sum(lens) * (4.0 * HQ * D + 4.0 * H * D + 4.0 * HQ), "flops": sum(2.0 * D * HQ * n * (n + 1) for n in lens)}
    if c["kind"] == "append":
        # rows in, bytes out; a block partly in use may have to be read and written again, but need not
        x = sum(_rows(c)) * H * D
        return {"bytes": 6.0 * x, "flops": 4.0 * x}
    used = _used(c)
    b = sum((2.0 * n * D + 2.0 * n / BLOCK) * H + 4.0 * u * H * D + u * HQ * (4.0 * D + 4.0) for n, u in zip(lens, used))
    return {"bytes": b, "flops": sum(4.0 * D * HQ * u * (n + 1) for n, u in zip(lens, used))}


# ---------------------------------------------------------------------------
# The same in 64 bits


def exact(case, seed):
    s = _inputs(case, seed)
    return {"rotate": _exact_rotate, "prompt": _exact_prompt, "append": _exact_append, "attend8": _exact_attend}[s["c"]["kind"]](s)


def _exact_rotate(s):
    """Each pair as a complex number, turned by exp(i angle)."""
    c, r = s["c"], s["c"]["rot"]
    unit = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), torch.outer(s["pos"].double(), s["inv_freq"].double()))
    out = {}
    for name in ("q", "k"):
        x = s[name].double()
        if c["norm"]:
            x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / c["dim"] + EPS) * s[name + "_weight"].double()
        else:
            x = x.clone()
        re, im = (slice(0, r // 2), slice(r // 2, r)) if c["pairs"] == "halves" else (slice(0, r, 2), slice(1, r, 2))
        z = torch.complex(x[..., re].contiguous(), x[..., im].contiguous()) * unit[:, None]
        x[..., re], x[..., im] = z.real, z.imag
        out[name] = x
    return out


def _exact_prompt(s):
    c = s["c"]
    D, H, HQ = c["dim"], c["kv_heads"], c["q_heads"]
    G = HQ // H
    out = torch.empty((s["q"].shape[0], HQ, D), dtype=torch.float64, device="cuda")
    lse = torch.empty((s["q"].shape[0], HQ), dtype=torch.float64, device="cuda")
    start = s["start"].tolist()
    for first, last in zip(start, start[1:]):
        for h in range(HQ):
            k, v = s["k"][first:last, h // G].double(), s["v"][first:last, h // G].double()
            for i in range(first, last, 8192):
                j = min(i + 8192, last)
                x = s["q"][i:j, h].double() @ k[:j - first].T.contiguous() / math.sqrt(D)
                x = x.tril_(i - first) + torch.full_like(x, -math.inf).triu_(i - first + 1)
                lse[i:j, h] = x.logsumexp(-1)
                out[i:j, h] = x.softmax(-1) @ v[:j - first]
    return {"out": out, "lse": lse}


def _near(x):
    """The nearest value with 3 bits after the leading one, or a multiple of 2^-9; ties to even."""
    step = torch.exp2(torch.frexp(x).exponent.double().clamp(min=-5) - 4)
    return torch.round(x / step) * step


def _exact_append(s):
    """Block by block, from the values that the cache stands for."""
    c = s["c"]
    out = {"k_exp": None, "v_exp": None, "new_len": None}
    for name in ("k", "v"):
        old = s[name].double()
        got = old.clone()
        for b, (n, m) in enumerate(zip(_old(c), _rows(c))):
            pick = s["path"][b, :m].tolist() if c["nodes"] else None
            rows = (s["fresh_" + name][b, pick] if c["nodes"] else s["fresh_" + name][s["start"][b]:s["start"][b + 1]]).double()
            i = n // BLOCK
            had = s[name + "_exp"][b, :, i].double() - 127 if n % BLOCK else None
            edge = min(m, BLOCK - n % BLOCK) if n % BLOCK else 0
            if edge:  # joins the rows that the block has
                most = rows[:edge].abs().amax((0, 2))
                e = torch.maximum(torch.ceil(torch.log2(most / 448)), had)
                part = old[b, i * BLOCK:n] * torch.exp2(had - e)[:, None]
                got[b, i * BLOCK:n] = torch.where((had == e)[:, None], old[b, i * BLOCK:n], _near(part))
                got[b, n:n + edge] = _near(rows[:edge] * torch.exp2(-e)[:, None])
            for j in range(edge, m, 4096):
                x = rows[j:min(m, j + 4096)]
                pad = torch.zeros((-len(x) % BLOCK, *x.shape[1:]), dtype=torch.float64, device="cuda")
                y = torch.cat([x, pad]).view(-1, BLOCK, *x.shape[1:])
                e = torch.ceil(torch.log2(y.abs().amax((1, 3), keepdim=True) / 448)).clamp(min=EXP_MIN)
                got[b, n + j:n + j + len(x)] = _near(y * torch.exp2(-e)).flatten(0, 1)[:len(x)]
        out[name] = got
    return out


def _exact_attend(s):
    c = s["c"]
    q = s["q"].double()
    B, N, HQ, D = q.shape
    H = c["kv_heads"]
    G = HQ // H
    parent = s["parent"].tolist()
    out = torch.zeros((B, N, HQ, D), dtype=torch.float64, device="cuda")
    lse = torch.zeros((B, N, HQ), dtype=torch.float64, device="cuda")
    for b, (n, used) in enumerate(zip(_lengths(c), _used(c))):
        sees = torch.zeros((used, used), dtype=torch.bool, device="cuda")
        for i in range(used):
            j = i
            while j >= 0:
                sees[i, j] = True
                j = parent[b][j]
        block = torch.arange(n, device="cuda") // BLOCK
        for h in range(H):
            heads = slice(h * G, (h + 1) * G)
            k, v = (torch.cat([s[x][b, :n, h].double() * torch.exp2(s[x + "_exp"][b, h].double() - 127)[block, None],
                               s["fresh_" + x][b, :used, h].double()]) for x in "kv")
            dots = (q[b, :used, heads].reshape(-1, D) @ k.T.contiguous() / math.sqrt(D)).view(used, G, -1)
            dots[:, :, n:].masked_fill_(~sees[:, None], -math.inf)
            lse[b, :used, heads] = dots.logsumexp(-1)
            out[b, :used, heads] = dots.softmax(-1) @ v
    return {"out": out, "lse": lse}
