"""The tree calls' definitions in 64 bits on the CPU, one row at a time, with
bounds on how far f32 sums and roundings to the inputs' type may be off."""
import math

import numpy as np
import torch

F32 = 2.0**-24  # half a step of f32, relative


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def sees(parent, n):
    """List per node of what it sees of the tree (itself and its ancestors), or None
    where its chain of parents is broken."""
    out = []
    for i in range(n):
        chain, j = [], i
        while True:
            chain.append(j)
            p = int(parent[j])
            if p == -1:
                break
            if p < 0 or p >= j:
                chain = None
                break
            j = p
        out.append(chain)
    return out


def attend(q, k, v, lens, fk, fv, parent, used, scale):
    """(out, lse, out tolerance, lse tolerance), f64 [seqs, nodes, q heads(, size)]; rows that
    are not written are NaN.  The tolerances: a score's f32 dot product over size elements is off by
    at most (size + 4) F32 sum |q k| scale, so a weight by twice that (its own and the sum's), plus
    the f32 sums over the keys; then each weight is rounded to the type once, and the output once."""
    B, N, HQ, D = q.shape
    H = k.shape[2]
    dtype = q.dtype
    q, k, v, fk, fv = (t.double().cpu() for t in (q, k, v, fk, fv))
    out = torch.full((B, N, HQ, D), math.nan, dtype=torch.float64)
    lse = torch.full((B, N, HQ), math.nan, dtype=torch.float64)
    tol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
    u = half_step(dtype)
    for b in range(B):
        chains = sees(parent[b].tolist(), used[b])
        for h in range(HQ):
            g = h // (HQ // H)
            for i, chain in enumerate(chains):
                if chain is None:
                    out[b, i, h], lse[b, i, h] = 0.0, -math.inf
                    continue
                keys = torch.cat([k[b, :lens[b], g], fk[b, chain, g]])
                values = torch.cat([v[b, :lens[b], g], fv[b, chain, g]])
                s = keys @ q[b, i, h] * scale
                if bool((s == -math.inf).all()):
                    out[b, i, h], lse[b, i, h] = 0.0, -math.inf
                    continue
                p = torch.softmax(s, 0)
                live = p > 0
                live |= ~torch.isfinite(p)
                out[b, i, h] = p[live] @ values[live]
                lse[b, i, h] = math.nan if bool((s == math.inf).any()) else torch.logsumexp(s, 0)
                off = (D + 4) * F32 * float((keys.abs() @ q[b, i, h].abs()).nan_to_num(0, 0, 0).max()) * abs(scale)
                off += 8 * F32 * (1 + float(s.abs().nan_to_num(0, 0, 0).max()))
                n = len(s)
                around = p[live] @ values[live].abs()
                tol[b, i, h] = u * out[b, i, h].abs() * 1.01 + around * (u * 1.01 + 2 * off + 2 * (n + 8) * F32)
                if dtype == torch.float16:  # the least half step of float16, where it stops being relative
                    tol[b, i, h] += 2.0**-25 * (1 + n)
                ltol[b, i, h] = off + (n + 8) * F32 + 4 * F32 * abs(float(lse[b, i, h]))
    return out, lse, tol, ltol


def commit_mass(q, lse, k, lens, fk, path, m, scale, mass):
    """(new mass of slots [0, len + m), its tolerance) per sequence, f64 [kv heads, len + m]."""
    HQ, D = q.shape[2:]
    H = k.shape[2]
    G = HQ // H
    q, k, fk, lse, mass = (t.double().cpu() for t in (q, k, fk, lse, mass))
    out = []
    for b in range(q.shape[0]):
        n, mb = lens[b], m[b]
        w, t = torch.zeros((2, H, n + mb), dtype=torch.float64)
        for g in range(H):
            nodes = [int(x) for x in path[b][:mb]]
            keys = torch.cat([k[b, :n, g], fk[b, nodes, g]])
            for r, i in enumerate(nodes):
                for h in range(g * G, (g + 1) * G):
                    if float(lse[b, i, h]) == -math.inf:
                        continue
                    s = keys[:n + r + 1] @ q[b, i, h] * scale
                    e = (s - lse[b, i, h]).exp()
                    off = (D + 4) * F32 * (keys[:n + r + 1].abs() @ q[b, i, h].abs()) * abs(scale)
                    off = off + 8 * F32 * (1 + s.abs() + abs(float(lse[b, i, h])))
                    w[g, :n + r + 1] += e
                    t[g, :n + r + 1] += e * off
            t[g] += (G * mb + 2) * F32 * (w[g] + torch.cat([mass[b, g, :n].abs(), torch.zeros(mb, dtype=torch.float64)]))
            w[g, :n] += mass[b, g, :n]
        out.append((w, t))
    return out


def evict_sources(mass, pos, n, next_pos, keep, sinks, recent):
    """For one head: source[i] of the slot i of the cut cache (numpy, n > keep)."""
    order = sorted(range(n), key=lambda s: (
        0 if pos[s] < sinks or pos[s] >= next_pos - recent else 1,
        0.0 if pos[s] < sinks or pos[s] >= next_pos - recent else (math.inf if math.isnan(mass[s]) else -float(mass[s])),
        0 if pos[s] < sinks or pos[s] >= next_pos - recent else int(math.isnan(mass[s])),
        int(pos[s]), s))
    kept = np.zeros(n, bool)
    kept[order[:keep]] = True
    late = [s for s in range(keep, n) if kept[s]]
    source = list(range(keep))
    for s in range(keep):
        if not kept[s]:
            source[s] = late.pop(0)
    assert not late
    return source


def walk(token, status, tokens, parent, n, budget, eog, done):
    """One sequence's xs_verify_tree walk: (accepted, path, committed, status)."""
    acc, path, com, cur = 0, [], [], 0
    while n > 0 and len(com) < budget:
        if status[cur]:
            return acc, path, com, int(status[cur])
        t = int(token[cur])
        path.append(cur)
        com.append(t)
        child = [j for j in range(cur + 1, n) if parent[j] == cur and tokens[j] == t]
        if not child:
            break
        acc += 1
        if t in eog or done[child[0]]:
            break
        cur = child[0]
    return acc, path, com, 0
