"""The definitions of qk_rotate, prompt_attend, cache_append8 and the 8-bit cache's values in
64 bits on the CPU, with bounds on how far f32 sums and roundings may be off."""
import math

import torch

from tests.treeref import F32, half_step

BLOCK = 32
EXP_MIN = -100


def rotate(x, w, eps, pos, inv_freq, neighbours):
    """(y, tolerance) of [tokens, heads, size], f64.  Relative to a norm's outputs, f32 leaves the
    sum of size squares (size + 8 half steps, halved by the root), the root, the quotient and two
    products; a cosine is off by the rounding of its angle in half turns (2^-25, so pi times that)
    and two steps of its own, 6 half steps in all, and by the f64 angle's three roundings; a pair's
    two products and their sum are three half steps more; the output is rounded once."""
    dtype = x.dtype
    x = x.double().cpu()
    T, H, D = x.shape
    rel = 0.0
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double().cpu()
        rel = (D / 2 + 12) * F32
    y = x.clone()
    size = x.abs().clone()
    extra = torch.zeros(T, 1, D, dtype=torch.float64)
    if inv_freq is not None:
        r = 2 * inv_freq.numel()
        t = pos.double().cpu()[:, None] * inv_freq.double().cpu()
        a, b = (x[..., 0:r:2], x[..., 1:r:2]) if neighbours else (x[..., :r // 2], x[..., r // 2:r])
        c, s = t.cos()[:, None], t.sin()[:, None]
        # (cos and sin of an f64 angle of 2^31 are as exact as the angle)
        off = 3 * 2.0**-53 * t.abs()[:, None]
        for i, (z, e) in enumerate(((a * c - b * s, 0), (b * c + a * s, 1))):
            at = (slice(i, r, 2) if neighbours else slice(i * (r // 2), (i + 1) * (r // 2)))
            y[..., at] = z
            size[..., at] = a.abs() + b.abs()
            extra[..., at] = 9 * F32 + 2 * off
    tol = half_step(dtype) * y.abs() * 1.01 + size * (rel + extra) * 1.01 + 1e-38
    if dtype == torch.float16:
        tol += 2.0**-25
    return y, tol


def prompt(q, k, v, start, scale):
    """(out, lse, out tolerance, lse tolerance) of packed prompts; rows of no sequence are NaN.  The
    tolerances are treeref.attend's."""
    T, HQ, D = q.shape
    H = k.shape[1]
    dtype = q.dtype
    u = half_step(dtype)
    q, k, v = (t.double().cpu() for t in (q, k, v))
    out = torch.full((T, HQ, D), math.nan, dtype=torch.float64)
    lse = torch.full((T, HQ), math.nan, dtype=torch.float64)
    tol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
    for first, last in zip(start, start[1:]):
        for h in range(HQ):
            kh, vh = k[first:last, h // (HQ // H)], v[first:last, h // (HQ // H)]
            for i in range(first, last):
                n = i - first + 1
                s = kh[:n] @ q[i, h] * scale
                if bool((s == -math.inf).all()):
                    out[i, h], lse[i, h] = 0.0, -math.inf
                    continue
                p = torch.softmax(s, 0)
                live = (p > 0) | ~torch.isfinite(p)
                out[i, h] = p[live] @ vh[:n][live]
                lse[i, h] = math.nan if bool((s == math.inf).any()) else torch.logsumexp(s, 0)
                off = (D + 4) * F32 * float((kh[:n].abs() @ q[i, h].abs()).nan_to_num(0, 0, 0).max()) * abs(scale)
                off += 8 * F32 * (1 + float(s.abs().nan_to_num(0, 0, 0).max()))
                around = p[live] @ vh[:n][live].abs()
                tol[i, h] = u * out[i, h].abs() * 1.01 + around * (u * 1.01 + 2 * off + 2 * (n + 8) * F32)
                if dtype == torch.float16:
                    tol[i, h] += 2.0**-25 * (1 + n)
                ltol[i, h] = off + (n + 8) * F32 + 4 * F32 * abs(float(lse[i, h]))
    return out, lse, tol, ltol


def agree(got_out, got_lse, want, left=None):
    """got against prompt()'s or treeref.attend()'s results; rows that are NaN there in out and lse
    with no tolerance are those of no sequence, which hold `left`."""
    out, lse, tol, ltol = want
    o, s = got_out.double().cpu(), got_lse.double().cpu()
    none = torch.isnan(lse) & (ltol == 0) & (tol.amax(-1) == 0)
    if left is not None:
        assert bool((o[none] == left).all()) and bool((s[none] == left).all())
    empty = lse == -math.inf
    assert bool((s[empty] == -math.inf).all()) and bool((o[empty] == 0.0).all())
    rest = ~empty & ~none
    x, y, t = o[rest], out[rest], tol[rest]
    assert bool((torch.isnan(x) == torch.isnan(y)).all())
    fine = torch.isfinite(y)
    assert bool((x[~fine & ~torch.isnan(y)] == y[~fine & ~torch.isnan(y)]).all())
    worst = ((x - y).abs() / t.clamp(min=1e-300))[fine]
    assert worst.numel() == 0 or float(worst.max()) <= 1.0, float(worst.max())
    x, y, t = s[rest], lse[rest], ltol[rest]
    assert bool((torch.isnan(x) == torch.isnan(y)).all())
    fine = torch.isfinite(y)
    assert bool(((x - y).abs()[fine] <= t[fine]).all())


def nearest_e4m3(x):
    """The e4m3 nearest to each x of |x| <= 448 (f64), ties to even; what is not finite is NaN."""
    step = torch.exp2(torch.frexp(x).exponent.double().clamp(min=-5) - 4)
    return torch.where(torch.isfinite(x), torch.round(x / step) * step, math.nan)


def exponent(most):
    """The least e >= EXP_MIN with most <= 448 * 2^e."""
    e = EXP_MIN
    while most > 448.0 * 2.0**e:
        e += 1
    return e


class Cache:
    """What an 8-bit cache stands for, appended to row by row in 64 bits: k, v [seqs, slots, heads,
    size] e4m3 values and their exponents [seqs, heads, blocks]."""

    def __init__(self, k, v, k_exp, v_exp, lens):
        self.byte = [t.double().cpu().clone() for t in (k, v)]
        self.exp = [t.int().cpu().clone() - 127 for t in (k_exp, v_exp)]
        self.lens = list(lens)

    def append(self, b, rows_k, rows_v):
        n, m = self.lens[b], rows_k.shape[0]
        H = rows_k.shape[1]
        for byte, exp, rows in zip(self.byte, self.exp, (rows_k, rows_v)):
            rows = rows.double().cpu()
            for j in range(n // BLOCK, (n + m + BLOCK - 1) // BLOCK):
                lo, hi = max(n, j * BLOCK), min(n + m, (j + 1) * BLOCK)
                had = lo > j * BLOCK
                for h in range(H):
                    x = rows[lo - n:hi - n, h]
                    fin = x[torch.isfinite(x)]
                    e = exponent(float(fin.abs().max()) if fin.numel() else 0.0)
                    if had:
                        old = int(exp[b, h, j])
                        e = max(e, old)
                        if e != old:
                            part = byte[b, j * BLOCK:lo, h]
                            byte[b, j * BLOCK:lo, h] = nearest_e4m3(part * 2.0**(old - e))
                    byte[b, lo:hi, h] = nearest_e4m3(x * 2.0**-e)
                    exp[b, h, j] = e
        self.lens[b] = n + m

    def values(self):
        """(k, v) f64, the values that the bytes stand for."""
        out = []
        for byte, exp in zip(self.byte, self.exp):
            cap = byte.shape[1]
            out.append(byte * torch.exp2(exp.double()).repeat_interleave(BLOCK, 2)[:, :, :cap].transpose(1, 2)[..., None])
        return out

    def check(self, k, v, k_exp, v_exp):
        """The device's cache holds the same, bit for bit but for the sign of NaN."""
        for byte, exp, t, e in zip(self.byte, self.exp, (k, v), (k_exp, v_exp)):
            for b, n in enumerate(self.lens):
                blocks = (n + BLOCK - 1) // BLOCK
                assert bool((e[b, :, :blocks].int().cpu() - 127 == exp[b, :, :blocks]).all()), b
            x = t.double().cpu()
            same = (x == byte) | (torch.isnan(x) & torch.isnan(byte))
            assert bool(same.all()), same.logical_not().nonzero()[:4].tolist()


def prompt_wide(q, k, v, start, scale):
    """prompt() of finite inputs on the device, a head's whole square of scores at a time."""
    T, HQ, D = q.shape
    H = k.shape[1]
    u = half_step(q.dtype)
    out = torch.full((T, HQ, D), math.nan, dtype=torch.float64)
    lse = torch.full((T, HQ), math.nan, dtype=torch.float64)
    tol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
    for first, last in zip(start, start[1:]):
        n = last - first
        if n == 0:
            continue
        seen = torch.ones((n, n), dtype=torch.bool, device=q.device).tril()
        count = torch.arange(1, n + 1, dtype=torch.float64, device=q.device)[:, None]
        for h in range(HQ):
            x, kh, vh = q[first:last, h].double(), k[first:last, h // (HQ // H)].double(), v[first:last, h // (HQ // H)].double()
            s = (x @ kh.T.contiguous() * scale).masked_fill_(~seen, -math.inf)
            p = s.softmax(-1)
            y, around, z = p @ vh, p @ vh.abs(), s.logsumexp(-1, keepdim=True)
            off = (D + 4) * F32 * ((x.abs() @ kh.abs().T.contiguous()) * seen).amax(-1, keepdim=True) * abs(scale)
            off = off + 8 * F32 * (1 + s.abs().masked_fill_(~seen, 0).amax(-1, keepdim=True))
            t = u * y.abs() * 1.01 + around * (u * 1.01 + 2 * off + 2 * (count + 8) * F32)
            if q.dtype == torch.float16:
                t = t + 2.0**-25 * (1 + count)
            out[first:last, h], lse[first:last, h], tol[first:last, h] = y.cpu(), z[:, 0].cpu(), t.cpu()
            ltol[first:last, h] = (off + (count + 8) * F32 + 4 * F32 * z.abs())[:, 0].cpu()
    return out, lse, tol, ltol
