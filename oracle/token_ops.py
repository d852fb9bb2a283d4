"""Float64 CPU restatement of the token operators (wst_amd.tokens), from their formulas, with bounds on the rounding
that the operators' own arithmetic may cause.

Bounds count, to first order: U32 = 2^-24 a rounding of a float32 operation (a sum of m terms at most m of them, fused
or not, of the sum of magnitudes), half(t) = eps(t) / 2 a rounding to type t.  Every function returns (value, bound)
pairs; |operator - value| <= bound is what the tests hold.
"""
import math

import torch

U32 = 2.0 ** -24
F64 = torch.float64


def half(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """What a rounding may lose below the type's normal numbers."""
    return torch.finfo(dtype).tiny * torch.finfo(dtype).eps


def layer_norm(x, weight, bias, eps, out_dtype, dy=None):
    """x (rows, n). Returns {"y": (value, bound)} and with dy also dx, dw, db."""
    x_dtype = x.dtype
    x = x.to(F64)
    rows, n = x.shape
    w = torch.ones(n, dtype=F64) if weight is None else weight.to(F64)
    b = torch.zeros(n, dtype=F64) if bias is None else bias.to(F64)
    mu = x.mean(1, keepdim=True)
    var = ((x - mu) ** 2).mean(1, keepdim=True)
    r = (var + eps) ** -0.5
    h = (x - mu) * r
    y = h * w + b
    # sums: a lane adds n / 64 values or fewer, six or more steps join lanes: m roundings of the magnitudes' sum
    m = n / 64 + 20
    e_mu = m * U32 * x.abs().mean(1, keepdim=True)
    # x - mu: the mean's error and one rounding; relative error of r: half that of the variance, whose terms carry twice
    # that of x - mu
    e_d = e_mu + U32 * (x - mu).abs()
    e_r = (m + 8) * U32 + ((x - mu).abs() * e_d).mean(1, keepdim=True) / (var + eps)
    e_h = e_d * r + h.abs() * (e_r + 2 * U32)
    out = {"y": (y, half(out_dtype) * y.abs() + tiny(out_dtype) + e_h * w.abs() + 4 * U32 * ((h * w).abs() + b.abs()))}
    if dy is None:
        return out
    dy = dy.to(F64)
    g = dy * w
    c1, c2 = g.mean(1, keepdim=True), (g * h).mean(1, keepdim=True)
    dx = r * (g - c1 - h * c2)
    e_c1 = (m + 2) * U32 * g.abs().mean(1, keepdim=True)
    e_c2 = ((m + 3) * U32 * (g * h).abs() + g.abs() * e_h).mean(1, keepdim=True)
    size = g.abs() + c1.abs() + (h * c2).abs()
    e_dx = r * (e_c1 + h.abs() * e_c2 + e_h * c2.abs() + (e_r + 6 * U32) * size)
    out["dx"] = (dx, half(x_dtype) * dx.abs() + tiny(x_dtype) + e_dx)
    # sums over rows: a thread walks its rows, groups and threads are joined after
    k = rows + 40
    wt = torch.float32 if weight is None else weight.dtype
    dw, db = (dy * h).sum(0), dy.sum(0)
    out["dw"] = (dw, half(wt) * dw.abs() + tiny(wt) + (k * U32 * (dy * h).abs() + dy.abs() * e_h).sum(0))
    bt = torch.float32 if bias is None else bias.dtype
    out["db"] = (db, half(bt) * db.abs() + tiny(bt) + k * U32 * dy.abs().sum(0))
    return out


def rotary(x, positions, sections, base, interleaved, inverse=False):
    """x (B, T, H, D), positions (B, T, A). Returns (value, bound)."""
    dtype = x.dtype
    x = x.to(F64)
    n = sum(sections)
    y = x.clone()
    bound = torch.zeros_like(x)
    p = 0
    for axis, count in enumerate(sections):
        for i in range(count):
            a = positions[..., axis].to(F64) * base ** (-i / count) * (-1.0 if inverse else 1.0)
            c, s = torch.cos(a)[..., None], torch.sin(a)[..., None]
            i0, i1 = (2 * p, 2 * p + 1) if interleaved else (p, p + n)
            x0, x1 = x[..., i0], x[..., i1]
            y[..., i0] = x0 * c - x1 * s
            y[..., i1] = x1 * c + x0 * s
            # the angle: float64 of a far position (2^-52 of it, a few times), and 2 pi of a rounded turn of at most a
            # half; sine and cosine within 2 ulp; two products and a sum
            e = (4 * 2.0 ** -52 * a.abs() + 2 * math.pi * U32 / 2 + 4 * U32)[..., None] + 3 * U32
            bound[..., i0] = bound[..., i1] = e * (x0.abs() + x1.abs())
            p += 1
    turned = torch.zeros_like(x)
    turned[..., :2 * n] = 1.0
    return y, bound + turned * (half(dtype) * y.abs() + tiny(dtype))


def seen(B, Tq, Tk, k_lengths=None, causal=False, prefix=None, q_documents=None, k_documents=None):
    """(B, Tq, Tk) truth values and place(i) - j (B, Tq, Tk)."""
    out = torch.zeros(B, Tq, Tk, dtype=torch.bool)
    away = torch.zeros(B, Tq, Tk, dtype=F64)
    for b in range(B):
        L = Tk if k_lengths is None else min(max(int(k_lengths[b]), 0), Tk)
        i = torch.arange(Tq)[:, None] + (L - Tq)
        j = torch.arange(Tk)[None]
        see = (j < L).expand(Tq, Tk)
        if causal or prefix is not None:
            ordered = j <= i
            if prefix is not None:
                ordered = ordered | (j < int(prefix[b]))
            see = see & ordered
        if q_documents is not None:
            qd = q_documents if q_documents.dim() == 1 else q_documents[b]
            kd = k_documents if k_documents.dim() == 1 else k_documents[b]
            see = see & (qd[:, None] == kd[None]) & (qd[:, None] >= 0)
        out[b], away[b] = see, (i - j).to(F64)
    return out, away


def attention(q, k, v, *, scale=None, cap=0.0, slopes=None, q_positions=None, k_positions=None, q_documents=None,
              k_documents=None, causal=False, prefix=None, k_lengths=None, do=None):
    """q (B, Tq, H, D), k, v (B, Tk, Hk, D) on the CPU. Returns {"o", "lse"[, "dq", "dk", "dv", "dslopes"]}, each a
    (value, bound) pair. What is not seen is cut out, so infinities and NaN there do not matter."""
    dtype = q.dtype
    u = half(dtype) if dtype != torch.float32 else 0.0       # weights and score gradients are rounded to 16-bit types
    B, Tq, H, D = q.shape
    Tk, Hk = k.shape[1:3]
    scale = D ** -0.5 if scale is None else scale
    see, away = seen(B, Tq, Tk, k_lengths, causal, prefix, q_documents, k_documents)
    z64 = lambda *s: torch.zeros(*s, dtype=F64)   # noqa: E731
    out = {n: (z64(*t.shape), z64(*t.shape)) for n, t in (("o", q), ("dq", q), ("dk", k), ("dv", v))}
    out["lse"] = (torch.full((B, H, Tq), -math.inf, dtype=F64), z64(B, H, Tq))
    out["dslopes"] = (z64(H), z64(H))
    for b in range(B):
        S = see[b]
        rows, cols = S.any(1), S.any(0)
        if slopes is not None:
            if q_positions is None:
                far = away[b].abs()
            else:
                qp = q_positions if q_positions.dim() == 2 else q_positions[b]
                kp = k_positions if k_positions.dim() == 2 else k_positions[b]
                far = (qp[:, None].to(F64) - kp[None].to(F64)).abs().sum(-1)
        for h in range(H):
            c = h // (H // Hk)
            # rows and keys that take part in nothing may hold anything
            Q = torch.where(rows[:, None], q[b, :, h].to(F64), 0.0)
            K = torch.where(cols[:, None], k[b, :, c].to(F64), 0.0)
            V = torch.where(cols[:, None], v[b, :, c].to(F64), 0.0)
            z = Q @ K.T * scale
            e = (D + 4) * U32 * (Q.abs() @ K.abs().T) * abs(scale)
            t = None
            if cap > 0:
                t = torch.tanh(z / cap)
                z = cap * t
                # tanh within a few roundings of one, times cap; in float32, and for caps beyond 64, of itself: 24 where
                # it is 1 - 2 / (e^2y + 1), so 8 of one from a third on and three times itself below, and fewer in its
                # series (the argument's two, the polynomial's few)
                near = u > 0 and cap <= 64
                e = e + 8 * U32 * cap * (1.0 if near else torch.clamp(3 * t.abs(), max=1.0))
            if slopes is not None:
                z = z - float(slopes[h]) * far
                e = e + 4 * U32 * (float(slopes[h]) * far).abs()
            e = e + 4 * U32 * z.abs()              # the exponent's own roundings
            z = torch.where(S, z, -math.inf)
            top = z.max(1, keepdim=True)[0]
            e = torch.where(S, e + 4 * U32 * torch.where(torch.isfinite(top), top, 0.0).abs(), 0.0)
            p = torch.where(S, torch.exp(z - torch.where(torch.isfinite(top), top, 0.0)), 0.0)
            total = p.sum(1, keepdim=True)
            p = torch.where(total > 0, p / total, 0.0)
            out["lse"][0][b, h] = torch.logsumexp(z, 1)
            e_row = (e.max(1, keepdim=True)[0]) * 2 + (Tk + 24) * U32   # of p, relative: its own and the sum's
            out["lse"][1][b, h] = (e_row + 4 * U32 * (1 + torch.where(torch.isfinite(top), top, 0.0).abs()))[:, 0]
            o = p @ V
            # a weight below float32's normal numbers may be taken for 0
            least = torch.where(S, torch.finfo(torch.float32).tiny, 0.0).to(F64)
            e_o = (u + e_row) * (p @ V.abs()) + least @ V.abs()
            out["o"][0][b, :, h] = o
            out["o"][1][b, :, h] = half(dtype) * o.abs() + e_o + tiny(dtype)
            if do is None:
                continue
            G = torch.where(rows[:, None], do[b, :, h].to(F64), 0.0)
            out["dv"][0][b, :, c] += p.T @ G
            out["dv"][1][b, :, c] += (p * (u + e_row + Tq * U32) + least).T @ G.abs()
            dp = G @ V.T
            delta = (p * dp).sum(1, keepdim=True)
            ds = p * (dp - delta)
            # delta is taken from the output and what rounding took from it
            e_delta = (G.abs() * (e_o + tiny(dtype) + (half(dtype) ** 2 + (2 * D + 8) * U32) * o.abs())).sum(1, keepdim=True)
            e_dp = (D + 4) * U32 * (G.abs() @ V.abs().T)
            e_ds = least * (dp.abs() + delta.abs()) + p * (e_dp + e_delta) + ds.abs() * (e_row + 4 * U32) + 2 * U32 * p * (dp.abs() + delta.abs())
            if slopes is not None:
                out["dslopes"][0][h] += -(ds * far).sum()
                out["dslopes"][1][h] += ((e_ds + (Tk + Tq + B * Tq) * U32 * ds.abs()) * far).sum()
            grad = torch.ones_like(z) if t is None else 1 - t * t
            dz = ds * grad * scale
            e_dz = e_ds * grad * abs(scale) + dz.abs() * (u + 4 * U32)
            if t is not None:
                # of 1 - t^2: t within its own roundings and the score's
                e_t = 12 * U32 + (1 - t * t) * e / cap
                e_dz = e_dz + 2 * e_t * ds.abs() * abs(scale)
            out["dq"][0][b, :, h] = dz @ K
            out["dq"][1][b, :, h] = (e_dz + Tk * U32 * dz.abs()) @ K.abs()
            out["dk"][0][b, :, c] += dz.T @ Q
            out["dk"][1][b, :, c] += (e_dz + Tq * (H // Hk) * U32 * dz.abs()).T @ Q.abs()
    for n in ("dq", "dk", "dv"):
        out[n] = (out[n][0], out[n][1] + half(dtype) * out[n][0].abs() + tiny(dtype))
    return out
