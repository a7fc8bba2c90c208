"""Plain 64-bit forms of the sequence operators, with elementwise bounds on what a kernel in fp32 arithmetic may be off.

u = half a step of the element type (eps / 2), f = 2^-24 that of fp32.  Sums of n products in fp32 are off by at most
n f times the sum of their magnitudes; products of bf16 values are exact in fp32.  A score s = scale q.k is then off by
(D + 4) f (scale |q|.|k|), and its exponential relative to the row's maximum by twice the largest such error of the row
(numerator and maximum / denominator), plus 8 f for exp2, logarithm and the scaled difference's own rounding, which
grows with |s| log2(e): 4 f max|s|."""
import math

import torch

F = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def attention(q, k, v, causal, mask, scale, dout=None):
    """{name: (value, bound)} of out and, with dout, of dq, dk, dv; all arguments in their element type."""
    u = half_step(q.dtype)
    Z, Lq, H, D = q.shape
    Lk, KVH = k.shape[1], k.shape[2]
    G = H // KVH
    q64, k64, v64 = (x.detach().cpu().double() for x in (q, k, v))
    vis = torch.ones(Z, Lq, Lk, dtype=torch.bool)
    if causal:
        vis &= torch.arange(Lk)[None, None] <= torch.arange(Lq)[None, :, None] + (Lk - Lq)
    if mask is not None:
        vis &= mask.cpu().bool()[:, None]
        hidden = ~mask.cpu().bool()
        k64 = k64.masked_fill(hidden[:, :, None, None], 0.0)
        v64 = v64.masked_fill(hidden[:, :, None, None], 0.0)
    q64 = q64.transpose(1, 2)                                              # [Z, H, Lq, D]
    k64, v64 = (x.transpose(1, 2).repeat_interleave(G, 1) for x in (k64, v64))
    vis = vis[:, None]
    kt = k64.transpose(-1, -2)
    s = (q64 @ kt) * scale
    sa = ((q64.abs() @ kt.abs()) * scale).masked_fill(~vis, 0.0)
    top = sa.amax(-1, keepdim=True) if Lk else torch.zeros(Z, H, Lq, 1, dtype=torch.float64)
    eps = 2 * (D + 4) * F * top + 8 * F + 4 * F * top                      # of a probability, relative
    s = s.masked_fill(~vis, -math.inf)
    m = s.amax(-1, keepdim=True).clamp_min(-1e300) if Lk else top
    e = torch.exp(s - m)
    p = e / e.sum(-1, keepdim=True).clamp_min(1e-300)
    eps = eps + Lk * F                                                     # the sum of the row
    out = p @ v64
    out_b = (p @ v64.abs()) * (u + eps + Lk * F) + u * out.abs()
    got = {"out": (out.transpose(1, 2), out_b.transpose(1, 2))}
    if dout is None:
        return got
    do = dout.detach().cpu().double().transpose(1, 2)
    shared = lambda x: x.view(Z, KVH, G, Lk, D).sum(2).transpose(1, 2)     # noqa: E731
    n = Lq * G * F
    dv, dv_b = p.transpose(-1, -2) @ do, (p * (u + eps + n)).transpose(-1, -2) @ do.abs()
    delta = (do * out).sum(-1, keepdim=True)
    delta_b = (do.abs() * out_b).sum(-1, keepdim=True) + D * F * (do * out).abs().sum(-1, keepdim=True)
    vt = v64.transpose(-1, -2)
    dp = do @ vt
    ds = p * (dp - delta)
    ds_b = ds.abs() * (u + eps) + p * (2 * D * F * (do.abs() @ vt.abs()) + delta_b + F * (dp.abs() + delta.abs()))
    dq = (ds @ k64) * scale
    dq_b = ((ds_b + ds.abs() * Lk * F) @ k64.abs()) * scale
    qa = q64.abs()
    dk = (ds.transpose(-1, -2) @ q64) * scale
    dk_b = ((ds_b + ds.abs() * n).transpose(-1, -2) @ qa) * scale
    dk, dk_b, dv, dv_b = (shared(x) for x in (dk, dk_b, dv, dv_b))
    dq, dq_b = dq.transpose(1, 2), dq_b.transpose(1, 2)
    for name, x, b in (("dq", dq, dq_b), ("dk", dk, dk_b), ("dv", dv, dv_b)):
        got[name] = (x, b + 2 * u * x.abs())
    return got


def beam_step(q, prefixes, kgen, vgen, anc, t, beam, scale):
    """(value, bound) of one new token per hypothesis over its prefixes, its ancestors' positions and its own."""
    u = half_step(q.dtype)
    M, H, D = q.shape
    KVH = kgen.shape[2]
    G = H // KVH
    out, bound = torch.zeros(M, H, D, dtype=torch.float64), torch.zeros(M, H, D, dtype=torch.float64)
    c = lambda x: x.detach().cpu().double()                                # noqa: E731
    q, kgen, vgen = c(q), c(kgen), c(vgen)
    levels = [(c(p[0]), c(p[1]), p[2].cpu().tolist() if len(p) == 3 else None) for p in prefixes]
    anc = None if anc is None else anc.cpu().long()
    for m in range(M):
        slots = [(s, m // beam * beam + int(anc[s, m])) for s in range(t)] + [(t, m)]
        for h in range(KVH):
            ks = [torch.stack([kgen[s, i, h] for s, i in slots])]
            vs = [torch.stack([vgen[s, i, h] for s, i in slots])]
            for k, v, lens in levels:
                g = m // (M // k.shape[0])
                n = k.shape[2] if lens is None else min(max(lens[g], 0), k.shape[2])
                ks.append(k[g, h, :n])
                vs.append(v[g, h, :n])
            kk, vv = torch.cat(ks), torch.cat(vs)
            qq = q[m, h * G:(h + 1) * G]
            s = qq @ kk.t() * scale
            top = (qq.abs() @ kk.abs().t() * scale).amax(-1, keepdim=True)
            p = torch.softmax(s, -1)
            eps = 2 * (D + 4) * F * top + 8 * F + 4 * F * top + 2 * kk.shape[0] * F
            o = p @ vv
            out[m, h * G:(h + 1) * G] = o
            bound[m, h * G:(h + 1) * G] = (p @ vv.abs()) * (u + eps) + u * o.abs()
    return out, bound


def add_rms_norm(x, delta, w, eps, dx_out, dh):
    """{name: (value, bound)}: the sum as it is stored, the normed row, and the gradients."""
    u = half_step(x.dtype)
    c = lambda t: t.detach().cpu().double()                                # noqa: E731
    xs = c(x) if delta is None else c((x.detach().float() + delta.detach().float()).to(x.dtype))
    w64, n = c(w), x.shape[-1]
    r = torch.rsqrt(xs.square().mean(-1, keepdim=True) + eps)
    xh = xs * r
    h = w64 * xh
    re = (n + 8) * F                                                       # r, relative: the sum of squares, rsqrt
    got = {"x_out": (xs, torch.zeros_like(xs)), "h": (h, h.abs() * (2 * u + u * u + 2 * re))}
    go = torch.zeros_like(xs) if dx_out is None else c(dx_out)
    dh = c(dh)
    g = dh * w64
    mean, mean_a = (g * xh).mean(-1, keepdim=True), (g * xh).abs().mean(-1, keepdim=True)
    dx = go + r * (g - xh * mean)
    dx_b = r * (g.abs() * 2 * re + xh.abs() * mean_a * 4 * re) + 4 * F * (go.abs() + r * (g.abs() + xh.abs() * mean_a))
    rows = max(1, xs.numel() // n)
    dw = (dh * xh).reshape(-1, n).sum(0)
    dw_b = (dh * xh).abs().reshape(-1, n).sum(0) * (rows * F + 2 * re)
    got["dx"] = (dx, dx_b + u * (dx.abs() + dx_b))
    got["dw"] = (dw, dw_b + u * (dw.abs() + dw_b))
    return got


def within(got, want, what):
    value, bound = want
    got = got.detach().cpu().double()
    assert got.shape == value.shape, (what, got.shape, value.shape)
    assert bool(torch.isfinite(got).all()), f"{what}: not finite"
    tiny = 1e-37                                                           # results below the normal range
    over = ((got - value).abs() - bound - tiny)
    assert float(over.max() if over.numel() else -1.0) <= 0.0, \
        (what, float((got - value).abs().max()), float(((got - value).abs() / (bound + tiny)).max()))
