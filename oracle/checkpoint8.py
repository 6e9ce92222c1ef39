"""64-bit oracle of the 8-bit activation checkpoints and of the fused block norm (test infrastructure, CPU, elementwise
definitions with no shared code with the kernels)."""
import math

import torch

D = torch.float64
GROUP, BIAS, LOWEST, HIGHEST = 32, 127, 10, 246

# every finite e4m3 magnitude, in the order of its code
MAGNITUDES = torch.tensor([m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)], dtype=D)[:127]


def encode(x):
    """(codes uint8, scales uint8) of a (..., C) map."""
    c = x.shape[-1]
    v = x.to(D)
    finite = torch.isfinite(v)
    codes, scales = [], []
    for lo in range(0, c, GROUP):
        g, ok = v[..., lo:lo + GROUP], finite[..., lo:lo + GROUP]
        top = torch.where(ok, g.abs(), 0.0).amax(-1, keepdim=True)
        # smallest e with top <= 448 * 2^e, up to the one whose largest value is the largest below 2^128
        e = torch.full_like(top, LOWEST - BIAS)
        for k in range(LOWEST - BIAS, HIGHEST - BIAS):
            e = torch.where(top > 448.0 * 2.0 ** k, float(k + 1), e)
        y = torch.where(ok, g.abs(), 0.0) * torch.pow(torch.tensor(2.0, dtype=D), -e)
        # nearest magnitude, ties to the even code; what is not 0 stays so
        y = y.clamp(max=448.0)
        i = torch.searchsorted(MAGNITUDES, y.contiguous())
        below = (i - 1).clamp(min=0)
        d_up, d_dn = MAGNITUDES[i] - y, y - MAGNITUDES[below]
        code = torch.where(d_up < d_dn, i, torch.where(d_up > d_dn, below, torch.where(i % 2 == 0, i, below)))
        code = torch.where((g != 0) & (code == 0), 1, code)
        code = torch.where(ok, code, 127)
        code = code + 128 * torch.signbit(g).long()
        codes.append(code)
        scales.append(e + BIAS)
    return torch.cat(codes, -1).to(torch.uint8), torch.cat(scales, -1).to(torch.uint8)


def decode(codes, scales):
    code = codes.long()
    mag = MAGNITUDES[(code & 127).clamp(max=126)]
    mag = torch.where(code & 127 == 127, math.nan, mag)
    s = torch.pow(torch.tensor(2.0, dtype=D), scales.to(D) - BIAS).repeat_interleave(GROUP, -1)[..., :code.shape[-1]]
    return torch.where(code >= 128, -mag, mag) * s


def _norm(v, wb, kind, eps):
    mean = v.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(v[..., :1])
    rstd = (((v - mean) ** 2).mean(-1, keepdim=True) + eps) ** -0.5
    hat = (v - mean) * rstd
    out = hat * wb[0]
    return hat, rstd, out if wb[1] is None else out + wb[1]


def _gate(gate, x, act):
    if gate is None:
        return torch.ones((), dtype=D)
    g = gate.to(D)
    if g.shape != x.shape and g.dim() == 2:
        g = g.view((g.shape[0],) + (1,) * (x.dim() - 2) + (g.shape[1],))
    return torch.sigmoid(g) if act == "sigmoid" else g


def _wide(wb):
    return None if wb is None else tuple(None if t is None else t.to(D) for t in wb)


def norm_residual(x, h, post, gate, scale, pre, kind, act, eps=1e-6):
    """(r, n) and how large the terms are whose rounding they carry (r's, n's)."""
    x, post, pre = x.to(D), _wide(post), _wide(pre)
    r, mag = x, x.abs()
    if h is not None:
        p, pm = h.to(D), h.to(D).abs()
        if post is not None:
            hat, rstd, p = _norm(p, post, kind, eps)
            # a row's mean and variance carry errors in units of its largest value
            pm = (hat.abs() + 1) * (1 + pm.amax(-1, keepdim=True) * rstd) * post[0].abs() + (0 if post[1] is None else post[1].abs())
        g = _gate(gate, x, act)
        r = x + float(scale) * g * p
        mag = x.abs() + abs(float(scale)) * g.abs() * pm
    if pre is None:
        return (r, None), (mag, None)
    hat, rstd, n = _norm(r, pre, kind, eps)
    nm = (hat.abs() + 1) * (1 + mag.amax(-1, keepdim=True) * rstd) * pre[0].abs() + (0 if pre[1] is None else pre[1].abs())
    return (r, n), (mag, nm)


def norm_residual_bwd(h, r, dr, dn, post, gate, scale, pre, kind, act, learned, eps=1e-6):
    """dicts of the gradients and of the sizes of the terms that they are sums of."""
    post, pre = _wide(post), _wide(pre)
    like = dr if dr is not None else dn
    rows = tuple(range(like.dim() - 1))
    layer = kind == "layer"
    out, size = {}, {}

    def through(v, d, dsize, wb):
        hat, rstd, _ = _norm(v, wb, kind, eps)
        cond = 1 + v.abs().amax(-1, keepdim=True) * rstd
        u, us = d * wb[0], dsize * wb[0].abs()
        dv = rstd * (u - (u.mean(-1, keepdim=True) if layer else 0.0) - hat * (u * hat).mean(-1, keepdim=True))
        vs = rstd * cond * (us + us.mean(-1, keepdim=True) + hat.abs() * (us * hat.abs()).mean(-1, keepdim=True))
        return hat, cond, dv, vs, (d * hat).sum(rows), (dsize * (hat.abs() + 1) * cond).sum(rows), d.sum(rows), dsize.sum(rows)

    d = torch.zeros_like(like, dtype=D) if dr is None else dr.to(D)
    ds = d.abs()
    if pre is not None:
        _, _, dv, vs, out["dpre_weight"], size["dpre_weight"], out["dpre_bias"], size["dpre_bias"] = through(r.to(D), dn.to(D), dn.to(D).abs(), pre)
        d, ds = d + dv, ds + vs
    out["dx"], size["dx"] = d, ds
    if h is not None:
        g, s = _gate(gate, like, act), float(scale)
        p = h.to(D)
        ps = p.abs()
        dp, dps = s * g * d, abs(s) * g.abs() * ds
        out["dh"], size["dh"] = dp, dps
        if post is not None:
            hat, cond, out["dh"], size["dh"], out["dpost_weight"], size["dpost_weight"], out["dpost_bias"], size["dpost_bias"] = through(p, dp, dps, post)
            b = 0.0 if post[1] is None else post[1]
            p, ps = hat * post[0] + b, (hat.abs() + 1) * cond * post[0].abs() + abs(b)
        if gate is not None:
            f = g * (1 - g) if act == "sigmoid" else torch.ones((), dtype=D)
            dg, dgs = s * d * p * f, abs(s) * ds * ps * f
            if gate.shape != like.shape:
                over = rows if gate.dim() == 1 else tuple(range(1, like.dim() - 1))
                dg, dgs = dg.sum(over), dgs.sum(over)
            out["dgate"], size["dgate"] = dg, dgs
        if learned:
            out["dscale"], size["dscale"] = (d * g * p).sum(), (ds * g.abs() * ps).sum()
    for name, wb in (("dpost_bias", post), ("dpre_bias", pre)):
        if wb is not None and wb[1] is None:
            out.pop(name, None)
    return out, size
