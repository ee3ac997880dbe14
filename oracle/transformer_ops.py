"""64-bit restatement of the transformer-block operators (dropout, norm_residual, gated_linear): values, gradients, and for every
output a bound on what f32 arithmetic over inputs of the map's type may be off by (the sums of absolute terms that rounding errors scale
with).  CPU only; written from the formulas."""
import math

import numpy as np
import torch

U32 = 2.0 ** -24                             # half a step of f32


def philox4x32(counter, key, rounds=10):
    """Philox4x32 of the counters [n, 4] (uint64 arrays holding 32-bit words)"""
    c = [counter[:, i].astype(np.uint64) for i in range(4)]
    low, s = np.uint64(0xffffffff), np.uint64(32)
    for r in range(rounds):
        k0, k1 = np.uint64((key[0] + r * 0x9E3779B9) & 0xffffffff), np.uint64((key[1] + r * 0xBB67AE85) & 0xffffffff)
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> s) ^ c[1] ^ k0, b & low, (a >> s) ^ c[3] ^ k1, a & low]
    return np.stack(c, 1)


def keep_mask(n, threshold, seed, offset, first=0):
    """keep mask of the elements first .. first + n - 1"""
    q0, q1 = first // 8, (first + n + 7) // 8
    q = np.arange(q0, q1, dtype=np.uint64)
    cnt = np.stack([q & np.uint64(0xffffffff), q >> np.uint64(32), np.full_like(q, offset & 0xffffffff), np.full_like(q, offset >> 32)], 1)
    w = philox4x32(cnt, (seed & 0xffffffff, seed >> 32)).astype('<u4').view('<u2').reshape(-1)
    return torch.from_numpy(w[first - 8 * q0:first - 8 * q0 + n] >= threshold)


def threshold_of(p):
    return int(p * 65536 + 0.5)


def dropout(x, p, seed, offset):
    x, t = x.double(), threshold_of(p)
    return torch.where(keep_mask(x.numel(), t, seed, offset).view(x.shape), x / (1 - t / 65536) if t < 65536 else x, torch.zeros_like(x))


# ---- norm_residual --------------------------------------------------------------------------------------------------------
def _norm(v, w, b, layer, eps):
    c = v - v.mean(-1, keepdim=True) if layer else v
    r = 1 / (c.pow(2).mean(-1, keepdim=True) + eps).sqrt()
    return c * r * w + b, c * r, r


def _norm_back(g, hat, r, layer):
    d = g - hat * (g * hat).mean(-1, keepdim=True)
    return r * (d - g.mean(-1, keepdim=True) if layer else d)


def norm_residual(x, h, dy, dn, gate=None, scale=None, post=None, pre=None, layer=False, eps=1e-5, p=0.0, seed=0, offset=0):
    """maps [N, H, W, C] -> {name: (value, bound of the f32 error)}; dy, dn may be None.

    The bound: a row norm is a chain of at most 40 additions (eight channels a lane in up to four vectors, then six or eight halvings),
    one reciprocal root and a product, so a normalised row or a gradient through it is off by at most about 64 half steps of its largest
    term; post and pre follow each other and the gradient passes both again: 4 x 64 = 256 half steps of the largest value on the way."""
    x, C = x.double(), x.shape[-1]
    N = x.shape[0]
    one = torch.ones(C, dtype=torch.float64)
    zero = torch.zeros(C, dtype=torch.float64)
    par = lambda wb: [d if t is None else t.double() for t, d in zip(wb or (None, None), (one, zero))]
    (pw, pb), (qw, qb) = par(post), par(pre)
    f = (one if scale is None else scale.double()) * (torch.ones(N, 1, 1, C, dtype=torch.float64) if gate is None else gate.double().view(N, 1, 1, C))
    t = threshold_of(p)
    D = dropout(torch.ones_like(x), p, seed, offset) if t else torch.ones_like(x)
    out = {}
    unit = 256 * U32
    top = lambda *ts: unit * max([float(v.abs().max()) for v in ts if v.numel()] + [0.0])
    if h is None:
        hat = u = r = torch.zeros_like(x)
        y = x
    else:
        h = h.double()
        u, hat, r = _norm(h, pw, pb, layer, eps) if post else (h, h, None)
        y = x + f * torch.where(D > 0, u * D, torch.zeros_like(u))
        out['y'] = y, top(x, y, f * u * D)
    if pre:
        n, yhat, r2 = _norm(y, qw, qb, layer, eps)
        # an error of y is magnified by the reciprocal deviation
        out['n'] = n, top(n, yhat * qw, y.abs() * r2 * qw.abs().max())
    tt = torch.zeros_like(x)
    if dn is not None:
        dn = dn.double()
        tt = tt + _norm_back(dn * qw, yhat, r2, layer)
        out['pre_w'], out['pre_b'] = ((dn * yhat).sum((0, 1, 2)), unit * (dn * yhat).abs().sum((0, 1, 2)).max() + top(y.abs() * r2) * dn.abs().sum((0, 1, 2)).max()), \
            (dn.sum((0, 1, 2)), unit * dn.abs().sum((0, 1, 2)).max())
    if dy is not None:
        tt = tt + dy.double()
    if dy is None and dn is None:
        return out
    grow = top(tt, *([dn * qw * r2, y.abs() * r2 * tt.abs().max()] if dn is not None else []))      # bound of the error of tt
    out['x'] = tt, grow
    if h is None:
        return out
    rel = grow / max(float(tt.abs().max()), 1e-300)
    d = torch.where(D > 0, tt * D, torch.zeros_like(tt))
    du = d * f
    term = d * u
    out['gate'] = (term * (one if scale is None else scale.double())).sum((1, 2)), 4 * rel * float(((d.abs().amax() * u.abs()) * (1 if scale is None else scale.double().abs())).sum((1, 2)).max())
    out['scale'] = (term * (1 if gate is None else gate.double().view(N, 1, 1, C))).sum((0, 1, 2)), \
        4 * rel * float((d.abs().amax() * u.abs() * (1 if gate is None else gate.double().abs().view(N, 1, 1, C))).sum((0, 1, 2)).max())
    if post:
        out['post_w'] = (du * hat).sum((0, 1, 2)), 4 * rel * float(du.abs().max() * hat.abs().sum((0, 1, 2)).max())
        out['post_b'] = du.sum((0, 1, 2)), 4 * rel * float(du.abs().max() * x.shape[0] * x.shape[1] * x.shape[2])
        g = _norm_back(du * pw, hat, r, layer)
        out['h'] = g, 4 * rel * float((du.abs().max() * pw.abs().max() * r.max() * (1 + hat.abs().max())))
    else:
        out['h'] = du, 4 * rel * float(du.abs().max())
    return out


# ---- gated_linear ----------------------------------------------------------------------------------------------------------
def act(g, name):
    """activation, derivative, bound of the second derivative"""
    if name == 'relu':
        return g.clamp(min=0), (g > 0).to(g.dtype), 0.0
    if name == 'gelu':
        phi = 0.5 * torch.erfc(-g * math.sqrt(0.5))
        return g * phi, phi + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi), 0.8      # |phi''| <= 2 phi(0) = 0.798
    s = torch.sigmoid(g)
    return (s, s * (1 - s), 0.1) if name == 'sigmoid' else (g * s, s * (1 + g * (1 - s)), 0.5)


def gated_linear(x, wg, wu, bg, bu, dz, name, half):
    """x [M, K]; half: half a step of the map's type, relative (the backward pass rounds dg and du to it) -> {name: (value, bound)}.

    A dot product of n terms in f32 is off by at most (n + 2) half steps of the sum of absolute terms, whatever the order; the
    activation and its derivative are composed of a few operations of 1-2 ulp each: 16 half steps."""
    x, wg, wu = x.double(), wg.double(), wu.double()
    K, F, M = x.shape[1], wg.shape[0], x.shape[0]
    b = lambda t: torch.zeros(F, dtype=torch.float64) if t is None else t.double()
    g, u = x @ wg.t() + b(bg), x @ wu.t() + b(bu)
    eg, eu = ((K + 2) * U32 * (x.abs() @ w.abs().t() + b(t).abs()) for w, t in ((wg, bg), (wu, bu)))
    a, da, curve = act(g, name)
    ea = da.abs() * eg + 0.5 * curve * eg ** 2 + 16 * U32 * (a.abs() + g.abs() * da.abs() + (1e-30 if name == 'relu' else 0.3))
    out = {'z': (a * u, ea * u.abs() + (a.abs() + ea) * eu + 2 * U32 * (a * u).abs())}
    if dz is None:
        return out
    dz = dz.double()
    eda = curve * eg + 16 * U32 * (da.abs() + 0.3) + ((g.abs() <= eg).double() if name == 'relu' else 0)      # (relu: the step may fall either way)
    dg, du = dz * u * da, dz * a
    edg = dz.abs() * (u.abs() * eda + (da.abs() + eda) * eu) + 4 * U32 * dg.abs()
    edu = dz.abs() * ea + 4 * U32 * du.abs()
    rg, ru = edg + half * (dg.abs() + edg), edu + half * (du.abs() + edu)
    out['x'] = dg @ wg + du @ wu, rg @ wg.abs() + ru @ wu.abs() + (2 * F + 18) * U32 * (dg.abs() @ wg.abs() + du.abs() @ wu.abs())
    out['wg'] = dg.t() @ x, rg.t() @ x.abs() + (M + 2) * U32 * (dg.abs().t() @ x.abs())
    out['wu'] = du.t() @ x, ru.t() @ x.abs() + (M + 2) * U32 * (du.abs().t() @ x.abs())
    out['bg'] = dg.sum(0), edg.sum(0) + (M + 2) * U32 * dg.abs().sum(0)
    out['bu'] = du.sum(0), edu.sum(0) + (M + 2) * U32 * du.abs().sum(0)
    return out
