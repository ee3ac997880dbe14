"""Cases of the transformer-style operators of rdfc_gan_amd.functional: dropout, norm_residual and gated_linear.

The maps are pixel-major [N, H, W, C]; a pixel is a token.  Sizes are those of this repository's networks: a 228 x 304 input gives maps of
228 x 304, 114 x 152, 57 x 76, 29 x 38 and 15 x 19 pixels with 64 to 512 channels, batches of 8 (16 stacked), pooling pyramids of 6 x 6 bins.

Definitions
  dropout        y[e] = x[e] / (1 - T / 65536) where word16(e) >= T, else 0;  T = round(65536 p)
                 e = ((n H + y) W + x) C + c;  word16(e) = 16-bit half e % 8 (low halves first) of the four 32-bit words that Philox4x32-10
                 (Salmon et al., SC 2011) gives for counter (e / 8, offset), key seed
  norm_residual  y = x + scale[c] * gate[n, c] * dropout(N_post(h)),  n = N_pre(y);  N: RMS norm or layer norm over the channels
  gated_linear   z = act(x Wg^T + bg) * (x Wu^T + bu)
"""
import math

import numpy as np
import torch

own = False

_DT = {'f32': torch.float32, 'f16': torch.float16, 'bf16': torch.bfloat16}
_EPS = 1e-5
_MOST_ELEMENTS = 16 * 228 * 304 * 64        # of a map of the largest listed memory-bound case
_MOST_FLOPS = 12.0 * 34656 * 256 * 1024     # of the largest listed product


def listed():
    return [
        # -- dropout, forward and backward
        # the encoders' bottleneck map: every launch counts
        dict(name='dropout-bottleneck', op='dropout', dtype='f16', N=8, H=15, W=19, C=512, ld=512, p=0.1),
        # a channel slice of a concatenated map in the f32 parity mode: odd width, rows that are not whole vectors
        dict(name='dropout-slice', op='dropout', dtype='f32', N=4, H=57, W=76, C=67, ld=131, p=0.25),
        # a full-resolution map of two stacked batches in a residual block with use_dropout
        dict(name='dropout-fullres', op='dropout', dtype='bf16', N=16, H=228, W=304, C=64, ld=64, p=0.5),
        # -- norm_residual
        # one pixel at inference: latency only
        dict(name='residual-pixel', op='residual', dtype='bf16', N=1, H=1, W=1, C=512, norm='rms', post=True, gate=True, scale=True, p=0.0, train=False),
        # an odd channel count in the f32 parity mode, layer norm, every gradient
        dict(name='residual-odd', op='residual', dtype='f32', N=3, H=15, W=19, C=301, norm='layer', post=True, gate=True, scale=True, p=0.0, train=True),
        # the trunk of the depth-to-RGB generator in training, gate per sample, dropout on the block's output
        dict(name='residual-trunk', op='residual', dtype='bf16', N=8, H=57, W=76, C=256, norm='rms', post=True, gate=True, scale=True, p=0.1, train=True),
        # a wide trunk in training: layer norm before the next block only, no dropout
        dict(name='residual-wide', op='residual', dtype='f16', N=8, H=57, W=76, C=1024, norm='layer', post=False, gate=False, scale=True, p=0.0, train=True),
        # -- gated_linear
        # one pixel at inference: the weights are read once
        dict(name='gated-pixel', op='gated', dtype='bf16', N=1, H=1, W=1, C=512, F=2048, act='silu', bias=False, train=False),
        # the pooling pyramid's 6 x 6 bins of a batch, hidden width 8/3 of the channels (odd)
        dict(name='gated-bins', op='gated', dtype='f16', N=8, H=6, W=6, C=512, F=1365, act='silu', bias=True, train=False),
        # evaluation of a batch at 29 x 38
        dict(name='gated-eval', op='gated', dtype='bf16', N=8, H=29, W=38, C=512, F=2048, act='gelu', bias=True, train=False),
        # training at the trunk's size
        dict(name='gated-train', op='gated', dtype='f16', N=8, H=57, W=76, C=256, F=1024, act='silu', bias=True, train=True),
        # training in the f32 parity mode at the bottleneck, odd hidden width
        dict(name='gated-f32', op='gated', dtype='f32', N=8, H=15, W=19, C=512, F=1365, act='sigmoid', bias=True, train=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _pixels(rng, most):
    """N, H, W of a map of at most `most` pixels"""
    n = min(rng.choice([1, 2, 3, 8, 16]), most)
    hw = _log(rng, 1, max(1, most // n))
    h = max(1, min(hw, int(math.sqrt(hw * rng.uniform(0.5, 1.0)))))
    return n, h, max(1, hw // h)


def draw(rng):
    op = rng.choice(['dropout', 'residual', 'gated'])
    dtype = rng.choice(['f32', 'f16', 'bf16'])
    if op == 'dropout':
        C = _log(rng, 1, 2048)
        ld = C + rng.choice([0, 0, 0, 8, 64, 3])
        n, h, w = _pixels(rng, min(555000, _MOST_ELEMENTS // (2 * ld)))
        return dict(op=op, dtype=dtype, N=n, H=h, W=w, C=C, ld=ld, p=round(rng.uniform(0.02, 0.9), 3))
    if op == 'residual':
        C = _log(rng, 8, 4096)
        if rng.random() < 0.5:
            C = max(8, C // 8 * 8)
        n, h, w = _pixels(rng, min(139000, _MOST_ELEMENTS // (4 * C)))
        return dict(op=op, dtype=dtype, N=n, H=h, W=w, C=C, norm=rng.choice(['rms', 'layer']), post=rng.random() < 0.7, gate=rng.random() < 0.6,
                    scale=rng.random() < 0.6, p=rng.choice([0.0, 0.0, 0.1, 0.5]), train=rng.random() < 0.6)
    C, F = _log(rng, 16, 2048), _log(rng, 16, 4096)
    if rng.random() < 0.6:
        C, F = max(16, C // 8 * 8), max(16, F // 8 * 8)
    train = rng.random() < 0.5
    most = _MOST_FLOPS / (12.0 if train else 4.0) / (C * F) / (8 if dtype == 'f32' else 1)
    n, h, w = _pixels(rng, max(1, min(34656, int(most))))
    return dict(op=op, dtype=dtype, N=n, H=h, W=w, C=C, F=F, act=rng.choice(['silu', 'gelu', 'sigmoid', 'relu']), bias=rng.random() < 0.5, train=train)


# ------------------------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)
    dt = _DT[case['dtype']]
    N, H, W, C = case['N'], case['H'], case['W'], case['C']

    def rnd(*shape, std=1.0, mean=0.0, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device='cuda').mul_(std).add_(mean).to(dtype)

    s = dict(case, rng=(1_000_003 * seed + 17, 4 * seed + 5))
    if case['op'] == 'dropout':
        wide = rnd(N, H, W, case['ld'], dtype=dt)
        s['x'] = wide[..., :C].requires_grad_(True)
        s['gy'] = rnd(N, H, W, C, dtype=dt)
        return s
    train = case['train']
    if case['op'] == 'residual':
        # the residual stream grows over the blocks and has channels of different sizes
        s['x'] = (rnd(N, H, W, C) * rnd(C, std=0.3, mean=1.0)).to(dt)
        s['h'] = (rnd(N, H, W, C, std=0.5, mean=0.1)).to(dt)
        s['gate'] = rnd(N, C, std=0.5, mean=1.0) if case['gate'] else None
        s['scale'] = rnd(C, std=0.05, mean=0.5) if case['scale'] else None
        layer = case['norm'] == 'layer'
        s['post'] = (rnd(C, std=0.1, mean=1.0), rnd(C, std=0.1) if layer else None) if case['post'] else None
        s['pre'] = (rnd(C, std=0.1, mean=1.0), rnd(C, std=0.1) if layer else None)
        s['leaves'] = [t for t in (s['x'], s['h'], s['gate'], s['scale'], *(s['post'] or ()), *s['pre']) if t is not None]
        if train:
            s['gy'], s['gn'] = rnd(N, H, W, C, dtype=dt), rnd(N, H, W, C, dtype=dt)
    else:
        F = case['F']
        s['x'] = rnd(N, H, W, C, dtype=dt)
        s['wg'], s['wu'] = rnd(F, C, std=C ** -0.5, dtype=dt), rnd(F, C, std=C ** -0.5, dtype=dt)
        s['bg'], s['bu'] = (rnd(F, std=0.1), rnd(F, std=0.1)) if case['bias'] else (None, None)
        s['leaves'] = [t for t in (s['x'], s['wg'], s['wu'], s['bg'], s['bu']) if t is not None]
        if train:
            s['gz'] = rnd(N, H, W, F, dtype=dt)
    if train:
        for t in s['leaves']:
            t.requires_grad_(True)
    return s


# ------------------------------------------------------------------------------------------------------------------ the operators in plain form
def _mulhi(a, m):
    """high and low 32 bits of the product of 32-bit words kept in int64"""
    p = a * m                                 # (wraps modulo 2^64: the bits are those of the unsigned product)
    return (p >> 32) & 0xffffffff, p & 0xffffffff


def _keep(n, p, rng, device):
    """boolean keep mask of n elements"""
    seed, offset = rng
    q = torch.arange((n + 7) // 8, device=device, dtype=torch.int64)
    c0, c1 = q & 0xffffffff, q >> 32
    c2, c3 = torch.full_like(q, offset & 0xffffffff), torch.full_like(q, (offset >> 32) & 0xffffffff)
    k0, k1 = seed & 0xffffffff, (seed >> 32) & 0xffffffff
    for _ in range(10):                       # the generator's ten rounds
        h0, l0 = _mulhi(c0, 0xD2511F53)
        h1, l1 = _mulhi(c2, 0xCD9E8D57)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & 0xffffffff, (k1 + 0xBB67AE85) & 0xffffffff
    w = torch.stack([c0 & 0xffff, c0 >> 16, c1 & 0xffff, c1 >> 16, c2 & 0xffff, c2 >> 16, c3 & 0xffff, c3 >> 16], 1).reshape(-1)[:n]
    return w >= _threshold(p)


def _threshold(p):
    return int(p * 65536 + 0.5)


def _norm(v, wb, layer):
    """-> (normalised * weight + bias, normalised, reciprocal deviation)"""
    c = v - v.mean(-1, keepdim=True) if layer else v
    r = torch.rsqrt((c * c).mean(-1, keepdim=True) + _EPS)
    hat = c * r
    out = hat * wb[0]
    return (out + wb[1] if wb[1] is not None else out), hat, r


def _norm_grad(g, hat, r, w, layer):
    t = g * w
    d = t - hat * (t * hat).mean(-1, keepdim=True)
    return r * (d - t.mean(-1, keepdim=True) if layer else d)


def _rows(t):
    return t.sum((0, 1, 2))


def _plain_residual(s):
    dt, layer = s['x'].dtype, s['norm'] == 'layer'
    x, h = s['x'].float(), s['h'].float()
    f = torch.ones((), device=x.device)
    if s['scale'] is not None:
        f = f * s['scale']
    if s['gate'] is not None:
        f = f * s['gate'][:, None, None, :]
    u, hat, r = _norm(h, s['post'], layer) if s['post'] else (h, None, None)
    if s['p'] > 0:
        m = _keep(h.numel(), s['p'], s['rng'], x.device).view(h.shape)
        inv = 1.0 / (1.0 - _threshold(s['p']) / 65536)
        u = torch.where(m, u * inv, torch.zeros_like(u))
    y = x + f * u
    n, hat2, r2 = _norm(y, s['pre'], layer)
    out = [y.to(dt), n.to(dt)]
    if not s['train']:
        return out
    gy, gn = s['gy'].float(), s['gn'].float()
    t = gy + _norm_grad(gn, hat2, r2, s['pre'][0], layer)
    dgate = dscale = None
    if s['gate'] is not None:
        dgate = (t * u).sum((1, 2)) if s['scale'] is None else (t * u).sum((1, 2)) * s['scale']
    if s['scale'] is not None:
        dscale = _rows(t * u) if s['gate'] is None else _rows(t * u * s['gate'][:, None, None, :])
    du = t * f
    if s['p'] > 0:
        du = torch.where(m, du * inv, torch.zeros_like(du))
    dpost = ()
    if s['post']:
        dpost = (_rows(du * hat), _rows(du))
        du = _norm_grad(du, hat, r, s['post'][0], layer)
    out += [t.to(dt), du.to(dt)] + [d for d in (dgate, dscale) if d is not None] + list(dpost[:2 if layer else 1])
    return out + [_rows(gn * hat2), _rows(gn)][:2 if layer else 1]


def _act(g, name):
    """activation and its derivative"""
    if name == 'relu':
        return torch.clamp(g, min=0), (g > 0).to(g.dtype)
    if name == 'gelu':
        phi = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
        return g * phi, phi + g * torch.exp(-0.5 * g * g) * (1 / math.sqrt(2 * math.pi))
    sig = 1 / (1 + torch.exp(-g))
    return (sig, sig * (1 - sig)) if name == 'sigmoid' else (g * sig, sig * (1 + g * (1 - sig)))


def _plain_gated(s):
    dt, shape = s['x'].dtype, s['x'].shape
    x = s['x'].float().reshape(-1, shape[3])
    wg, wu = s['wg'].float(), s['wu'].float()
    g, u = x @ wg.t(), x @ wu.t()
    if s['bg'] is not None:
        g, u = g + s['bg'], u + s['bu']
    a, da = _act(g, s['act'])
    out = [(a * u).to(dt).view(*shape[:3], -1)]
    if not s['train']:
        return out
    gz = s['gz'].float().reshape(g.shape)
    dg, du = gz * u * da, gz * a
    out += [(dg @ wg + du @ wu).to(dt).view(shape), (dg.t() @ x).to(dt), (du.t() @ x).to(dt)]
    return out + ([dg.sum(0), du.sum(0)] if s['bg'] is not None else [])


def _plain_dropout(s):
    dt = s['x'].dtype
    m = _keep(s['x'].numel(), s['p'], s['rng'], s['x'].device).view(s['x'].shape)
    f = torch.where(m, 1.0 / (1.0 - _threshold(s['p']) / 65536), 0.0)
    return [(s['x'].float() * f).to(dt), (s['gy'].float() * f).to(dt)]


def run(s):
    if not own:
        with torch.no_grad():
            return {'dropout': _plain_dropout, 'residual': _plain_residual, 'gated': _plain_gated}[s['op']](s)
    from rdfc_gan_amd import functional as Fh
    if s['op'] == 'dropout':
        y = Fh.dropout(s['x'], s['p'], rng=s['rng'])
        return [y, *torch.autograd.grad(y, [s['x']], s['gy'])]
    if s['op'] == 'residual':
        y, n = Fh.norm_residual(s['x'], s['h'], gate=s['gate'], scale=s['scale'], post=s['post'], pre=s['pre'], norm=s['norm'], eps=_EPS, p=s['p'],
                                rng=s['rng'])
        return [y, n, *(torch.autograd.grad([y, n], s['leaves'], [s['gy'], s['gn']]) if s['train'] else ())]
    z = Fh.gated_linear(s['x'], s['wg'], s['wu'], s['bg'], s['bu'], act=s['act'])
    return [z, *(torch.autograd.grad(z, s['leaves'], s['gz']) if s['train'] else ())]


# ------------------------------------------------------------------------------------------------------------------ bytes and operations
def work(case):
    b = 4 if case['dtype'] == 'f32' else 2
    m, C = case['N'] * case['H'] * case['W'], case['C']
    if case['op'] == 'dropout':
        return {'bytes': 4 * b * m * C, 'flops': 2 * m * C}
    if case['op'] == 'residual':
        cols = 4 * C * ((1 if case['norm'] == 'rms' else 2) * (2 if case['post'] else 1) + bool(case['scale']) + (case['N'] if case['gate'] else 0))
        if not case['train']:
            return {'bytes': 4 * b * m * C + cols, 'flops': 14 * m * C}
        return {'bytes': 8 * b * m * C + 2 * cols, 'flops': 45 * m * C}            # x, h, two cotangents in; y, n, two gradients out
    F = case['F']
    w = 2 * b * F * C + (8 * F if case['bias'] else 0)
    if not case['train']:
        return {'bytes': b * m * (C + F) + w, 'flops': 4 * m * C * F}
    return {'bytes': 2 * (b * m * (C + F) + w), 'flops': 12 * m * C * F}


# ------------------------------------------------------------------------------------------------------------------ the operators in 64 bits
def _philox_numpy(n, p, rng):
    """the keep mask from unsigned arithmetic on the host"""
    u = np.uint64
    low, s32 = u(0xffffffff), u(32)
    ctr = [np.arange(-(-n // 8), dtype=np.uint64) & low, np.arange(-(-n // 8), dtype=np.uint64) >> s32, u(rng[1]) & low, u(rng[1]) >> s32]
    key = [int(rng[0]) & 0xffffffff, int(rng[0]) >> 32 & 0xffffffff]
    for r in range(10):
        a, b = ctr[0] * u(0xD2511F53), ctr[2] * u(0xCD9E8D57)
        ctr = [(b >> s32) ^ ctr[1] ^ u((key[0] + r * 0x9E3779B9) & 0xffffffff), b & low,
               (a >> s32) ^ ctr[3] ^ u((key[1] + r * 0xBB67AE85) & 0xffffffff), a & low]
    words = np.stack([np.broadcast_to(c, ctr[0].shape) for c in ctr], 1).astype('<u4').view('<u2')
    return torch.from_numpy(words.reshape(-1)[:n] >= round(p * 65536)).cuda()


def _leaf64(t):
    return None if t is None else t.detach().double().requires_grad_(True)


def _norm64(v, wb, kind):
    if kind == 'layer':
        v = v - v.mean(-1, keepdim=True)
    v = v / (v.pow(2).mean(-1, keepdim=True) + _EPS).sqrt() * wb[0]
    return v if wb[1] is None else v + wb[1]


def exact(case, seed):
    s = prepare(case, seed)
    x = _leaf64(s['x'])
    if s['op'] == 'dropout':
        keep = _philox_numpy(x.numel(), s['p'], s['rng']).view(x.shape)
        y = x * keep / (1 - round(s['p'] * 65536) / 65536)
        return [y, *torch.autograd.grad(y, [x], s['gy'].double())]
    if s['op'] == 'residual':
        h, gate, scale = _leaf64(s['h']), _leaf64(s['gate']), _leaf64(s['scale'])
        post = tuple(map(_leaf64, s['post'])) if s['post'] else None
        pre = tuple(map(_leaf64, s['pre']))
        v = h if post is None else _norm64(h, post, s['norm'])
        if s['p'] > 0:
            v = v * _philox_numpy(v.numel(), s['p'], s['rng']).view(v.shape) / (1 - round(s['p'] * 65536) / 65536)
        if gate is not None:
            v = v * gate.view(s['N'], 1, 1, -1)
        y = x + (v if scale is None else v * scale)
        n = _norm64(y, pre, s['norm'])
        leaves = [t for t in (x, h, gate, scale, *(post or ()), *pre) if t is not None]
        return [y, n, *(torch.autograd.grad([y, n], leaves, [s['gy'].double(), s['gn'].double()]) if s['train'] else ())]
    wg, wu, bg, bu = map(_leaf64, (s['wg'], s['wu'], s['bg'], s['bu']))
    g, u = torch.nn.functional.linear(x, wg, bg), torch.nn.functional.linear(x, wu, bu)
    act = {'relu': torch.relu, 'sigmoid': torch.sigmoid, 'silu': torch.nn.functional.silu, 'gelu': torch.nn.functional.gelu}[s['act']]
    z = act(g) * u
    leaves = [t for t in (x, wg, wu, bg, bu) if t is not None]
    return [z, *(torch.autograd.grad(z, leaves, s['gz'].double()) if s['train'] else ())]
