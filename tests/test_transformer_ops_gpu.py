"""The transformer-block operators (csrc/dropout.hip, norm_residual.hip, gated_linear.hip) against the 64-bit oracle.

Tolerances: an output of the map's type is off by at most half a step of that type (finfo.eps / 2, relative) plus what f32 arithmetic on the
way adds, which the oracle bounds from the sums of absolute terms (oracle/transformer_ops.py); f32 outputs by the latter and half an f32 step.
f16 results below the normal range are off by at most half a subnormal step, 2^-25."""
import pytest
import torch

from oracle import transformer_ops as O

pytestmark = pytest.mark.gpu

DEV = 'cuda'
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ['f32', 'bf16', 'f16']


def Fh():
    from rdfc_gan_amd import functional
    return functional


def rnd(*shape, seed, dtype=torch.float32, std=1.0, mean=0.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std + mean).to(dtype)


def lay(t, how):
    """the map t on the device as: dense, a channel slice of a wider map, or a view that is not pixel-major"""
    t = t.to(DEV)
    if how == 'slice':
        wide = torch.full((*t.shape[:3], t.shape[3] + 11), 3.0, dtype=t.dtype, device=DEV)
        wide[..., 5:5 + t.shape[3]] = t
        return wide[..., 5:5 + t.shape[3]]
    if how == 'aligned-slice':
        wide = torch.full((*t.shape[:3], t.shape[3] + 24), 3.0, dtype=t.dtype, device=DEV)
        wide[..., 8:8 + t.shape[3]] = t
        return wide[..., 8:8 + t.shape[3]]
    if how == 'nchw':
        return t.permute(0, 3, 1, 2).contiguous().permute(0, 2, 3, 1)
    return t


def check(got, want, bound, what):
    """elementwise: half a step of got's type, relative to the value, plus the bound"""
    got64, want, bound = got.detach().double().cpu(), want.reshape(got.shape), torch.as_tensor(bound, dtype=torch.float64)
    if bound.dim():
        bound = bound.reshape(got.shape)
    half = torch.finfo(got.dtype).eps / 2
    tol = half * (want.abs() + bound) + bound + (2.0 ** -25 if got.dtype == torch.float16 else 0.0)
    bad = (got64 - want).abs() > tol
    bad |= ~torch.isfinite(got64)
    if bad.any():
        at = bad.reshape(-1).nonzero()[0, 0]
        raise AssertionError(f'{what}: {int(bad.sum())} of {bad.numel()} off, first at {int(at)}: {got64.reshape(-1)[at]} for {want.reshape(-1)[at]}, '
                             f'tolerance {tol.reshape(-1)[at]}')


# ---- dropout --------------------------------------------------------------------------------------------------------------
MAPS = [(1, 1, 1, 1), (1, 1, 1, 8), (1, 1, 3, 5), (2, 3, 5, 64), (3, 7, 1, 67), (2, 15, 19, 129), (1, 5, 7, 512), (4, 1, 1, 24), (1, 40, 41, 8)]


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('how', ['dense', 'slice', 'aligned-slice', 'nchw'])
@pytest.mark.parametrize('shape', MAPS, ids=str)
def test_dropout(shape, how, dtype):
    x, gy = rnd(*shape, seed=1, dtype=dtype), rnd(*shape, seed=2, dtype=dtype)
    for p, rng in ((0.3, (0, 0)), (0.5, (0xfedcba9876543210, (1 << 63) + 77)), (1.0, (1, 2))):
        xd = lay(x, how).detach().requires_grad_(True)
        y = Fh().dropout(xd, p, rng=rng)
        gx, = torch.autograd.grad(y, xd, lay(gy, how))
        for got, src in ((y, x), (gx, gy)):
            want = O.dropout(src, p, *rng)
            assert torch.equal((got == 0).cpu() | (src == 0), (want == 0))
            check(got, want, 2 * O.U32 * want.abs(), 'dropout')           # the scale's own rounding and the product's


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
def test_dropout_hides_what_it_drops(dtype):
    """NaN and infinities in dropped places do not come through; in kept places they do"""
    x = torch.full((1, 4, 8, 64), float('nan'), dtype=dtype, device=DEV)
    x[..., 1::2] = float('inf')
    y = Fh().dropout(x, 0.5, rng=(5, 6))
    keep = O.keep_mask(x.numel(), 1 << 15, 5, 6).view(x.shape).to(DEV)
    assert bool((y[~keep] == 0).all()) and not bool(torch.isfinite(y[keep]).any())


def test_dropout_second_derivative_is_the_mask():
    x = torch.randn(1, 2, 2, 8, device=DEV, requires_grad=True)
    g = torch.randn(1, 2, 2, 8, device=DEV, requires_grad=True)
    y = Fh().dropout(x, 0.5, rng=(1, 2))
    gx, = torch.autograd.grad(y, x, g, create_graph=True)
    gg, = torch.autograd.grad(gx.sum(), g)
    assert torch.equal(gg, Fh().dropout(torch.ones_like(x), 0.5, rng=(1, 2)).detach())


def test_dropout_from_torchs_generator():
    """manual_seed repeats the draws, two calls differ, evaluation and p = 0 draw nothing"""
    x = torch.ones(2, 8, 8, 64, device=DEV)
    torch.manual_seed(3)
    a, b = Fh().dropout(x, 0.4), Fh().dropout(x, 0.4)
    torch.manual_seed(3)
    assert Fh().dropout(x, 0.0) is x and Fh().dropout(x, 0.4, training=False) is x
    assert torch.equal(a, Fh().dropout(x, 0.4)) and torch.equal(b, Fh().dropout(x, 0.4)) and not torch.equal(a, b)
    assert abs(float((a == 0).float().mean()) - 0.4) < 5 * (0.24 / a.numel()) ** 0.5


def test_dropout_from_several_threads():
    """every call takes an offset of its own"""
    import threading
    x = torch.ones(1, 4, 4, 64, device=DEV)
    out, gate = [], threading.Barrier(4)

    def work():
        gate.wait()
        for _ in range(20):
            out.append(Fh().dropout(x, 0.5))
    torch.manual_seed(11)
    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    masks = {bytes((o != 0).cpu().numpy().tobytes()) for o in out}
    assert len(out) == 80 and len(masks) == 80


def test_dropout_beside_torchs_own_draws():
    """dropout and torch's random kernels from two threads: the generator has advanced by the draws of both, four each, and none is lost"""
    import threading
    x = torch.ones(1, 1, 1, 64, device=DEV)
    n, start = 1500, threading.Barrier(2)

    def work(draw):
        start.wait()
        for _ in range(n):
            draw()
    torch.manual_seed(12)
    torch.cuda.synchronize()
    gen = torch.cuda.default_generators[torch.cuda.current_device()]
    first = gen.get_offset()
    threads = [threading.Thread(target=work, args=(f,)) for f in (lambda: Fh().dropout(x, 0.5), lambda: torch.rand(64, device=DEV))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert gen.get_offset() - first == 2 * n * 4


def test_dropout_empty_map():
    x = torch.zeros(0, 3, 4, 8, device=DEV, requires_grad=True)
    y = Fh().dropout(x, 0.5, rng=(1, 2))
    assert y.shape == x.shape and torch.autograd.grad(y.sum(), x)[0].shape == x.shape


def test_dropout_state_in_a_captured_graph():
    """every replay draws the next mask, and its backward pass the same one; eager draws in between take part in the count"""
    x, g = torch.randn(2, 5, 7, 24, device=DEV), torch.randn(2, 5, 7, 24, device=DEV)
    state = Fh().DropoutState(seed=(1 << 64) - 5, device=torch.device(DEV, torch.cuda.current_device()))

    def step():
        leaf = x.detach().requires_grad_(True)
        y = Fh().dropout(leaf, 0.5, rng=state)
        return y.detach(), torch.autograd.grad(y, leaf, g)[0]
    want = lambda k: (O.dropout(x.cpu(), 0.5, (1 << 64) - 5, k), O.dropout(g.cpu(), 0.5, (1 << 64) - 5, k))
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        first = step()
    torch.cuda.synchronize()
    for a, b in zip(first, want(0)):
        check(a, b, 2 * O.U32 * b.abs(), 'eager')
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    count = 1
    for rep in range(4):
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want(count)):
            check(a, b, 2 * O.U32 * b.abs(), f'replay {rep}')
        count += 1
        if rep == 1:
            for a, b in zip(step(), want(count)):
                check(a, b, 2 * O.U32 * b.abs(), 'eager between')
            count += 1


def test_dropout_without_a_state_is_refused_in_a_graph():
    x = torch.randn(1, 2, 2, 8, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match='DropoutState'):
            Fh().dropout(x, 0.5)
        y = x + 1
    graph.replay()
    assert torch.equal(y, x + 1)


def test_dropout_state_on_two_streams_at_once():
    """draws that overlap get keys of their own"""
    state = Fh().DropoutState(3, torch.device(DEV, torch.cuda.current_device()))
    torch.cuda.synchronize()
    keys, streams = [], [torch.cuda.Stream() for _ in range(2)]
    for i in range(40):
        with torch.cuda.stream(streams[i % 2]):
            keys.append(state.draw())
    torch.cuda.synchronize()
    assert sorted(int(k[1]) for k in keys) == list(range(40)) and int(state.state[1]) == 40


def test_dropout_beyond_32_bit_indexes():
    """a map of more than 2^32 elements: the last elements against the oracle's window of the mask"""
    shape = (1, 8193, 8192, 64)
    x = torch.ones(shape, dtype=torch.bfloat16, device=DEV)
    n = x.numel()
    assert n > 1 << 32
    y = Fh().dropout(x, 0.5, rng=(7, 1 << 60)).view(-1)
    for first in (0, (1 << 32) - 5000, (1 << 32) - 8, n - 100_003):
        m = min(10_000, n - first)
        assert torch.equal(y[first:first + m].cpu() != 0, O.keep_mask(m, 1 << 15, 7, 1 << 60, first=first)), first
    del y
    y = Fh().dropout(x[..., :63], 0.25, rng=(7, 8))                   # element by element, 64-bit rows
    first = y.numel() - 9_999
    assert torch.equal(y.view(-1)[first:].cpu() != 0, O.keep_mask(9_999, 1 << 14, 7, 8, first=first))


# ---- norm_residual --------------------------------------------------------------------------------------------------------
def residual_case(shape, dtype, how, layer, post, pre, gated, scaled, p, seed=0, dy=True, dn=True):
    """runs norm_residual with its gradients and holds every output against the oracle"""
    N, H, W, C = shape
    rng = (seed * 7919 + 3, seed + 1)
    x, h = rnd(*shape, seed=seed, dtype=dtype, std=2.0), rnd(*shape, seed=seed + 1, dtype=dtype, std=0.7, mean=0.2)
    gy, gn = rnd(*shape, seed=seed + 2, dtype=dtype), rnd(*shape, seed=seed + 3, dtype=dtype)
    gate, scale = rnd(N, C, seed=seed + 4, mean=1.0) if gated else None, rnd(C, seed=seed + 5) if scaled else None
    wb = lambda on, k: (rnd(C, seed=seed + k, std=0.3, mean=1.0), rnd(C, seed=seed + k + 1) if layer else None) if on else None
    post, pre = wb(post, 6), wb(pre, 8)
    want = O.norm_residual(x, h, gy if dy else None, gn if dn and pre else None, gate, scale, post, pre, layer, 1e-5, p, *rng)
    names = dict(x=lay(x, how), h=lay(h, how), gate=gate, scale=scale, post_w=post and post[0], post_b=post and post[1], pre_w=pre and pre[0],
                 pre_b=pre and pre[1])
    v = {k: t.to(DEV).detach().requires_grad_(True) for k, t in names.items() if t is not None}
    get = v.get
    y, n = Fh().norm_residual(v['x'], v['h'], gate=get('gate'), scale=get('scale'), post=post and (get('post_w'), get('post_b')),
                              pre=pre and (get('pre_w'), get('pre_b')), norm='layer' if layer else 'rms', p=p, rng=rng)
    assert y.is_contiguous() and y.dtype == dtype and (n is None) == (pre is None)
    check(y, *want['y'], 'y')
    if pre:
        check(n, *want['n'], 'n')
    outs, cots = ([y] if dy else []) + ([n] if pre and dn else []), ([lay(gy, how)] if dy else []) + ([lay(gn, how)] if pre and dn else [])
    grads = torch.autograd.grad(outs, list(v.values()), cots, allow_unused=True)
    for (k, t), g in zip(v.items(), grads):
        if k not in want:
            assert g is None or not bool(g.any()), k
            continue
        assert g.dtype == t.dtype and g.shape == t.shape
        check(g, *want[k], f'gradient of {k}')


RES_MAPS = [(1, 1, 1, 1), (1, 1, 1, 8), (2, 1, 3, 5), (2, 3, 5, 64), (3, 7, 3, 67), (2, 5, 9, 128), (1, 15, 19, 129), (2, 3, 3, 256), (2, 4, 4, 301), (1, 5, 7, 512),
            (2, 3, 2, 777), (1, 2, 3, 1024), (2, 1, 2, 1536), (1, 1, 3, 2048), (1, 3, 1, 4000), (1, 2, 1, 8192)]


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('layer', [False, True], ids=['rms', 'layer'])
@pytest.mark.parametrize('shape', RES_MAPS, ids=str)
def test_norm_residual(shape, layer, dtype):
    residual_case(shape, dtype, 'dense', layer, True, True, True, True, 0.0)
    residual_case(shape, dtype, 'dense', layer, True, True, False, True, 0.3, seed=20)


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('how', ['slice', 'aligned-slice', 'nchw'])
@pytest.mark.parametrize('shape', [(2, 3, 5, 64), (1, 4, 3, 129), (2, 2, 2, 1040)], ids=str)
def test_norm_residual_layouts(shape, how, dtype):
    residual_case(shape, dtype, how, True, True, True, True, False, 0.5)


def rounded_norm(v, ev, layer, eps):
    """row norm of v, itself off by ev, in f32 -> (normalised, its error, reciprocal deviation, its relative error), each element's for itself.

    A sum over the channels is a chain of at most 40 additions (eight channels a lane in up to four vectors, then eight halvings): it is off by 40
    half steps of the sum of absolute terms, the mean by two more.  The root and the division: six."""
    U, mean = O.U32, lambda t: t.mean(-1, keepdim=True)
    c, ec = v, ev
    if layer:
        c = v - mean(v)
        ec = ev + mean(ev) + 42 * U * mean(v.abs()) + U * c.abs()
    var = mean(c * c) + eps
    r = 1 / var.sqrt()
    er = 0.5 * (43 * U + 2 * mean(c.abs() * ec) / var) + 6 * U
    hat = c * r
    return hat, r * ec + hat.abs() * (er + 2 * U), r, er


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('layer', [False, True], ids=['rms', 'layer'])
@pytest.mark.parametrize('shape', [(2, 3, 5, 67), (2, 5, 9, 128), (1, 7, 9, 256), (2, 2, 3, 777), (1, 2, 5, 2048)], ids=str)
def test_norm_residual_small_elements(shape, layer, dtype):
    """y, n and the gradient of x element by element: bounds that shrink with the element's own terms, not the map's largest value (channels
    here differ by up to 2^12 in size)"""
    N, H, W, C = shape
    U, mean = O.U32, lambda t: t.mean(-1, keepdim=True)
    size = torch.exp2(-(torch.arange(C) % 13).float())
    x, h, gy, gn = ((rnd(*shape, seed=30 + i) * size).to(dtype) for i in range(4))
    gate, scale, pw, qw = rnd(N, C, seed=34, mean=1.0), rnd(C, seed=35), rnd(C, seed=36, std=0.3, mean=1.0), rnd(C, seed=37, std=0.3, mean=1.0)
    pb, qb = (rnd(C, seed=38) * size, rnd(C, seed=39) * size) if layer else (None, None)
    v = [t if t is None else t.to(DEV) for t in (x, h, gate, scale, pw, pb, qw, qb, gy, gn)]
    v[0].requires_grad_(True)
    y, n = Fh().norm_residual(v[0], v[1], gate=v[2], scale=v[3], post=(v[4], v[5]), pre=(v[6], v[7]), norm='layer' if layer else 'rms', p=0.25, rng=(8, 9))
    gx, = torch.autograd.grad([y, n], [v[0]], v[8:])
    x, h, gy, gn, gate, scale, pw, qw = (t.double() for t in (x, h, gy, gn, gate, scale, pw, qw))
    pb, qb = (torch.zeros(C, dtype=torch.float64) if t is None else t.double() for t in (pb, qb))
    f = O.dropout(torch.ones(shape), 0.25, 8, 9) * scale * gate[:, None, None, :]
    hat, e_hat, _, _ = rounded_norm(h, torch.zeros(shape, dtype=torch.float64), layer, 1e-5)
    want = x + f * (hat * pw + pb)
    e_y = (f * pw).abs() * e_hat + 8 * U * f.abs() * ((hat * pw).abs() + pb.abs()) + 2 * U * want.abs()
    check(y, want, e_y, 'y')
    yhat, e_yhat, r, er = rounded_norm(want, e_y, layer, 1e-5)
    n64 = yhat * qw + qb
    check(n, n64, qw.abs() * e_yhat + 2 * U * (n64.abs() + qb.abs()), 'n')
    g = gn * qw
    S, Z = mean(g * yhat), mean(g) if layer else torch.zeros_like(mean(g))
    e_S, e_Z = 43 * U * mean((g * yhat).abs()) + mean(g.abs() * e_yhat), 43 * U * mean(g.abs()) if layer else 0.0
    inner = g - yhat * S - Z
    e_inner = yhat.abs() * e_S + S.abs() * e_yhat + e_Z + 6 * U * (g.abs() + (yhat * S).abs() + Z.abs())
    t = gy + r * inner
    check(gx, t, r * e_inner + (r * inner).abs() * (er + 2 * U) + 2 * U * (gy.abs() + t.abs()), 'gradient of x')


@pytest.mark.parametrize('parts', range(16))
def test_norm_residual_parts(parts):
    """every combination of post, pre, gate and scale, with and without dropout and either cotangent"""
    post, pre, gated, scaled = (bool(parts >> i & 1) for i in range(4))
    for p, dy, dn in ((0.0, True, True), (0.4, True, False), (0.2, not pre, True)):
        residual_case((2, 3, 4, 40), torch.float32, 'dense', parts % 3 == 0, post, pre, gated, scaled, p, seed=parts, dy=dy, dn=dn)


def test_norm_residual_many_rows():
    """several chunks of rows per sample, a last one that is not whole"""
    residual_case((3, 61, 67, 64), torch.bfloat16, 'dense', False, True, True, True, True, 0.1)
    residual_case((1, 61, 157, 40), torch.float32, 'dense', True, True, True, False, True, 0.0)


def test_norm_residual_constant_and_zero_rows():
    """a row without variance: eps alone under the root (layer norm of a constant row is the bias)"""
    for layer in (False, True):
        x, h = torch.zeros(1, 2, 2, 16, device=DEV), torch.zeros(1, 2, 2, 16, device=DEV)
        x[0, 0] = 3.0
        b = torch.arange(16., device=DEV)
        y, n = Fh().norm_residual(x, h, post=(None, b), pre=(None, b), norm='layer' if layer else 'rms')
        want = O.norm_residual(x.cpu(), h.cpu(), None, None, None, None, (None, b.cpu()), (None, b.cpu()), layer)
        check(y, *want['y'], 'y')
        check(n, *want['n'], 'n')


def test_norm_residual_is_reproducible_and_takes_two_streams():
    """the same bits every run, alone and beside another call on another stream"""
    v = [rnd(4, 29, 38, 256, seed=i).to(DEV) for i in range(4)]
    w = rnd(256, seed=9).to(DEV).requires_grad_(True)
    gate = rnd(4, 256, seed=10).to(DEV).requires_grad_(True)

    def run():
        y, n = Fh().norm_residual(v[0], v[1], gate=gate, post=(w, None), pre=(w, None), p=0.2, rng=(1, 2))
        return [y, n, *torch.autograd.grad([y, n], [w, gate], v[2:])]
    first = run()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in streams:
        with torch.cuda.stream(s):
            outs.append(run())
    torch.cuda.synchronize()
    for o in outs:
        for a, b in zip(o, first):
            assert torch.equal(a, b)


def test_row_norm():
    for shape, dtype, layer in (((2, 3, 4, 40), torch.float32, True), ((1, 1, 1, 512), torch.bfloat16, False), ((2, 5, 1, 33), torch.float16, True)):
        x, g = rnd(*shape, seed=1, dtype=dtype, std=3.0), rnd(*shape, seed=2, dtype=dtype)
        w, b = rnd(shape[3], seed=3, mean=1.0), rnd(shape[3], seed=4) if layer else None
        want = O.norm_residual(x, None, None, g, None, None, None, (w, b), layer)
        leaves = [t.to(DEV).requires_grad_(True) for t in (x, w, b) if t is not None]
        n = Fh().row_norm(*leaves, norm='layer' if layer else 'rms') if layer else Fh().row_norm(*leaves)
        check(n, *want['n'], 'n')
        for t, k in zip(torch.autograd.grad(n, leaves, g.to(DEV)), ('x', 'pre_w', 'pre_b')):
            check(t, *want[k], k)


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
def test_norm_residual_hides_what_it_drops(dtype):
    """NaN and infinities in dropped places of h reach neither the maps nor a gradient"""
    shape, rng = (2, 3, 5, 40), (5, 6)
    keep = O.keep_mask(2 * 3 * 5 * 40, O.threshold_of(0.4), *rng).view(shape)
    x, h, gy = (rnd(*shape, seed=i, dtype=dtype) for i in range(3))
    scale, gate = rnd(40, seed=4), rnd(2, 40, seed=5)
    bad = torch.where(keep, h, torch.full_like(h, float('nan')))
    bad[0, 0] = torch.where(keep[0, 0], h[0, 0], torch.full_like(h[0, 0], float('inf')))
    outs = []
    for t in (h, bad):
        v = [a.to(DEV).detach().requires_grad_(True) for a in (x, t, gate, scale)]
        y, _ = Fh().norm_residual(v[0], v[1], gate=v[2], scale=v[3], p=0.4, rng=rng)
        outs.append([y, *torch.autograd.grad(y, v, gy.to(DEV))])
    for a, b in zip(*outs):
        assert bool(torch.isfinite(a).all()) and torch.equal(a, b)


def test_norm_residual_takes_activations_as_gate_and_scale():
    """a 16-bit gate [N, 1, 1, C] that another layer produced gets its gradient in its own type"""
    x, h = rnd(2, 3, 4, 24, seed=1, dtype=torch.bfloat16).to(DEV), rnd(2, 3, 4, 24, seed=2, dtype=torch.bfloat16).to(DEV)
    gate = rnd(2, 1, 1, 24, seed=3, dtype=torch.bfloat16).to(DEV).requires_grad_(True)
    y, _ = Fh().norm_residual(x, h, gate=gate)
    f = gate.detach().float().flatten(1).requires_grad_(True)
    z, _ = Fh().norm_residual(x, h, gate=f)
    a, b = torch.autograd.grad(y, gate, torch.ones_like(y))[0], torch.autograd.grad(z, f, torch.ones_like(z))[0]
    assert torch.equal(y, z) and a.dtype == torch.bfloat16 and a.shape == gate.shape and torch.equal(a.flatten(1), b.to(torch.bfloat16))


def test_norm_residual_misaligned_parameters():
    """parameters inside a flat buffer (as an optimizer lays them out), at offsets that are not whole vectors"""
    C = 64
    x, h = rnd(2, 3, 5, C, seed=1).to(DEV), rnd(2, 3, 5, C, seed=2).to(DEV)
    flat = rnd(4 * C + 1, seed=3).to(DEV)
    v = [flat[1 + i * C:1 + (i + 1) * C] for i in range(4)]
    a = Fh().norm_residual(x, h, scale=v[0], post=(v[1], v[2]), pre=(v[3], None))
    b = Fh().norm_residual(x, h, scale=v[0].clone(), post=(v[1].clone(), v[2].clone()), pre=(v[3].clone(), None))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_norm_residual_beyond_32_bit_indexes():
    """maps of more than 2^32 elements: the last rows are those of a small call on them, and their dropout the oracle's window"""
    shape, tail = (1, 8193, 8192, 64), 5000
    x = torch.zeros(shape, dtype=torch.bfloat16, device=DEV)
    h = torch.zeros(shape, dtype=torch.bfloat16, device=DEV)
    for t, seed in ((x, 1), (h, 2)):
        t.view(-1, 64)[-tail:] = rnd(tail, 64, seed=seed, dtype=torch.bfloat16).to(DEV)
    small = [t.view(-1, 64)[-tail:].reshape(1, 1, tail, 64) for t in (x, h)]
    w = rnd(64, seed=3, mean=1.0).to(DEV)
    y, n = Fh().norm_residual(x, h, post=(w, None), pre=(w, None))
    ys, ns = Fh().norm_residual(*small, post=(w, None), pre=(w, None))
    assert torch.equal(y.view(-1, 64)[-tail:], ys.view(-1, 64)) and torch.equal(n.view(-1, 64)[-tail:], ns.view(-1, 64))
    del y, n
    y, _ = Fh().norm_residual(torch.zeros_like(x), torch.ones_like(h), p=0.5, rng=(5, 6))
    first = x.numel() - tail * 64
    assert torch.equal(y.view(-1)[first:].cpu() != 0, O.keep_mask(tail * 64, 1 << 15, 5, 6, first=first))


def test_norm_residual_empty_and_unused():
    x = torch.zeros(2, 0, 4, 8, device=DEV, requires_grad=True)
    w = torch.ones(8, device=DEV, requires_grad=True)
    gate = torch.ones(2, 8, device=DEV, requires_grad=True)
    y, n = Fh().norm_residual(x, x.detach(), gate=gate, pre=(w, None))
    gx, gw, gg = torch.autograd.grad([y, n], [x, w, gate], [torch.zeros_like(y), torch.zeros_like(n)])
    assert gx.shape == x.shape and not bool(gw.any()) and not bool(gg.any())
    x = torch.randn(2, 1, 1, 8, device=DEV, requires_grad=True)
    y, n = Fh().norm_residual(x, x.detach(), pre=(w, None))
    assert torch.equal(torch.autograd.grad(y, x, torch.ones_like(y))[0], torch.ones_like(x))      # n unused


# ---- gated_linear ---------------------------------------------------------------------------------------------------------
def gated_case(M, K, F, dtype, act, bias=True, how='dense', train=True, seed=0, master=False):
    N, H, W = M
    x, gz = rnd(N, H, W, K, seed=seed, dtype=dtype), rnd(N, H, W, F, seed=seed + 1, dtype=dtype)
    wdt = torch.float32 if master else dtype
    wg, wu = (rnd(F, K, seed=seed + 2 + i, std=K ** -0.5, dtype=dtype).to(wdt) for i in range(2))
    bg, bu = (rnd(F, seed=seed + 4 + i, std=0.5) for i in range(2)) if bias else (None, None)
    want = O.gated_linear(x.reshape(-1, K), wg, wu, bg, bu, gz.reshape(-1, F) if train else None, act, 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2)
    names = dict(x=lay(x, how), wg=wg, wu=wu, bg=bg, bu=bu)
    v = {k: t.to(DEV).detach().requires_grad_(train) for k, t in names.items() if t is not None}
    z = Fh().gated_linear(*(v.get(k) for k in ('x', 'wg', 'wu', 'bg', 'bu')), act=act)
    assert z.shape == (N, H, W, F) and z.dtype == dtype and z.is_contiguous()
    check(z, *want['z'], 'z')
    if train:
        for (k, t), g in zip(v.items(), torch.autograd.grad(z, list(v.values()), lay(gz, how))):
            assert g.dtype == t.dtype and g.shape == t.shape
            check(g, *want[k], f'gradient of {k}')


GATED = [((1, 1, 1), 1, 1), ((1, 1, 1), 8, 8), ((1, 1, 1), 64, 40), ((1, 1, 1), 513, 129), ((1, 1, 1), 512, 1000), ((1, 1, 3), 16, 24), ((2, 3, 3), 72, 136),
         ((1, 4, 4), 33, 65), ((1, 5, 7), 128, 256), ((2, 8, 8), 64, 64), ((1, 13, 10), 200, 88), ((3, 9, 11), 129, 67), ((2, 17, 19), 40, 300), ((1, 33, 31), 256, 160)]


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('case', GATED, ids=str)
def test_gated_linear(case, dtype):
    gated_case(*case, dtype, 'silu')
    gated_case(*case, dtype, 'gelu', bias=False, train=False, seed=7)


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('act', ['silu', 'gelu', 'sigmoid', 'relu'])
def test_gated_linear_activations(act, dtype):
    gated_case((2, 5, 7), 72, 48, dtype, act)
    gated_case((2, 15, 10), 136, 200, dtype, act, bias=False)


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
@pytest.mark.parametrize('how', ['slice', 'aligned-slice', 'nchw'])
def test_gated_linear_layouts(how, dtype):
    gated_case((2, 9, 8), 64, 72, dtype, 'silu', how=how)
    gated_case((1, 1, 2), 45, 31, dtype, 'silu', how=how)


@pytest.mark.parametrize('dtype', DTYPES[1:], ids=IDS[1:])
def test_gated_linear_f32_masters(dtype):
    gated_case((2, 9, 8), 64, 72, dtype, 'silu', master=True)


def test_gated_linear_weights_of_a_1x1_convolution_and_of_one_matrix():
    """[F, K, 1, 1] weights, and the two halves of one [2 F, K] matrix (views, transposed storage)"""
    x = rnd(1, 3, 5, 24, seed=1).to(DEV)
    w = rnd(2, 40, 24, seed=2).to(DEV)
    z = Fh().gated_linear(x, w[0], w[1])
    both = w.reshape(80, 24)
    assert torch.equal(z, Fh().gated_linear(x, both[:40], both[40:]))
    assert torch.equal(z, Fh().gated_linear(x, w[0].view(40, 24, 1, 1), w[1].view(40, 24, 1, 1).to(memory_format=torch.channels_last)))
    assert torch.equal(z, Fh().gated_linear(x, w[0].t().contiguous().t(), w[1].t().contiguous().t()))
    wide = torch.zeros(40, 31, device=DEV)
    wide[:, 3:27] = w[0]
    assert torch.equal(z, Fh().gated_linear(x, wide[:, 3:27], w[1]))


def test_gated_linear_beyond_32_bit_indexes():
    """a map of more than 2^32 elements: the last rows are those of a small call on them"""
    M, K, F, tail = (1 << 24) + 77, 264, 16, 500
    x = torch.zeros(1, 1, M, K, dtype=torch.bfloat16, device=DEV)
    x[0, 0, -tail:] = rnd(tail, K, seed=1, dtype=torch.bfloat16).to(DEV)
    w = [rnd(F, K, seed=2 + i, std=0.1, dtype=torch.bfloat16).to(DEV) for i in range(2)]
    assert x.numel() > 1 << 32
    z = Fh().gated_linear(x, *w)
    assert torch.equal(z[0, 0, -tail:], Fh().gated_linear(x[:, :, -tail:].contiguous(), *w)[0, 0])
    assert not bool(z[0, 0, :1000].any())


def test_gated_linear_takes_expanded_cotangents_and_runs_backward_twice():
    x, w = rnd(1, 5, 6, 24, seed=1).to(DEV).requires_grad_(True), rnd(2, 40, 24, seed=2).to(DEV).requires_grad_(True)
    z = Fh().gated_linear(x, w[0], w[1])
    a = torch.autograd.grad(z.sum(), [x, w], retain_graph=True)
    b = torch.autograd.grad(z, [x, w], torch.ones_like(z))
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_gated_linear_extreme_gates():
    """gates far out: no overflow turns into NaN, forward or backward"""
    for dtype in DTYPES:
        x = torch.tensor([200.0, -200.0, 0.0, 30.0], dtype=dtype, device=DEV).view(1, 1, 4, 1).requires_grad_(True)
        w = torch.ones(8, 1, dtype=dtype, device=DEV)
        for act in ('silu', 'gelu', 'sigmoid', 'relu'):
            z = Fh().gated_linear(x, w, w, act=act)
            gx, = torch.autograd.grad(z, x, torch.ones_like(z))
            assert bool(torch.isfinite(z).all()) and bool(torch.isfinite(gx).all()), (act, dtype)


@pytest.mark.parametrize('dtype,far,up', [(torch.bfloat16, -12.0, 1.0), (torch.float16, -6.0, 32768.0)], ids=IDS[1:])
def test_gated_linear_gelu_tail_is_relatively_accurate(dtype, far, up):
    """gates from 0 far into the negative tail, alone in their dot products, so that gelu(g) and its derivative come out scaled by a power of two and normal
    numbers of the type: relative errors of half a step of the type a rounding (z: one; dx: dg and dx), and 2^-15 for the f32 arithmetic: the fit of
    phi and the rounding of the exponential's argument (g^2 / 2 half steps of f32 at most 72, 4.3e-6 each of them) are 1.1e-5, twice that where the
    derivative's two terms partly cancel.  (Left out: around the derivative's zero at -0.7518, where the terms cancel altogether.)"""
    import math
    half = torch.finfo(dtype).eps / 2
    g = torch.linspace(0.0, far, 3001).to(dtype).unique()
    x = torch.stack([g, torch.ones_like(g)], 1).view(1, 1, -1, 2).to(DEV).requires_grad_(True)
    wg, wu = (torch.tensor([row], dtype=dtype, device=DEV).expand(8, 2).contiguous() for row in ([1.0, 0.0], [0.0, up]))
    z = Fh().gated_linear(x, wg, wu, act='gelu')
    dz = torch.zeros_like(z)
    dz[..., 3] = 1.0
    dx, = torch.autograd.grad(z, x, dz)
    g = g.double()
    phi, pdf = 0.5 * torch.special.erfc(-g * math.sqrt(0.5)), torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    for got, want, steps in ((z[0, 0, :, 3], g * phi * up, 1), (dx[0, 0, :, 0], (phi + g * pdf) * up, 2)):
        got, use = got.detach().double().cpu(), torch.ones_like(g, dtype=torch.bool) if steps == 1 else (g < -1.2) | (g > -0.4)
        off = (got - want).abs() - (2.0 ** -25 if dtype == torch.float16 else 0.0) * steps
        rel = (off / want.abs())[use & (want != 0)]
        worst = float(rel.max())
        assert worst <= steps * half * (1 + half) + 2.0 ** -15, (steps, worst)


def test_gated_linear_keeps_nan_rows_apart():
    """a NaN or infinite pixel spoils its own row only"""
    for M, K, F in ((5, 64, 40), (150, 72, 136), (300, 40, 264)):
        x = rnd(1, 1, M, K, seed=3).to(torch.bfloat16)
        w = rnd(2, F, K, seed=4).to(torch.bfloat16).to(DEV)
        clean = Fh().gated_linear(x.to(DEV), w[0], w[1])
        x[0, 0, 2, 5], x[0, 0, 3, 0] = float('nan'), float('inf')
        z = Fh().gated_linear(x.to(DEV), w[0], w[1])
        assert bool(torch.isnan(z[0, 0, 2]).all())
        rows = [i for i in range(M) if i not in (2, 3)]
        assert torch.equal(z[0, 0, rows], clean[0, 0, rows])


def test_gated_linear_empty_and_partial_gradients():
    w = torch.randn(8, 16, device=DEV, requires_grad=True)
    x = torch.zeros(0, 2, 2, 16, device=DEV, requires_grad=True)
    z = Fh().gated_linear(x, w, w.detach())
    gx, gw = torch.autograd.grad(z, [x, w], torch.zeros_like(z))
    assert z.shape == (0, 2, 2, 8) and gx.shape == x.shape and not bool(gw.any())
    x = torch.randn(1, 2, 2, 16, device=DEV)
    z = Fh().gated_linear(x, w, w.detach())
    both = torch.autograd.grad(Fh().gated_linear(x, w, w), w, torch.ones_like(z))[0]
    one = torch.autograd.grad(z, w, torch.ones_like(z))[0]
    assert one.shape == w.shape and not torch.equal(one, both)


def test_gated_linear_is_reproducible_and_takes_two_streams():
    x, g = (rnd(2, 38, 29, c, seed=c, dtype=torch.bfloat16).to(DEV) for c in (128, 200))
    w = [rnd(200, 128, seed=i, std=0.1, dtype=torch.bfloat16).to(DEV).requires_grad_(True) for i in range(2)]
    b = [rnd(200, seed=i).to(DEV).requires_grad_(True) for i in range(2)]
    x.requires_grad_(True)

    def run():
        z = Fh().gated_linear(x, *w, *b)
        return [z, *torch.autograd.grad(z, [x, *w, *b], g)]
    first = run()
    torch.cuda.synchronize()
    outs = []
    for s in [torch.cuda.Stream() for _ in range(2)]:
        with torch.cuda.stream(s):
            outs.append(run())
    torch.cuda.synchronize()
    for o in outs:
        for p, q in zip(o, first):
            assert torch.equal(p, q)


@pytest.mark.parametrize('dtype', DTYPES, ids=IDS)
def test_no_grad_gives_the_same_values_without_what_a_backward_pass_needs(dtype):
    """parameters under no_grad and inference_mode: the outputs of a training call, and no memory beyond them"""
    x, h = rnd(2, 29, 38, 64, seed=1, dtype=dtype).to(DEV), rnd(2, 29, 38, 64, seed=2, dtype=dtype).to(DEV)
    w = torch.nn.Parameter(rnd(64, seed=3, mean=1.0).to(DEV))
    m = [torch.nn.Parameter(rnd(256, 64, seed=4 + i, std=0.1, dtype=dtype).to(DEV)) for i in range(2)]

    def run():
        return [*Fh().norm_residual(x, h, post=(w, None), pre=(w, None)), Fh().row_norm(x, w), Fh().gated_linear(x, *m)]
    want = run()
    for off in (torch.no_grad, torch.inference_mode):
        with off():
            torch.cuda.synchronize()
            torch.cuda.reset_peak_memory_stats()
            before = torch.cuda.memory_stats()['requested_bytes.all.current']
            got = run()
            grown = torch.cuda.memory_stats()['requested_bytes.all.peak'] - before
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert grown == sum(t.numel() * t.element_size() for t in got)


def test_gradients_through_saved_tensor_hooks():
    """channel slices whose saved copies come back dense, from the host, or inside a wider buffer: the gradients of a run without hooks, bit for bit"""
    def wider(t):
        wide = torch.full((*t.shape[:-1], t.shape[-1] + 13), 7.0, dtype=torch.float64, device=DEV).to(t.dtype)
        wide[..., 8:8 + t.shape[-1]] = t
        return wide[..., 8:8 + t.shape[-1]]
    relays = [(lambda t: t, lambda t: t), (lambda t: t.clone(memory_format=torch.contiguous_format), lambda t: t),
              (lambda t: t.cpu(), lambda t: t.to(DEV)), (lambda t: wider(t) if t.dim() > 1 and t.is_floating_point() else t, lambda t: t)]
    for dtype in DTYPES:
        x, h, gy, gn = (lay(rnd(2, 3, 5, 67, seed=i, dtype=dtype), 'slice').requires_grad_(i < 2) for i in range(4))
        gate, w = (rnd(*s, seed=6, mean=1.0).to(DEV).requires_grad_(True) for s in ((2, 67), (67,)))
        wide = rnd(80, 131, seed=7, std=0.1, dtype=dtype).to(DEV)
        wg, wu = (wide[40 * i:40 * i + 40, 3:70].detach().requires_grad_(True) for i in range(2))
        gz = rnd(2, 3, 5, 40, seed=8, dtype=dtype).to(DEV)
        want = None
        for pack, unpack in relays:
            with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
                y, n = Fh().norm_residual(x, h, gate=gate, post=(w, None), pre=(w, None), p=0.2, rng=(3, 4))
                z = Fh().gated_linear(x, wg, wu)
            got = torch.autograd.grad([y, n], [x, h, gate, w], [gy, gn]) + torch.autograd.grad(z, [x, wg, wu], gz)
            want = want or got
            for i, (a, b) in enumerate(zip(got, want)):
                assert torch.equal(a, b), (dtype, i)


# ---- together -------------------------------------------------------------------------------------------------------------
def plain_trunk(trunk, x, gate, keeps):
    """the trunk in f64 from its parameters; keeps: dropout factors per block"""
    d = lambda t: None if t is None else t.detach().double().cpu().requires_grad_(True)
    par = {k: d(v) for k, v in trunk.named_parameters()}

    def norm(v, pre, kind):
        if kind == 'layer':
            v = v - v.mean(-1, keepdim=True)
        v = v / (v.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt() * par[pre + '.weight']
        return v + par[pre + '.bias'] if pre + '.bias' in par else v
    for i, blk in enumerate(trunk.blocks):
        k = f'blocks.{i}.'
        n = norm(x, k + 'pre', blk.norm)
        lin = lambda t, name: torch.nn.functional.linear(t, par[k + name + '.weight'].flatten(1), par.get(k + name + '.bias'))
        a = lin(n, 'gate_proj')
        h = lin(torch.nn.functional.silu(a) * lin(n, 'up_proj'), 'down_proj')
        u = norm(h, k + 'post', blk.norm) if blk.post is not None else h
        if keeps is not None:
            u = u * keeps[i]
        x = x + u * (gate[:, None, None, :] if gate is not None else 1) * par.get(k + 'scale', torch.ones(()).double())
    return x, par


@pytest.mark.parametrize('norm,post,p', [('rms', True, 0.2), ('layer', False, 0.0)])
def test_trunk_of_feed_forward_blocks(norm, post, p):
    """row_norm, gated_linear, the 1x1 convolution and norm_residual chained over three blocks, values and every gradient (f32: the products'
    rounding, a few hundred half steps of the largest value through three blocks; 2^-12 relative to the largest leaves room)"""
    from rdfc_gan_amd.layers import GatedFeedForwardTrunk
    torch.manual_seed(5)
    trunk = GatedFeedForwardTrunk(3, 48, 128, norm=norm, post=post, p=p, bias=True, scale=0.5).to(DEV)
    x = rnd(2, 6, 5, 48, seed=1).to(DEV).requires_grad_(True)
    gate = rnd(2, 48, seed=2, mean=1.0).to(DEV).requires_grad_(True)
    for i, blk in enumerate(trunk.blocks):
        blk.rng = (99, i)
    g = rnd(2, 6, 5, 48, seed=3)
    y = trunk(x, gate)
    names = [k for k, _ in trunk.named_parameters()]
    got = torch.autograd.grad(y, [x, gate, *trunk.parameters()], g.to(DEV))
    x64, gate64 = x.detach().double().cpu().requires_grad_(True), gate.detach().double().cpu().requires_grad_(True)
    keeps = [O.dropout(torch.ones(2, 6, 5, 48), p, 99, i) for i in range(3)] if p else None
    y64, par = plain_trunk(trunk, x64, gate64, keeps)
    want = torch.autograd.grad(y64, [x64, gate64, *(par[k] for k in names)], g.double())
    for k, a, b in zip(['y', 'x', 'gate', *names], [y, *got], [y64, *want]):
        assert float((a.double().cpu() - b).abs().max()) <= 2.0 ** -12 * float(b.abs().max()), k


def test_trunk_trains_in_16_bits_and_replays_from_a_graph():
    """a captured forward and backward of a bf16 trunk with dropout and f32 masters: every replay equals the eager pass with the same draws"""
    from rdfc_gan_amd.layers import GatedFeedForwardTrunk
    torch.manual_seed(6)
    trunk = GatedFeedForwardTrunk(2, 64, 160, p=0.25).to(DEV)
    x, g = rnd(2, 9, 7, 64, seed=1, dtype=torch.bfloat16).to(DEV), rnd(2, 9, 7, 64, seed=2, dtype=torch.bfloat16).to(DEV)
    dev = torch.device(DEV, torch.cuda.current_device())
    params = list(trunk.parameters())

    def run(state):
        for b in trunk.blocks:
            b.rng = state
        y = trunk(x)
        return [y.detach(), *torch.autograd.grad(y, params, g)]
    eager = Fh().DropoutState(4, dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(Fh().DropoutState(0, dev))                  # packs the down projections' operands before the capture
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    replayed = Fh().DropoutState(4, dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(replayed)
    for rep in range(3):
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        want = run(eager)
        torch.cuda.synchronize()
        for i, (a, b) in enumerate(zip(got, want)):
            name = 'y' if i == 0 else [k for k, _ in trunk.named_parameters()][i - 1]
            if 'down_proj' in name:                     # (the convolution's weight gradient adds with atomics)
                assert float((a - b).abs().max()) <= 2.0 ** -16 * float(b.abs().max()) * 126, name
            else:
                assert torch.equal(a, b), (rep, name)
        torch.cuda.synchronize()


def test_trunk_under_the_flat_optimizer():
    """a step of FlatAdam on a bf16 trunk of odd hidden width, f32 masters in its flat buffer: gradients land there, weights move, and the
    next forward uses them"""
    from rdfc_gan_amd.layers import GatedFeedForwardTrunk
    from rdfc_gan_amd.optim import FlatAdam
    torch.manual_seed(7)
    trunk = GatedFeedForwardTrunk(2, 36, 45, p=0.1, bias=True, scale=1.0).to(DEV)
    x = rnd(2, 6, 5, 36, seed=1, dtype=torch.bfloat16).to(DEV)
    opt = FlatAdam(trunk.parameters(), lr=1e-2)
    before = [p.detach().clone() for p in trunk.parameters()]
    first = trunk.eval()(x)
    opt.zero_grad()
    trunk.train()(x).float().square().mean().backward()
    opt.step()
    for (k, p), b in zip(trunk.named_parameters(), before):
        unused = k == 'blocks.0.pre.bias'
        assert bool(torch.isfinite(p).all()) and (unused or not torch.equal(p.detach(), b)), k
    assert not torch.equal(first, trunk.eval()(x))


def test_graph_mode_with_dropout():
    """RDFCGAN.enable_graph() with a dropout generator: the replayed steps run and draw a new mask each"""
    from cases import STEP_HP, step_batch
    from rdfc_gan_amd import functional
    from rdfc_gan_amd.rdfc_gan import RDFCGAN
    old = functional.compute_dtype()
    functional.set_compute_dtype(torch.float16)
    try:
        norm = dict(norm_cfg=dict(type='BN2d'), activation='LeakyReLU')
        cfg = dict(local_rank=0, lr=2e-3, beta1=0.5, beta2=0.999, gan_loss_type='lsgan',
                   model=dict(G_A2B=dict(type='RDFGenerator', pretrained_on_imagenet=False),
                              G_B2A=dict(type='ResnetGenerator', input_channels=1, output_channels=3, ngf=64, norm_layer='IN2d', use_dropout=True),
                              D_A=dict(type='PatchGANDiscriminator', in_channels=1, **norm), D_B=dict(type='PatchGANDiscriminator', in_channels=3, **norm)))
        m = RDFCGAN(torch.device(DEV), False, cfg, is_train=True)
        m.train()
        data, nA, _ = step_batch(0, 2, STEP_HP['H'], STEP_HP['W'])
        data['gt_normal'] = nA
        counts = []
        for it in range(5):                              # (two eager steps first: the convolutions' own buffers cannot be allocated in a capture)
            if it == 2:
                m.enable_graph(True)
                state = next(d for d in m.G_B2A.modules() if isinstance(d, torch.nn.Dropout)).rng.state
            m.set_input(data)
            losses = m.optimize_parameters()
            assert all(v == v and abs(v) < 1e6 for v in losses.values()), losses
            torch.cuda.synchronize()
            if it >= 2:
                counts.append(int(state[1]))
        assert m._graph_mode and m._graphs is not None, 'capture fell back to eager launches'
        assert counts[2] > counts[1] > counts[0] > 0, counts
        m.enable_graph(False)
    finally:
        functional.set_compute_dtype(old)


def test_graph_mode_masks_of_two_layers_differ():
    """the dropout layers of a generator in a captured step: in every replay each of the six draws its own mask, and a new one"""
    from cases import STEP_HP, step_batch
    from rdfc_gan_amd import functional
    from rdfc_gan_amd.rdfc_gan import RDFCGAN
    old, many = functional.compute_dtype(), functional.multi_stream()
    functional.set_compute_dtype(torch.float16)
    try:
        norm = dict(norm_cfg=dict(type='BN2d'), activation='LeakyReLU')
        cfg = dict(local_rank=0, lr=2e-3, beta1=0.5, beta2=0.999, gan_loss_type='lsgan',
                   model=dict(G_A2B=dict(type='RDFGenerator', pretrained_on_imagenet=False),
                              G_B2A=dict(type='ResnetGenerator', input_channels=1, output_channels=3, ngf=64, norm_layer='IN2d', use_dropout=True),
                              D_A=dict(type='PatchGANDiscriminator', in_channels=1, **norm), D_B=dict(type='PatchGANDiscriminator', in_channels=3, **norm)))
        m = RDFCGAN(torch.device(DEV), False, cfg, is_train=True)
        m.train()
        drops = [d for d in m.G_B2A.modules() if isinstance(d, torch.nn.Dropout)]
        data, nA, _ = step_batch(0, 2, STEP_HP['H'], STEP_HP['W'])
        data['gt_normal'] = nA
        masks, seen = {}, []
        # (the first forward of a step; the last write of a captured step is what a replay leaves)
        for i, d in enumerate(drops):
            d.register_forward_hook(lambda mod, args, out, i=i: masks.__setitem__(i, (args[0] != 0) & (out == 0)))
        for it in range(4):
            if it == 2:
                m.enable_graph(True)
            m.set_input(data)
            m.optimize_parameters()
            torch.cuda.synchronize()
            assert len(drops) == 6 and len(masks) == 6
            step = [masks[i].clone() for i in range(6)]
            for a in range(6):
                assert 0.3 < float(step[a].float().mean()) < 0.7
                for b in range(a):
                    assert float((step[a] != step[b]).float().mean()) > 0.3, (it, a, b)
            for before in seen:
                assert all(float((p != q).float().mean()) > 0.3 for p, q in zip(before, step))
            seen.append(step)
        assert m._graph_mode and m._graphs is not None, 'capture fell back to eager launches'
        m.enable_graph(False)
    finally:
        functional.set_multi_stream(many)
        functional.set_compute_dtype(old)


def test_generator_with_dropout():
    """ResnetGenerator(use_dropout=True): training masks and scales between the two convolutions of a block, evaluation equals the
    generator without dropout"""
    from rdfc_gan_amd import functional
    from rdfc_gan_amd.generator import ResnetGenerator
    old = functional.compute_dtype()
    functional.set_compute_dtype(torch.float32)
    try:
        torch.manual_seed(0)
        a, b = (ResnetGenerator(1, 3, ngf=16, norm_layer='IN2d', use_dropout=d, n_blocks=2).to(DEV) for d in (True, False))
        b.load_state_dict({k.replace('conv_block.6', 'conv_block.5'): v for k, v in a.state_dict().items()})
        x = rnd(2, 1, 28, 36, seed=1).to(DEV).requires_grad_(True)
        assert torch.equal(a.eval()(x), b.eval()(x))
        a.train()
        torch.manual_seed(1)
        y1 = a(x)
        torch.manual_seed(1)
        y2 = a(x)
        assert torch.equal(y1, y2) and not torch.equal(y1, a(x)) and not torch.equal(y1, b.train()(x))
        gx, = torch.autograd.grad(y1, x, torch.ones_like(y1))
        assert bool(torch.isfinite(gx).all()) and bool(gx.any())
    finally:
        functional.set_compute_dtype(old)
