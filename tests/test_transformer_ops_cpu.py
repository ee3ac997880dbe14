"""The transformer-block operators without a GPU: the 64-bit oracle against published vectors, autograd and differences; every call that
the Python surface and the C ABI refuse."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import transformer_ops as O


def test_philox_known_answers():
    """the test vectors published with the generator (Random123, philox4x32-10)"""
    f = 0xffffffff
    for counter, key, want in (((0, 0, 0, 0), (0, 0), (0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8)),
                               ((f, f, f, f), (f, f), (0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd)),
                               ((0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344), (0xa4093822, 0x299f31d0),
                                (0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1))):
        got = O.philox4x32(np.array([counter], dtype=np.uint64), key)[0]
        assert tuple(int(v) for v in got) == want


def test_keep_mask_windows_and_rate():
    full = O.keep_mask(100_000, O.threshold_of(0.3), 7, 1 << 40)
    assert torch.equal(full[1237:5000], O.keep_mask(5000 - 1237, O.threshold_of(0.3), 7, 1 << 40, first=1237))
    rate = 1 - float(full.double().mean())
    assert abs(rate - 0.3) < 5 * (0.3 * 0.7 / 100_000) ** 0.5
    far = O.keep_mask(64, 1 << 15, 3, 9, first=(1 << 35) + 3)               # element indexes beyond 32 bits move the second counter word
    assert not torch.equal(far, O.keep_mask(64, 1 << 15, 3, 9, first=3))


def _rnd(*shape, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)


@pytest.mark.parametrize('layer', [False, True])
@pytest.mark.parametrize('post,pre,gated,p', [(True, True, True, 0.25), (False, True, False, 0.0), (True, False, True, 0.0), (False, False, False, 0.5)])
def test_oracle_norm_residual_gradients(layer, post, pre, gated, p):
    N, H, W, C = 2, 2, 3, 5
    x, h, dy, dn = (_rnd(N, H, W, C, seed=i) for i in range(4))
    gate, scale = (_rnd(N, C, seed=5), _rnd(C, seed=6)) if gated else (None, None)
    post = (_rnd(C, seed=7), _rnd(C, seed=8)) if post else None
    pre = (_rnd(C, seed=9), _rnd(C, seed=10)) if pre else None
    leaves = dict(x=x, h=h, gate=gate, scale=scale, post_w=post and post[0], post_b=post and post[1], pre_w=pre and pre[0], pre_b=pre and pre[1])
    leaves = {k: v.clone().requires_grad_(True) for k, v in leaves.items() if v is not None}

    def loss(v):
        from torch.nn import functional as F

        def norm(t, w, b):
            return F.layer_norm(t, (C,), w, b, 1e-5) if layer else F.rms_norm(t, (C,), w, 1e-5) + b
        u = norm(v['h'], v['post_w'], v['post_b']) if post else v['h']
        if p:
            u = u * O.dropout(torch.ones(N, H, W, C), p, 11, 12)
        for k in ('scale', 'gate'):
            if k in v:
                u = u * (v[k].view(N, 1, 1, C) if k == 'gate' else v[k])
        y = v['x'] + u
        return (y * dy).sum() + ((norm(y, v['pre_w'], v['pre_b']) * dn).sum() if pre else 0)

    got = O.norm_residual(x, h, dy, dn if pre else None, gate, scale, post, pre, layer, 1e-5, p, 11, 12)
    want = torch.autograd.grad(loss(leaves), list(leaves.values()))
    for (k, v), w in zip(leaves.items(), want):
        assert torch.allclose(got[k][0], w, rtol=1e-10, atol=1e-10), k
        e = torch.zeros_like(v.detach()).view(-1)                          # a central difference along one coordinate: error O(eps^2)
        e[0] = 1e-5
        e = e.view(v.shape)
        dif = (loss({**leaves, k: v + e}) - loss({**leaves, k: v - e})) / 2e-5
        assert abs(float(dif) - float(w.reshape(-1)[0])) < 1e-6 * (1 + abs(float(dif))), k


@pytest.mark.parametrize('name', ['silu', 'gelu', 'sigmoid', 'relu'])
def test_oracle_gated_linear_gradients(name):
    M, K, F = 5, 4, 6
    v = [_rnd(*s, seed=i).requires_grad_(True) for i, s in enumerate([(M, K), (F, K), (F, K), (F,), (F,)])]
    dz = _rnd(M, F, seed=9)
    fn = dict(silu=torch.nn.functional.silu, gelu=torch.nn.functional.gelu, sigmoid=torch.sigmoid, relu=torch.relu)[name]

    def value(x, wg, wu, bg, bu):
        return fn(x @ wg.t() + bg) * (x @ wu.t() + bu)
    got = O.gated_linear(*(t.detach() for t in v), dz, name, 0.0)
    assert torch.allclose(got['z'][0], value(*v), rtol=1e-10, atol=1e-12)
    for k, w in zip(('x', 'wg', 'wu', 'bg', 'bu'), torch.autograd.grad(value(*v), v, dz)):
        assert torch.allclose(got[k][0], w, rtol=1e-10, atol=1e-10), k
    assert torch.autograd.gradcheck(value, v)


# ---- refusals -------------------------------------------------------------------------------------------------------------
def test_dropout_refusals():
    from rdfc_gan_amd import functional as Fh
    x = torch.zeros(1, 2, 3, 8)
    for bad in (torch.zeros(2, 8), torch.zeros(1, 2, 3, 0), 3):
        with pytest.raises(ValueError):
            Fh.dropout(bad, 0.5, rng=(1, 2))
    with pytest.raises(TypeError):
        Fh.dropout(x.double(), 0.5, rng=(1, 2))
    for p in (-0.1, 1.1, float('nan')):
        with pytest.raises(ValueError, match='probability'):
            Fh.dropout(x, p, rng=(1, 2))
    for rng in ((-1, 0), (0, 1 << 64)):
        with pytest.raises(ValueError, match='64-bit'):
            Fh.dropout(x, 0.5, rng=rng)
    for rng in (None, (1, 2)):
        with pytest.raises(ValueError, match='device'):
            Fh.dropout(x, 0.5, rng=rng)
    assert Fh.dropout(x, 0.5, training=False) is x and Fh.dropout(x, 0.0) is x and Fh.dropout(x, 1e-6) is x


def test_norm_residual_refusals():
    from rdfc_gan_amd import functional as Fh
    x = torch.zeros(2, 2, 3, 8)
    w = torch.ones(8)
    for kw in (dict(h=torch.zeros(2, 2, 3, 7)), dict(h=x.half()), dict(gate=torch.ones(8)), dict(gate=torch.ones(2, 3, 8)), dict(scale=torch.ones(7)),
               dict(post=(torch.ones(7), None)), dict(pre=(w, torch.ones(9))), dict(norm='batch', pre=(w, None)), dict(eps=-1.0), dict(p=2.0),
               dict(scale=torch.ones(8, dtype=torch.int32)), dict()):
        with pytest.raises(ValueError):
            Fh.norm_residual(x, kw.pop('h', x), **kw)
    wide = torch.zeros(1, 1, 1, 8193)
    with pytest.raises(ValueError, match='8192'):
        Fh.norm_residual(wide, wide)
    with pytest.raises(ValueError, match='8192'):
        Fh.row_norm(wide)
    with pytest.raises(ValueError):
        Fh.row_norm(x, torch.ones(9))
    with pytest.raises(ValueError, match='device'):
        Fh.row_norm(x, w)


def test_gated_linear_refusals():
    from rdfc_gan_amd import functional as Fh
    x, w = torch.zeros(1, 2, 3, 8), torch.zeros(5, 8)
    b = torch.zeros(5)
    for args, kw in (((w, torch.zeros(6, 8)), {}), ((torch.zeros(5, 7),) * 2, {}), ((torch.zeros(0, 8),) * 2, {}), ((torch.zeros(5, 8, 3, 3),) * 2, {}),
                     ((w, w, b), {}), ((w, w, b, torch.zeros(4)), {}), ((w, w), dict(act='tanh')), ((w.half(), w.half()), {}), ((w, w.half()), {}),
                     ((torch.zeros(8),) * 2, {}), ((w, w, b, b), {})):
        with pytest.raises(ValueError):
            Fh.gated_linear(x, *args, **kw)
    with pytest.raises(ValueError, match='device'):
        Fh.gated_linear(x, w, w)


def test_c_abi_refusals():
    from rdfc_gan_amd import hip
    lib = hip.lib()
    err = lambda: lib.rdfc_last_error()
    assert lib.rdfc_dropout(None, None, 4, 8, 8, 8, 0, 65537, 0, 0, None, None) and b'threshold' in err()
    assert lib.rdfc_dropout(None, None, 4, 8, 7, 8, 0, 5, 0, 0, None, None) and b'bad sizes' in err()
    assert lib.rdfc_dropout(None, None, 4, 8, 8, 8, 3, 5, 0, 0, None, None) and b'dtype' in err()
    assert lib.rdfc_dropout(None, None, 4, 8, 8, 8, 0, 5, 0, 0, None, None) and b'null' in err()
    assert lib.rdfc_dropout(None, None, 0, 8, 8, 8, 0, 5, 0, 0, None, None) == 0
    assert lib.rdfc_dropout_draw(None, None, None)
    nr = lambda **k: hip.NormResidualDesc(**{**dict(rows=4, samples=2, C=8, ldx=8, ldh=8, dtype=0, pre=1, eps=1e-5), **k})
    fwd = lambda d: lib.rdfc_norm_residual(ctypes.byref(d), *[None] * 13)
    assert fwd(nr()) and b'null' in err()
    assert fwd(nr(C=8193, ldx=9000, ldh=9000)) and b'8192' in err()
    assert fwd(nr(ldx=7)) and b'ld smaller' in err()
    assert fwd(nr(threshold=-1)) and b'threshold' in err()
    assert fwd(nr(samples=70000)) and b'bad sizes' in err()
    assert fwd(nr(rows=0)) == 0
    assert lib.rdfc_norm_residual(ctypes.byref(nr()), 16, 16, *[None] * 7, 16, 16, 8, None) and b'aligned' in err()       # stats at 8
    assert lib.rdfc_norm_residual_scratch_floats(ctypes.byref(nr(C=0)), 0) == 0
    bwd = lambda d, lddy=8, lddn=8: lib.rdfc_norm_residual_backward(ctypes.byref(d), *[None] * 9, None, lddy, None, lddn, *[None] * 10)
    assert bwd(nr()) and b'null' in err()
    assert bwd(nr(rows=0)) == 0
    gl = lambda **k: hip.GatedDesc(**{**dict(M=4, K=8, F=8, ldx=8, ldwg=8, ldwu=8, dtype=1, act=16), **k})
    fwd = lambda d: lib.rdfc_gated_linear(ctypes.byref(d), *[None] * 9)
    assert fwd(gl()) and b'null' in err()
    assert fwd(gl(act=2)) and b'activation' in err()
    assert fwd(gl(ldwu=4)) and b'ld smaller' in err()
    assert fwd(gl(K=0)) and b'bad sizes' in err()
    assert fwd(gl(F=(1 << 20) + 1)) and b'bad sizes' in err()
    assert fwd(gl(F=1 << 19, K=1 << 18, ldx=1 << 18, ldwg=1 << 18, ldwu=1 << 18)) and b'too large' in err()
    assert fwd(gl(M=0)) == 0
    assert lib.rdfc_gated_linear(ctypes.byref(gl()), 16, 16, 16, None, None, None, 16, 16, None) and b'f32 maps' in err()   # pre beside a 16-bit map
    assert lib.rdfc_gated_linear(ctypes.byref(gl()), 2, 16, 16, None, None, None, 16, None, None) and b'scratch' in err()   # misaligned x, no scratch
    assert lib.rdfc_gated_linear_scratch_bytes(ctypes.byref(gl(dtype=9)), None, None, None, 0) == 0
    assert lib.rdfc_gated_linear_scratch_bytes(ctypes.byref(gl()), 16, 32, 48, 0) == 0
    assert lib.rdfc_gated_linear_scratch_bytes(ctypes.byref(gl()), 2, 32, 48, 0) == 256
    bwd = lambda d, lddz=8, dw=0: lib.rdfc_gated_linear_backward(ctypes.byref(d), *[None] * 7, lddz, None, None, None, None, dw, None, None, None)
    assert bwd(gl()) and b'null' in err()
    assert bwd(gl(), lddz=7) and b'lddz' in err()
    assert bwd(gl(), dw=2) and b'weight gradients' in err()


# ---- what reaches the C ABI: the entry points are recorded, not called -----------------------------------------------------
@pytest.fixture
def calls(monkeypatch):
    from rdfc_gan_amd import functional as Fh
    from rdfc_gan_amd import hip
    seen = []

    def record(name, t, *args):
        d = args[0]._obj if hasattr(args[0], '_obj') else None
        seen.append((name, {k: getattr(d, k) for k, _ in d._fields_} if d is not None else None, args))
    monkeypatch.setattr(hip, '_call', record)
    monkeypatch.setattr(Fh, '_check_device', lambda t, what: None)
    return seen


def _slice(shape, lead, tail):
    wide = torch.zeros(*shape[:-1], lead + shape[-1] + tail)
    return wide[..., lead:lead + shape[-1]]


# what a saved-tensor hook may do to strides: everything dense (as moving it to the host and back does), or everything a slice of something wider
RELAY = {'dense': lambda t: t.clone(memory_format=torch.contiguous_format), 'wide': lambda t: _slice(t.shape, 8, 5).copy_(t)}


@pytest.mark.parametrize('relay', list(RELAY))
def test_backward_passes_take_the_strides_of_what_hooks_return(calls, relay):
    """the strides that a backward pass hands to its kernels are those of the tensors it reads, not those of the forward call"""
    from rdfc_gan_amd import functional as Fh
    x, h = (_slice((2, 3, 5, 67), 3, 61).requires_grad_(True) for _ in range(2))
    gate, w = torch.ones(2, 67, requires_grad=True), torch.ones(67, requires_grad=True)
    with torch.autograd.graph.saved_tensors_hooks(RELAY[relay], lambda t: t):
        y, n = Fh.norm_residual(x, h, gate=gate, post=(w, None), pre=(w, None))
    torch.autograd.grad([y, n], [x, gate], [torch.zeros_like(y)] * 2)
    (_, fwd, _), (name, bwd, args) = calls
    assert fwd['ldx'] == fwd['ldh'] == 131 and name == 'rdfc_norm_residual_backward'
    assert bwd['ldx'] == bwd['ldh'] == {'dense': 67, 'wide': 80}[relay]
    calls.clear()
    wg, wu = (_slice((40, 67), 3, 61).requires_grad_(True) for _ in range(2))
    with torch.autograd.graph.saved_tensors_hooks(RELAY[relay], lambda t: t):
        z = Fh.gated_linear(x, wg, wu)
    torch.autograd.grad(z, [x, wg], torch.zeros_like(z))
    (_, fwd, _), (name, bwd, args) = calls
    assert [fwd[k] for k in ('ldx', 'ldwg', 'ldwu')] == [131] * 3 and name == 'rdfc_gated_linear_backward'
    assert [bwd[k] for k in ('ldx', 'ldwg', 'ldwu')] == [{'dense': 67, 'wide': 80}[relay]] * 3


@pytest.mark.parametrize('wrong', [lambda t: t.double() if t.is_floating_point() else t, lambda t: t[:1] if t.dim() == 4 else t], ids=['type', 'shape'])
def test_backward_passes_refuse_other_values_from_hooks(calls, wrong):
    from rdfc_gan_amd import functional as Fh
    x = torch.zeros(2, 3, 5, 8, requires_grad=True)
    w = torch.zeros(4, 8, requires_grad=True)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, wrong):
        outs = Fh.row_norm(x), Fh.gated_linear(x, w, w)
    for o in outs:
        with pytest.raises(RuntimeError, match='saved-tensor hook'):
            torch.autograd.grad(o, x, torch.zeros_like(o))


def test_calls_that_no_backward_pass_can_follow_keep_nothing_for_one(calls):
    """parameters under no_grad or inference_mode, and plain tensors: no statistics, no kept projections; with grad mode on: both"""
    from rdfc_gan_amd import functional as Fh
    x, plain = torch.zeros(2, 3, 5, 8), torch.ones(8)
    w, m = torch.nn.Parameter(torch.ones(8)), torch.nn.Parameter(torch.zeros(4, 8))

    def kept():
        calls.clear()
        Fh.norm_residual(x, x, post=(w, None), pre=(w, None))
        Fh.row_norm(x, w)
        Fh.gated_linear(x, m, m)
        return [args[-1] for _, _, args in calls]            # (the last argument of either entry point: stats, pre)
    assert None not in kept()
    for off in (torch.no_grad, torch.inference_mode):
        with off():
            assert kept() == [None] * 3
    w, m = plain, m.detach()
    assert kept() == [None] * 3


def test_dropout_draws_from_torchs_generator_through_torch(calls, monkeypatch):
    """a key drawn by a torch call: nothing sets the generator's offset, where a draw of another thread could be undone"""
    from rdfc_gan_amd import functional as Fh

    class Untouched:
        def __getattr__(self, name):
            raise AssertionError(f'{name} of a generator')
    monkeypatch.setattr(torch.cuda, 'default_generators', [Untouched()] * 8)
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: False)
    x, keys = torch.zeros(1, 2, 3, 8), []
    drop = Fh.hip.dropout
    monkeypatch.setattr(Fh.hip, 'dropout', lambda x, t, seed, offset, key: keys.append(key.clone()) or drop(x, t, seed, offset, key))
    for _ in range(2):
        torch.manual_seed(3)
        Fh.dropout(x, 0.5)
        Fh.dropout(x, 0.5)
    assert torch.equal(keys[0], keys[2]) and torch.equal(keys[1], keys[3]) and not torch.equal(keys[0], keys[1])
    assert all(k.dtype == torch.int64 and k.shape == (2,) for k in keys)


def test_scratch_sizes_are_right_and_do_not_pile_up():
    from rdfc_gan_amd import hip
    for rows in range(1, 2000):
        for gated in (False, True):
            d = hip.NormResidualDesc(rows=rows, samples=2, C=24, ldx=35, ldh=24, dtype=1, layer=1, post=1, pre=1)
            assert hip._nr_scratch(rows, 2, 24, gated) == hip.lib().rdfc_norm_residual_scratch_floats(ctypes.byref(d), int(gated)) > 0
    assert hip._nr_scratch.cache_info().currsize <= 256


def test_residual_block_with_dropout_has_upstream_indices():
    """use_dropout puts nn.Dropout(0.5) behind the first activation: the second convolution is conv_block.6"""
    from rdfc_gan_amd.generator import ResnetGenerator
    g = ResnetGenerator(1, 3, ngf=8, norm_layer='IN2d', use_dropout=True, n_blocks=1)
    keys = [k for k in g.state_dict() if 'conv_block' in k]
    assert {k.split('conv_block.')[1] for k in keys} == {'1.weight', '1.bias', '6.weight', '6.bias'}
    plain = ResnetGenerator(1, 3, ngf=8, norm_layer='IN2d', n_blocks=1)
    assert {k.split('conv_block.')[1] for k in plain.state_dict() if 'conv_block' in k} == {'1.weight', '1.bias', '5.weight', '5.bias'}


def test_unseeded_states_are_streams_of_their_own():
    from rdfc_gan_amd.functional import DropoutState
    torch.manual_seed(5)
    a, b = (DropoutState(device='cpu').state.clone() for _ in range(2))
    torch.manual_seed(5)
    c, d = (DropoutState(device='cpu').state.clone() for _ in range(2))
    assert torch.equal(a, c) and torch.equal(b, d) and int(a[0]) != int(b[0]) and int(a[1]) == int(b[1]) == 0
    assert torch.equal(DropoutState(7, 'cpu').state, DropoutState(7, 'cpu').state)


def _graph_model():
    """what enable_graph needs of an RDFCGAN: two generators, one with dropout, no optimizers"""
    from rdfc_gan_amd.generator import ResnetGenerator
    from rdfc_gan_amd.rdfc_gan import RDFCGAN
    m = RDFCGAN.__new__(RDFCGAN)
    m.use_label_net, m.G_normal, m.optimizers, m.device = False, None, {}, torch.device('cpu')
    m.G_A2B = ResnetGenerator(1, 3, ngf=8, norm_layer='IN2d', n_blocks=1)
    m.G_B2A = ResnetGenerator(1, 3, ngf=8, norm_layer='IN2d', use_dropout=True, n_blocks=4)
    return m, [d for d in m.G_B2A.modules() if isinstance(d, torch.nn.Dropout)]


def test_graph_mode_gives_every_dropout_layer_a_state_of_its_own():
    from rdfc_gan_amd import functional as Fh
    many = Fh.multi_stream()
    try:
        m, drops = _graph_model()
        own = drops[0].rng = (1, 2)
        m.enable_graph(True)
        states = [d.rng for d in drops[1:]]
        assert drops[0].rng is own and len({int(s.state[0]) for s in states}) == 3
        m.enable_graph(False)                            # eager steps follow torch's generator again
        assert drops[0].rng is own and all(d.rng is None for d in drops[1:])
        m.enable_graph(True)                             # and graph mode goes on where it was
        assert [d.rng for d in drops[1:]] == states
    finally:
        Fh.set_multi_stream(many)


def test_dropout_states_are_in_the_checkpoint(tmp_path, monkeypatch):
    """a resumed run goes on with the masks that come next, whether graph mode is on before the checkpoint is read or only afterwards"""
    from rdfc_gan_amd import functional as Fh
    many = Fh.multi_stream()

    def model():
        m, drops = _graph_model()
        m.is_train, m.scaler, m.lr_schedulers, m.models = True, None, {}, {}
        return m, drops
    try:
        m, drops = model()
        m.save_ckpt(tmp_path / 'none.pth')
        assert 'dropout_state_dict' not in torch.load(tmp_path / 'none.pth')
        drops[0].rng = Fh.DropoutState((1 << 64) - 3, 'cpu')                  # the caller's own; draws: counters move
        m.enable_graph(True)
        for i, d in enumerate(drops):
            d.rng.state[1] += 10 + i
        want = [d.rng.state.clone() for d in drops]
        m.save_ckpt(tmp_path / 'a.pth')
        for early in (True, False):
            r, drops = model()
            if early:
                r.enable_graph(True)
                held = [d.rng.state for d in drops]
            r.resume_from(tmp_path / 'a.pth')
            assert early or all(d.rng is None for d in drops)
            r.enable_graph(True)
            assert all(torch.equal(d.rng.state, w) for d, w in zip(drops, want))
            assert not early or all(d.rng.state is h for d, h in zip(drops, held))        # (in place: a captured step reads it there)
        with monkeypatch.context() as mp:                # another rank reading rank 0's file: the counters, its own seeds
            mp.setattr(torch.distributed, 'is_initialized', lambda: True)
            mp.setattr(torch.distributed, 'get_rank', lambda: 1)
            o, drops = model()
            o.enable_graph(True)
            seeds = [int(d.rng.state[0]) for d in drops]
            o.resume_from(tmp_path / 'a.pth')
            assert [d.rng.state.tolist() for d in drops] == [[s, int(w[1])] for s, w in zip(seeds, want)]
        r.enable_graph(False)
        r.save_ckpt(tmp_path / 'b.pth')                  # (graph mode is off, its states are kept)
        assert torch.load(tmp_path / 'b.pth')['dropout_state_dict'] == torch.load(tmp_path / 'a.pth')['dropout_state_dict']
    finally:
        Fh.set_multi_stream(many)
