"""The sequence operators at their edges: offsets in the wrong order, infinities where a block is filled up, forward-mode
derivatives.  Cases, references and tolerances are those of test_sequence_ops_gpu."""
import numpy as np
import pytest
import torch

import seq_reference as R
from test_sequence_ops_gpu import F, ConvCase, ScanCase, U32, HALF, close, f64, gen, rnd      # noqa: F401

pytestmark = pytest.mark.gpu


def inside_nan(t):
    """the same values in memory that is NaN before and behind them"""
    if t is None:
        return None
    pad = 4096
    big = torch.full((t.numel() + 2 * pad,), float('nan'), dtype=t.dtype, device='cuda')
    view = big[pad:pad + t.numel()].view(t.shape)
    view.copy_(t)
    return view


WRONG = [[15, 10], [2, 2], [2, 2, 40], [0, 100], [-5, 3, 2, 60], [40, 30, 20, 10, 0], [7, 0, 40], [39, 1, 39, 2, 39], [90, 80],
         [-9, -8], [0, 20, 10, 30], [13, 12, 14, 13, 15], [0, 40, 0, 40]]


@pytest.mark.parametrize('scale', [1, 7])
@pytest.mark.parametrize('off', WRONG)
def test_offsets_in_the_wrong_order_reach_nothing_outside(F, off, scale):
    """What is in a sequence then is not defined, but every value read lies in the tensors: NaN around all of them reaches
    neither the outputs nor a gradient."""
    T, S = 40 * scale, len(off) - 1
    offsets = torch.tensor(off, dtype=torch.int32, device='cuda') * scale
    for D, W, N, dtype in ((64, 4, 16, torch.bfloat16), (5, 2, 3, torch.float32), (130, 3, 8, torch.float32)):
        c = ConvCase(D, W, dtype, lengths=[T], seed=D)
        v = {k: inside_nan(t) for k, t in c.gpu.items()}
        v['state'] = inside_nan(rnd(gen(1), S, W - 1, D).to(dtype))
        v = {k: t.requires_grad_() for k, t in v.items()}
        out, state = F.short_conv(v['x'], v['weight'], v['bias'], silu=True, state=v['state'], offsets=offsets,
                                  return_state=True)
        got = torch.autograd.grad((out, state), list(v.values()),
                                  (inside_nan(c.dout), inside_nan(rnd(gen(2), S, W - 1, D).to(dtype))))
        for k, t in zip(('out', *v), (out, *got)):
            assert torch.isfinite(t).all(), ('conv', k, D, W)
        c = ScanCase(D, N, 1, dtype, lengths=[T], seed=D)
        v = {k: inside_nan(t) for k, t in c.gpu.items()}
        v['state'] = inside_nan(rnd(gen(3), S, D, N))
        v = {k: t.requires_grad_() for k, t in v.items()}
        out, state = F.selective_scan(v['u'], v['delta'], v['A'], v['B'], v['C'], D=v['D'], z=v['z'], delta_bias=v['bias'],
                                      delta_softplus=True, state=v['state'], offsets=offsets, return_state=True)
        got = torch.autograd.grad((out, state), list(v.values()), (inside_nan(c.dout), inside_nan(rnd(gen(4), S, D, N))))
        for k, t in zip(('out', *v), (out, *got)):
            assert torch.isfinite(t).all(), ('scan', k, D, N)


# ------------------------------------------------------------------------------------------------ models.SSMEncoder
def ssm(**more):
    import models
    torch.manual_seed(5)
    return models.SSMEncoder(**{**dict(input_dim=24, hidden_dim=32, num_layers=2, state_dim=8), **more}).cuda()


@pytest.mark.parametrize('shape,off', [((0, 24), [0, 0, 0]), ((3, 0, 24), None), ((0, 5, 24), None)])
def test_encoder_without_tokens(shape, off):
    """outputs of 0 and the states as they were, as the operators have it"""
    m = ssm()
    off = None if off is None else torch.tensor(off, dtype=torch.int32, device='cuda')
    n = shape[0] if off is None else len(off) - 1
    x = torch.empty(shape, device='cuda')
    y, states = m(x, offsets=off)
    assert y.shape == (n, 32) and not y.any() and len(states) == 2
    assert all(a.shape == (n, 3, 64) and b.shape == (n, 64, 8) and not a.any() and not b.any() for a, b in states)
    y, _ = m(x, return_sequence=True, offsets=off)
    assert y.shape == (*shape[:-1], 32)
    given = [(torch.randn_like(a), torch.randn_like(b)) for a, b in states]
    _, ends = m(x, states=given, offsets=off)
    for one, two in zip(given, ends):
        for a, b in zip(one, two):
            assert torch.equal(a, b) and (a is not b)


@pytest.mark.parametrize('off', [[0, 9, 60], [0, 90, 95], [20, 3, 3, 0], [-4, -2, 7]])
def test_encoder_takes_no_output_from_outside(off):
    """offsets behind the last token, before the first, in the wrong order: an output of some token, or 0"""
    m = ssm()
    x = torch.randn(40, 24, device='cuda', requires_grad=True)
    y, _ = m(x, offsets=torch.tensor(off, dtype=torch.int32, device='cuda'))
    (g,) = torch.autograd.grad(y.square().sum(), (x,))
    assert y.shape == (len(off) - 1, 32) and torch.isfinite(y).all() and torch.isfinite(g).all()
    for s in range(len(off) - 1):
        assert off[s + 1] > off[s] or not y[s].any()


# ------------------------------------------------------------------------------------------------ infinities
def same_where_finite(name, got, ref, size, count, u_out):
    """not a finite number in the same places, and close elsewhere"""
    got = f64(got)
    assert np.array_equal(np.isfinite(got), np.isfinite(ref)), (name, np.argwhere(np.isfinite(got) != np.isfinite(ref))[:4])
    ok = np.isfinite(ref)
    close(name, torch.from_numpy(got[ok]), ref[ok], size[ok], count, u_out)


@pytest.mark.parametrize('what', ['u', 'B', 'C', 'dout'])
@pytest.mark.parametrize('L,D,N', [(3, 16, 4), (8, 16, 16), (11, 70, 16), (13, 64, 8), (700, 10, 16), (515, 16, 5)])
def test_an_infinity_at_the_last_token_stays_where_the_formulas_put_it(F, L, D, N, what):
    """in the state that is kept, in that token's values; not in what has to do with the tokens before it only, such as dA"""
    for packed in (False, True):
        c = ScanCase(D, N, 1, torch.float32, rows=None if packed else (1, L), lengths=[L] if packed else None, seed=17)
        at = {'u': (L - 1, 5), 'B': (L - 1, 0, 2), 'C': (L - 1, 0, 1), 'dout': (L - 1, 5)}[what]
        for t in (c.dout,) if what == 'dout' else (c.cpu[what], c.gpu[what]):
            t[at] = float('inf')
        with np.errstate(all='ignore'):
            r, m = c.ref(), c.ref(True)
        v = {k: t.clone().requires_grad_() for k, t in c.gpu.items()}
        out, state = c.call(F, v)
        count = 12 * L + N + 64
        flat = lambda t: t if packed else t.flatten(0, 1)                              # noqa: E731
        same_where_finite('out', flat(out), r['out'], m['out'], count, U32)
        same_where_finite('state', state, r['state'], m['state'], count, U32)
        if what in ('u', 'B'):
            assert np.array_equal(np.isinf(f64(state)), np.isinf(r['state']))
        got = torch.autograd.grad((flat(out), state), list(v.values()), (c.dout.cuda(), c.dstate.cuda()))
        for k, t in zip(v, got):
            key = 'state_in' if k == 'state' else k
            same_where_finite('d' + k, t, r[key], m[key], count + L + D, U32)
