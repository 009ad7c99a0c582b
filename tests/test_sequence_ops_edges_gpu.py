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


# ------------------------------------------------------------------------------------------------ the norm's node
def norm_leaves(shape, dtype=torch.float32, rtype=torch.float32, seed=0):
    g = gen(seed)
    return (rnd(g, *shape).to(dtype).cuda().requires_grad_(), rnd(g, *shape).to(rtype).cuda().requires_grad_(),
            (1 + rnd(g, shape[-1], scale=0.3)).cuda().requires_grad_())


@pytest.mark.parametrize('dtype,rtype', [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
                                         (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize('shape', [(96,), (1, 96), (6, 96), (2, 3, 96), (2, 3, 1), (5, 13)])
def test_norm_gradients_in_any_layout(F, shape, dtype, rtype):
    """incoming gradients that are transposed, cut out of something wider, or one row for all: as their contiguous copies"""
    x, r, w = norm_leaves(shape, dtype, rtype)
    y, s = F.add_rms_norm(x, r, w)
    g = gen(3)
    dy, ds = rnd(g, *shape).to(dtype).cuda(), rnd(g, *shape).to(rtype).cuda()
    grads = lambda a, b: torch.autograd.grad((y, s), (x, r, w), (a, b), retain_graph=True)                # noqa: E731
    turned = lambda t: t.transpose(0, -1).contiguous().transpose(0, -1) if t.dim() > 1 else t.repeat_interleave(2)[::2]  # noqa: E731
    cut = lambda t: torch.nn.functional.pad(t, (3, 5), value=9.0)[..., 3:-5]                              # noqa: E731
    want = grads(dy, ds)
    for f in (turned, cut):
        assert torch.equal(f(dy), dy)
        # (the cut rows are no longer on 16 bytes and take the other kernel: its sums are in another order)
        for a, b in zip(want, grads(f(dy), f(ds))):
            torch.testing.assert_close(a, b, rtol=2 * HALF[a.dtype] if a.dtype != torch.float32 else 1e-5, atol=1e-5)
    row = dy.reshape(-1, shape[-1])[:1].reshape((1,) * (len(shape) - 1) + (-1,)).expand(shape)
    for a, b in zip(grads(row, ds), grads(row.contiguous(), ds)):
        torch.testing.assert_close(a, b, rtol=2 * HALF[a.dtype] if a.dtype != torch.float32 else 1e-5, atol=1e-5)


def test_norm_with_one_of_its_outputs_used(F):
    x, r, w = norm_leaves((7, 64), torch.bfloat16, torch.float32)
    y, s = F.add_rms_norm(x, r, w)
    d = torch.randn_like(s)
    dx, dr, dw = torch.autograd.grad(s, (x, r, w), d, retain_graph=True)
    assert torch.equal(dr, d) and torch.equal(dx, d.bfloat16()) and not dw.any()
    one = torch.autograd.grad(y, (x, r, w), torch.ones_like(y), retain_graph=True)
    two = torch.autograd.grad((y, s), (x, r, w), (torch.ones_like(y), torch.zeros_like(s)))
    assert all(torch.equal(a, b) for a, b in zip(one, two))


@pytest.mark.parametrize('which', [0, 1, 2])
def test_norm_with_one_leaf(F, which):
    leaves = norm_leaves((9, 64))
    y, s = F.add_rms_norm(*leaves)
    want = torch.autograd.grad((y, s), leaves, (torch.ones_like(y), torch.ones_like(s)))
    some = [t.detach() for t in leaves]
    some[which].requires_grad_()
    y, s = F.add_rms_norm(*some)
    (got,) = torch.autograd.grad((y, s), (some[which],), (torch.ones_like(y), torch.ones_like(s)))
    assert torch.equal(got, want[which])
    with torch.no_grad():
        assert not F.add_rms_norm(*leaves)[0].requires_grad
    assert not F.add_rms_norm(*(t.detach() for t in leaves))[0].requires_grad


def test_norm_of_no_rows_has_gradients(F):
    for shape in ((0, 64), (2, 0, 64)):
        x, r, w = norm_leaves(shape, torch.bfloat16, torch.float32)
        y, s = F.add_rms_norm(x, r, w)
        dx, dr, dw = torch.autograd.grad((y, s), (x, r, w), (torch.ones_like(y), torch.ones_like(s)))
        assert dx.shape == x.shape and dr.shape == r.shape and dw.shape == w.shape and not dw.any()
        q, scale, total = F.add_rms_norm_q8(x.detach(), r.detach(), w.detach())
        assert q.shape == shape and scale.shape == shape[:-1] and total.dtype == torch.float32


def test_norm_backward_twice_again_and_after_a_change(F):
    leaves = norm_leaves((5, 64))
    y, s = F.add_rms_norm(*leaves)
    d = torch.ones_like(y)
    a = torch.autograd.grad(y, leaves, d, retain_graph=True)
    b = torch.autograd.grad(y, leaves, d, retain_graph=True)
    assert all(torch.equal(u, v) for u, v in zip(a, b))
    with pytest.raises(RuntimeError, match='differentiated again'):
        torch.autograd.grad(y, leaves, d, retain_graph=True, create_graph=True)
    with torch.no_grad():
        s.add_(1.0)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        torch.autograd.grad(y, leaves, d)
    y, _ = F.add_rms_norm(leaves[0], None, leaves[2])
    with torch.no_grad():
        leaves[0].add_(1.0)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        torch.autograd.grad(y, leaves[0], d)


def test_norm_gradients_on_another_stream(F):
    leaves = norm_leaves((3000, 256))
    y, s = F.add_rms_norm(*leaves)
    want = torch.autograd.grad((y, s), leaves, (torch.ones_like(y), torch.ones_like(s)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        mine = [(t.detach() * 1.0).requires_grad_() for t in leaves]
        y, s = F.add_rms_norm(*mine)
        got = torch.autograd.grad((y, s), mine, (torch.ones_like(y), torch.ones_like(s)))
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize('packed', [False, True])
def test_encoder_that_returns_no_states_makes_none(F, monkeypatch, packed):
    m = ssm()
    x = torch.randn(*((23,) if packed else (3, 9)), 24, device='cuda')
    off = torch.tensor([0, 5, 5, 23], dtype=torch.int32, device='cuda') if packed else None
    want, states = m(x, return_sequence=True, offsets=off)
    asked = []
    for name in ('short_conv', 'selective_scan'):
        real = getattr(F, name)
        monkeypatch.setattr(F, name, lambda *a, real=real, **k: asked.append(k.get('return_state', False)) or real(*a, **k))
    m.return_states = False
    y, none = m(x, return_sequence=True, offsets=off)
    assert none is None and asked == [False] * 4 and torch.equal(y, want)


# ------------------------------------------------------------------------------------------------ roundings, quantity by quantity
def check_each(F, c):
    """Every output and gradient with the roundings of its own sums: 12 per token of the longest sequence for the decays that a
    term passes, one per summed state, 64 for step sizes and gates; where a sum runs over channels (dB, dC) or tokens (dA, dD,
    ddelta_bias), one for each of those."""
    D, N = c.cpu['A'].shape
    base = 12 * c.longest + N + 64
    more = {'B': D, 'C': D, 'A': c.T, 'D': c.T, 'bias': c.T}
    r, m = c.ref(), c.ref(True)
    flat = lambda t: t.flatten(0, 1) if c.rows else t                                  # noqa: E731
    v = {k: None if t is None else t.clone().requires_grad_() for k, t in c.gpu.items()}
    out, state = c.call(F, v)
    close('out', flat(out), r['out'], m['out'], base, HALF[c.dtype])
    close('state', state, r['state'], m['state'], base, U32)
    names = [k for k in v if v[k] is not None]
    got = torch.autograd.grad((flat(out), state), [v[k] for k in names], (c.dout.cuda(), c.dstate.cuda()))
    for k, t in zip(names, got):
        key = 'state_in' if k == 'state' else k
        close('d' + k, t, r[key], m[key], base + more.get(k, 0), HALF[t.dtype])


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('D,N,G', [(20, 16, 1), (70, 8, 2), (33, 5, 1), (24, 13, 2), (8, 1, 1)])
@pytest.mark.parametrize('lengths,tail', [([3] * 300, 0), ([64, 64, 500, 0, 1, 700, 63], 5), ([0, 900, 0], 200)])
def test_packed_gradients_over_several_chunks(F, lengths, tail, D, N, G, dtype):
    check_each(F, ScanCase(D, N, G, dtype, lengths=lengths, tail=tail, seed=N))


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('rows,D,N,G', [((2, 17), 96, 8, 3), ((3, 33), 256, 16, 1), ((2, 130), 24, 13, 1), ((1, 700), 64, 16, 1),
                                        ((2, 515), 10, 16, 1), ((1, 1025), 130, 8, 2), ((800, 70), 40, 16, 1)])
def test_roundings_of_each_quantity(F, rows, D, N, G, dtype):
    check_each(F, ScanCase(D, N, G, dtype, rows=rows, seed=3))


def test_gradients_past_2_to_the_31_elements(F):
    """the last tokens' gradient of u, in the first and the last channels, against the formulas"""
    D, T, n, N = 32768, 66000, 40, 4
    off = torch.tensor([0, 7, T - n, T], dtype=torch.int32, device='cuda')
    x = torch.zeros(T, D, dtype=torch.bfloat16, device='cuda')
    x[T - n:] = torch.randn(n, D, device='cuda').bfloat16()
    delta = x.detach()
    A = -torch.rand(D, N, device='cuda') - 0.5
    B = torch.randn(T, N, device='cuda').bfloat16()
    x = x.requires_grad_()
    out = F.selective_scan(x, delta, A, B, B, delta_softplus=True, offsets=off)
    d = torch.zeros_like(out)
    d[T - n:] = torch.randn(n, D, device='cuda').bfloat16()
    (g,) = torch.autograd.grad(out, (x,), d)
    assert not g[:T - n].any()
    for c in (slice(0, 64), slice(D - 64, D)):
        tail = lambda t: f64(t[T - n:])                                                # noqa: E731
        args = (tail(x[:, c]), tail(delta[:, c]), f64(A[c]), tail(B)[:, None], tail(B)[:, None], [0, n])
        r, m = (R.scan(*args, dout=tail(d[:, c]), size=s) for s in (False, True))
        count = 12 * n + N + 64
        close('out', out[T - n:, c], r['out'], m['out'], count, HALF[torch.bfloat16])
        close('du', g[T - n:, c], r['u'], m['u'], count, HALF[torch.bfloat16])


@pytest.mark.parametrize('form', ['clips', 'packed', 'long'])
def test_encoder_in_captured_steps(form):
    """training steps and forward passes from captured graphs, with eager work between the replays, as the eager ones"""
    from hipvae.graph import GraphedForward, GraphedTrainStep
    from hipvae.optim import FusedAdam
    off = torch.tensor([0, 9, 9, 40, 41], dtype=torch.int32, device='cuda') if form == 'packed' else None
    shape = {'clips': (5, 11, 24), 'packed': (43, 24), 'long': (1, 333, 24)}[form]
    data = [rnd(gen(k), *shape).cuda() for k in range(4)]
    loss_of = lambda m, x: {'total_loss': (m(x, offsets=off)[0] - 0.3).square().mean()}      # noqa: E731
    models_, losses = [ssm(), ssm()], []
    for m, captured in zip(models_, (False, True)):
        m.return_states = False
        opt = FusedAdam(m.parameters(), lr=1e-2)
        if captured:
            step = GraphedTrainStep(m, opt, loss_of, data[0])
            losses.append([])
            for x in data:
                losses[-1].append(float(step(x)['total_loss'].detach()))
                loss_of(models_[0], x)
        else:
            losses.append([])
            for x in data:
                opt.zero_grad(set_to_none=True)
                loss = loss_of(m, x)['total_loss']
                loss.backward()
                opt.step()
                losses[-1].append(float(loss.detach()))
                del loss
    assert losses[0] == pytest.approx(losses[1], rel=1e-6) and len(set(losses[0])) == 4
    for (k, a), b in zip(models_[0].state_dict().items(), models_[1].state_dict().values()):
        # (the captured optimizer takes its step count from device memory: its bias corrections differ in the last bits)
        assert float((a - b).abs().max()) <= 1e-6 + 1e-5 * float(a.abs().max()), k
    m = models_[0].eval()
    run = GraphedForward(m, data[0], fn=lambda m, x: m(x, return_sequence=True, offsets=off)[0])
    for x in data[::-1] + data:
        y = run(x).clone()
        with torch.no_grad():
            assert torch.equal(y, m(x, return_sequence=True, offsets=off)[0])


def test_function_transforms_are_refused(F):
    """transforms that wrap tensors: an error, never a call that ignores the wrapping"""
    x, w, a, bc = (torch.randn(*s, device='cuda') for s in ((2, 5, 8), (8, 4), (8,), (2, 5, 4)))
    calls = [lambda t: F.add_rms_norm(t, None, a)[0], lambda t: F.add_rms_norm(t, t, a)[1], lambda t: F.add_rms_norm_q8(t, None, a)[1],
             lambda t: F.short_conv(t, w), lambda t: F.selective_scan(t, t, -w.abs(), bc, bc)]
    for i, f in enumerate(calls):
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda t: f(t).sum())(x)
            pytest.fail(f'grad {i}')
        with pytest.raises(RuntimeError, match='forward-mode'):
            torch.func.jvp(f, (x,), (x,))
        with pytest.raises(RuntimeError):
            torch.vmap(f)(x[None])
            pytest.fail(f'vmap {i}')
