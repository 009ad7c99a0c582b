"""selective_scan, short_conv and add_rms_norm against 64-bit restatements, token by token.

Tolerances count roundings.  u32 = 2^-24 is half a step of fp32, u = eps/2 of the output's type.  The reference also gives
the size M of what is summed (every term by its absolute value).  A term of a scan passes at most L multiplications by a
decay; one such step rounds the product with the step size (twice, A enters scaled by log2 e), the exponential (one whole
step) and the fused multiply-add, and the step size itself carries softplus's few roundings, which reach the decay times
|dt A| < 1 of a term that still counts: 12 u32 a step are more than that.  Sums over a row's channels, tokens or rows add
one rounding per term.  So an output is off by at most (12 L + terms + 64) u32 M + u |value|.
"""
import numpy as np
import pytest
import torch

import seq_reference as R

pytestmark = pytest.mark.gpu
U32 = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


@pytest.fixture(scope='module')
def F():
    from hipvae import functional
    assert torch.cuda.is_available()
    return functional


def gen(seed):
    return torch.Generator().manual_seed(seed)


def rnd(g, *shape, scale=1.0):
    return torch.randn(*shape, generator=g) * scale


def f64(t):
    return None if t is None else t.detach().cpu().double().numpy()


def close(name, got, ref, size, count, u_out):
    got = f64(got)
    assert got.shape == ref.shape, (name, got.shape, ref.shape)
    bound = count * U32 * size + u_out * np.abs(ref) + 1e-37
    bad = ~(np.abs(got - ref) <= bound)
    assert not bad.any(), (name, int(bad.sum()), bad.size, float(np.nanmax(np.abs(got - ref) / bound)),
                           np.argwhere(bad)[:3].tolist())


def offsets_of(lengths):
    return [0] + np.cumsum(lengths).tolist()


class ScanCase:
    """inputs of a scan, as tokens [T, ...] on the GPU; rows: (B, L), or lengths with a tail of tokens in no sequence"""

    def __init__(self, D, N, G, dtype, rows=None, lengths=None, tail=0, seed=0, state=True, D_=True, z=True, bias=True,
                 plus=True, delta_scale=1.0):
        g = gen(seed)
        self.rows, self.dtype, self.plus = rows, dtype, plus
        lens = [rows[1]] * rows[0] if rows else lengths
        self.off = offsets_of(lens)
        T, S = self.off[-1] + tail, len(lens)
        self.T, self.S, self.longest = T, S, max(lens + [1])
        q = lambda t: t.to(dtype)                                                     # noqa: E731
        v = dict(u=q(rnd(g, T, D)), delta=q(rnd(g, T, D, scale=delta_scale) - (0 if plus else 0.2)),
                 A=-torch.exp(rnd(g, D, N, scale=0.5)), B=q(rnd(g, T, G, N)), C=q(rnd(g, T, G, N)))
        if not plus:
            v['delta'] = q(v['delta'].float().abs() * 0.3)
        v['D'] = rnd(g, D) if D_ else None
        v['z'] = q(rnd(g, T, D)) if z else None
        v['bias'] = rnd(g, D, scale=0.5) - 1 if bias else None
        if bias and not plus:
            v['bias'] = v['bias'].abs() * 0.1
        v['state'] = rnd(g, S, D, N) if state else None
        self.dout, self.dstate = q(rnd(g, T, D)), rnd(g, S, D, N)
        self.cpu = v
        self.gpu = {k: None if t is None else t.cuda() for k, t in v.items()}
        self.offsets = None if rows else torch.tensor(self.off, dtype=torch.int32, device='cuda')

    def lead(self, t):
        return t if t is None or not self.rows else t.unflatten(0, self.rows)

    def call(self, F, v, state=True, **kw):
        L = self.lead
        return F.selective_scan(L(v['u']), L(v['delta']), v['A'], L(v['B']), L(v['C']), D=v['D'], z=L(v['z']),
                                delta_bias=v['bias'], delta_softplus=self.plus, state=v['state'], offsets=self.offsets,
                                return_state=state, **kw)

    def ref(self, size=False, grads=True, dstate=True):
        c = self.cpu
        return R.scan(f64(c['u']), f64(c['delta']), f64(c['A']), f64(c['B']), f64(c['C']), self.off, f64(c['D']),
                      f64(c['z']), f64(c['bias']), self.plus, f64(c['state']), f64(self.dout) if grads else None,
                      f64(self.dstate) if grads and dstate else None, size)

    def check(self, F, grads=True):
        count = 12 * self.longest + self.T + self.cpu['u'].shape[1] + 64
        r, m = self.ref(grads=grads), self.ref(True, grads)
        flat = lambda t: t.flatten(0, 1) if self.rows else t                          # noqa: E731
        if not grads:
            out, state = self.call(F, self.gpu)
            close('out', flat(out), r['out'], m['out'], count, HALF[self.dtype])
            close('state', state, r['state'], m['state'], count, U32)
            return
        v = {k: None if t is None else t.clone().requires_grad_() for k, t in self.gpu.items()}
        out, state = self.call(F, v)
        close('out', flat(out), r['out'], m['out'], count, HALF[self.dtype])
        close('state', state, r['state'], m['state'], count, U32)
        names = [k for k in v if v[k] is not None]
        got = torch.autograd.grad((flat(out), state), [v[k] for k in names], (self.dout.cuda(), self.dstate.cuda()))
        for k, t in zip(names, got):
            key = 'state_in' if k == 'state' else k
            assert t.dtype == v[k].dtype and t.shape == v[k].shape
            close('d' + k, t, r[key], m[key], count, HALF[t.dtype])


SHAPES = [  # (B, L), channels, states, groups
    ((1, 1), 1, 1, 1), ((2, 1), 64, 16, 1), ((3, 7), 5, 4, 1), ((2, 8), 128, 16, 2), ((1, 9), 130, 16, 1),
    ((2, 17), 96, 8, 3), ((1, 65), 70, 5, 2), ((3, 33), 256, 16, 1), ((2, 130), 24, 13, 1),
]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('rows,D,N,G', SHAPES)
def test_scan_and_gradients(F, rows, D, N, G, dtype):
    ScanCase(D, N, G, dtype, rows=rows).check(F)


@pytest.mark.parametrize('off', ['state', 'D_', 'z', 'bias', 'plus', 'all'])
def test_scan_without_its_optional_parts(F, off):
    names = ['state', 'D_', 'z', 'bias', 'plus'] if off == 'all' else [off]
    ScanCase(40, 16, 1, torch.float32, rows=(2, 19), **{k: False for k in names}).check(F)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('lengths,tail', [([5, 0, 3, 1, 16, 0], 0), ([0, 0, 7], 3), ([1] * 19, 0), ([40, 9], 11),
                                          ([0], 4), ([8, 8, 0, 8], 8), ([100, 3, 61], 1)])
def test_scan_packed(F, lengths, tail, dtype):
    ScanCase(72, 16, 2, dtype, lengths=lengths, tail=tail).check(F)


# few channels and a long axis: the time axis is split over workgroups and joined
LONG = [((1, 700), 64, 16, 1), ((2, 515), 10, 16, 1), ((1, 1025), 130, 8, 2), ((1, 4100), 3, 16, 1)]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('rows,D,N,G', LONG)
def test_scan_long(F, rows, D, N, G, dtype):
    ScanCase(D, N, G, dtype, rows=rows).check(F)


@pytest.mark.parametrize('lengths,tail', [([1500], 0), ([64, 64, 500, 0, 1, 700, 63], 5), ([3] * 300, 0),
                                          ([0, 900, 0], 200), ([511, 513, 1, 1, 0, 31], 0)])
def test_scan_long_packed(F, lengths, tail):
    ScanCase(20, 16, 1, torch.float32, lengths=lengths, tail=tail).check(F)


def test_scan_reads_strided_views_and_writes_nothing_into_them(F):
    c = ScanCase(64, 16, 2, torch.bfloat16, rows=(2, 21), seed=3)
    want, wstate = c.call(F, c.gpu)
    v = dict(c.gpu)
    both = torch.full((c.T, 3 * 64 + 1), 7.0, dtype=c.dtype, device='cuda')           # odd row length: 2-byte alignment
    both[:, 64:128], both[:, 128:192] = v['u'], v['z']
    proj = torch.full((c.T, 5 + 4 * 16), 7.0, dtype=c.dtype, device='cuda')
    proj[:, 5:37], proj[:, 37:] = v['B'].flatten(1), v['C'].flatten(1)
    keep = both.clone(), proj.clone(), v['state'].clone()
    v['u'], v['z'] = both[:, 64:128], both[:, 128:192]
    v['B'], v['C'] = proj[:, 5:37].unflatten(1, (2, 16)), proj[:, 37:].unflatten(1, (2, 16))
    v['delta'] = v['delta'].t().contiguous().t()                                      # channels not contiguous: copied
    out, state = c.call(F, v)
    assert torch.equal(out, want) and torch.equal(state, wstate)
    assert torch.equal(both, keep[0]) and torch.equal(proj, keep[1]) and torch.equal(v['state'], keep[2])


def test_scan_broadcast_inputs_get_summed_gradients(F):
    """one row of B for every token (stride 0), one u for the whole batch: autograd sums the expanded gradients"""
    c = ScanCase(32, 8, 1, torch.float32, rows=(3, 11), seed=4)
    v = dict(c.gpu)
    b1 = v['B'][:1].clone().requires_grad_()
    u1 = v['u'][:11].clone().requires_grad_()
    full = dict(v, B=b1.expand(c.T, 1, 8), u=u1[None].expand(3, 11, 32).reshape(33, 32))
    plain = dict(v, B=full['B'].detach().clone().requires_grad_(), u=full['u'].detach().clone().requires_grad_())
    o1, o2 = c.call(F, full, False), c.call(F, plain, False)
    assert torch.equal(o1, o2)
    d = torch.ones_like(o1)
    gb, gu = torch.autograd.grad(o1, (b1, u1), d)
    hb, hu = torch.autograd.grad(o2, (plain['B'], plain['u']), d)
    torch.testing.assert_close(gb, hb.sum(0, keepdim=True), rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(gu, hu.view(3, 11, 32).sum(0), rtol=1e-5, atol=1e-5)


def test_scan_sequences_do_not_see_each_other_or_the_tail(F):
    """a NaN in one sequence stays there; NaN behind the last sequence reaches nothing, the parameters' gradients
    included"""
    c = ScanCase(40, 16, 1, torch.float32, lengths=[9, 13, 8], tail=6, seed=5)
    want, wstate = c.call(F, c.gpu)
    v = {k: None if t is None else t.clone() for k, t in c.gpu.items()}
    for k in ('u', 'delta', 'z', 'B', 'C'):
        v[k][30:] = float('nan')
    out, state = c.call(F, v)
    assert torch.equal(out, want) and torch.equal(state, wstate) and not out[30:].any()
    leaf = {k: t.clone().requires_grad_() for k, t in v.items()}
    o = c.call(F, leaf, False)
    for k, g in zip(leaf, torch.autograd.grad(o, list(leaf.values()), torch.full_like(o, 0.5).index_fill(
            0, torch.arange(30, 36, device='cuda'), float('nan')))):
        assert torch.isfinite(g).all(), k
        if k in ('u', 'delta', 'z', 'B', 'C'):
            assert not g[30:].any(), k
    v['u'][12] = float('nan')
    out, state = c.call(F, v)
    assert torch.equal(out[:9], want[:9]) and torch.equal(out[22:30], want[22:30])
    assert out[12:22].isnan().all() and torch.equal(out[9:12], want[9:12])
    assert torch.equal(state[0], wstate[0]) and torch.equal(state[2], wstate[2]) and state[1].isnan().all()


def test_scan_step_sizes_at_the_ends_of_softplus(F):
    """delta + bias from -80 to 80: step sizes from e^-80 (as good as none) to 80 (the state forgotten at once)"""
    c = ScanCase(33, 16, 1, torch.float32, rows=(1, 23), seed=6)
    for d in (c.cpu, c.gpu):
        d['delta'] = (torch.linspace(-80, 80, c.T * 33).view(c.T, 33)).to(d['delta'].device)
        d['bias'] = torch.zeros_like(d['bias'])
    c.check(F)


def test_scan_of_nothing(F):
    for shape in ((0, 5), (3, 0)):
        c = ScanCase(16, 4, 1, torch.float32, rows=shape)
        v = {k: t.clone().requires_grad_() for k, t in c.gpu.items()}
        out, state = c.call(F, v)
        assert out.shape == (*shape, 16)
        assert torch.equal(state, v['state'])
        g = torch.autograd.grad((out, state), list(v.values()), (torch.ones_like(out), torch.ones_like(state)))
        assert all(a.shape == b.shape for a, b in zip(g, v.values()))
        assert all(not a.any() for k, a in zip(v, g) if k != 'state') and torch.equal(g[-1], torch.ones_like(state))


def test_scan_packed_nothing(F):
    c = ScanCase(16, 4, 1, torch.float32, lengths=[0, 0])
    out, state = c.call(F, c.gpu)
    assert out.shape == (0, 16) and torch.equal(state, c.gpu['state'])
    x, w = torch.empty(0, 16, device='cuda'), torch.randn(16, 4, device='cuda')
    out, state = F.short_conv(x, w, offsets=c.offsets, return_state=True)
    assert out.shape == (0, 16) and not state.any() and state.shape == (2, 3, 16)


def test_scan_gradients_from_the_state_alone(F):
    """only the final states are used: the same gradients as with an output gradient of zeros"""
    c = ScanCase(24, 16, 1, torch.float32, lengths=[9, 0, 40, 3], tail=2, seed=9)
    names = list(c.gpu)
    res = []
    for both in (False, True):
        v = {k: t.clone().requires_grad_() for k, t in c.gpu.items()}
        out, state = c.call(F, v)
        outs, grads = ((out, state), (torch.zeros_like(out), c.dstate.cuda())) if both else ((state,), (c.dstate.cuda(),))
        res.append(torch.autograd.grad(outs, [v[k] for k in names], grads))
    for k, a, b in zip(names, *res):
        assert torch.equal(a, b), k
    assert torch.equal(res[0][-1][1], c.dstate.cuda()[1])                             # the empty sequence passes it on


def test_scan_infinite_inputs_and_rates(F):
    """lengths that end inside a block of eight: what fills the block up must not turn infinities into NaN.  An infinite
    rate forgets everything at once: as a rate so large that exp underflows."""
    for L in (3, 11):
        c = ScanCase(16, 4, 1, torch.float32, rows=(1, L), seed=12, z=False)
        v = {k: None if t is None else t.clone() for k, t in c.gpu.items()}
        v['A'][3] = float('-inf')
        w = dict(v, A=v['A'].clone())
        w['A'][3] = -1e30
        (o1, s1), (o2, s2) = c.call(F, v), c.call(F, w)
        assert torch.equal(o1, o2) and torch.equal(s1, s2) and torch.isfinite(o1).all()
        v = {k: None if t is None else t.clone() for k, t in c.gpu.items()}
        v['u'][L - 1, 5] = float('inf')
        v['B'] = v['B'].abs() + 0.1
        _, s = c.call(F, v)
        assert torch.isposinf(s[0, 5]).all() and torch.isfinite(s[0, :5]).all() and torch.isfinite(s[0, 6:]).all()


def test_a_second_backward_and_a_changed_input(F):
    c = ScanCase(24, 8, 1, torch.float32, rows=(2, 12), seed=10)
    v = {k: t.clone().requires_grad_() for k, t in c.gpu.items()}
    out = c.call(F, v, False)
    d = torch.ones_like(out)
    a = torch.autograd.grad(out, list(v.values()), d, retain_graph=True)
    b = torch.autograd.grad(out, list(v.values()), d, retain_graph=True)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    with pytest.raises(RuntimeError, match='differentiated again'):
        torch.autograd.grad(out, list(v.values()), d, retain_graph=True, create_graph=True)
    with torch.no_grad():
        v['delta'].add_(1.0)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        torch.autograd.grad(out, list(v.values()), d)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('rows,D,N,G', [(1, 1, 1, 1), (3, 96, 16, 2), (5, 70, 5, 1), (33, 512, 16, 1), (2, 64, 12, 1)])
def test_scan_steps_follow_the_scan(F, rows, D, N, G, dtype):
    L = 5
    c = ScanCase(D, N, G, dtype, rows=(rows, L), seed=7)
    v = c.gpu
    r, m = c.ref(grads=False), c.ref(True, grads=False)
    state = v['state'].clone()
    outs = []
    for t in range(L):
        at = lambda k: c.lead(v[k])[:, t]                                             # noqa: E731
        outs.append(F.selective_scan_step(state, at('u'), at('delta'), v['A'], at('B'), at('C'), D=v['D'], z=at('z'),
                                          delta_bias=v['bias'], delta_softplus=True))
    count = 12 * L + 64 + N
    close('out', torch.stack(outs, 1).flatten(0, 1), r['out'], m['out'], count, HALF[dtype])
    close('state', state, r['state'], m['state'], count, U32)
    bare = v['state'].clone()
    o = F.selective_scan_step(bare, c.lead(v['u'])[:, 0], c.lead(v['delta'])[:, 0].abs(), v['A'], c.lead(v['B'])[:, 0],
                              c.lead(v['C'])[:, 0])
    c1 = c.cpu
    rr = [R.scan(f64(c.lead(c1['u'])[:, 0]), f64(c.lead(c1['delta'])[:, 0].abs()), f64(c1['A']), f64(c.lead(c1['B'])[:, 0]),
                 f64(c.lead(c1['C'])[:, 0]), list(range(rows + 1)), plus=False, state=f64(c1['state']), size=s)
          for s in (False, True)]
    close('bare out', o, rr[0]['out'], rr[1]['out'], count, HALF[dtype])


# ------------------------------------------------------------------------------------------------ short convolution
class ConvCase:
    def __init__(self, D, W, dtype, rows=None, lengths=None, tail=0, seed=0, state=True, bias=True, act=True):
        g = gen(seed + 100)
        self.rows, self.dtype, self.act = rows, dtype, act
        lens = [rows[1]] * rows[0] if rows else lengths
        self.off = offsets_of(lens)
        self.T, self.S = self.off[-1] + tail, len(lens)
        v = dict(x=rnd(g, self.T, D).to(dtype), weight=rnd(g, D, W), bias=rnd(g, D) if bias else None,
                 state=rnd(g, self.S, W - 1, D).to(dtype) if state else None)
        self.dout, self.dstate = rnd(g, self.T, D).to(dtype), rnd(g, self.S, W - 1, D).to(dtype)
        self.cpu, self.gpu = v, {k: None if t is None else t.cuda() for k, t in v.items()}
        self.offsets = None if rows else torch.tensor(self.off, dtype=torch.int32, device='cuda')

    def call(self, F, v, state=True):
        x = v['x'].unflatten(0, self.rows) if self.rows else v['x']
        return F.short_conv(x, v['weight'], v['bias'], silu=self.act, state=v['state'], offsets=self.offsets,
                            return_state=state)

    def ref(self, size=False):
        c = self.cpu
        return R.conv(f64(c['x']), f64(c['weight']), self.off, f64(c['bias']), self.act, f64(c['state']), f64(self.dout),
                      f64(self.dstate), size)

    def check(self, F):
        # W products and the sum, the sigmoid's few roundings (its reciprocal and exponential one step each), and one
        # rounding per summed token in the weights' gradients
        count = 32 + self.T
        r, m = self.ref(), self.ref(True)
        flat = lambda t: t.flatten(0, 1) if self.rows else t                          # noqa: E731
        v = {k: None if t is None else t.clone().requires_grad_() for k, t in self.gpu.items()}
        out, state = self.call(F, v)
        close('out', flat(out), r['out'], m['out'], count, HALF[self.dtype])
        assert np.array_equal(f64(state), r['state'])                                 # copies
        names = [k for k in v if v[k] is not None]
        got = torch.autograd.grad((flat(out), state), [v[k] for k in names], (self.dout.cuda(), self.dstate.cuda()))
        for k, t in zip(names, got):
            key = 'state_in' if k == 'state' else k
            close('d' + k, t, r[key], m[key], count, HALF[t.dtype])
        with torch.no_grad():
            o2, s2 = self.call(F, self.gpu)
        assert torch.equal(o2, out) and torch.equal(s2, state)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('W', [2, 3, 4])
@pytest.mark.parametrize('rows,D', [((1, 1), 1), ((3, 2), 8), ((2, 16), 64), ((5, 20), 130), ((1, 77), 520), ((2, 65), 24)])
def test_conv_and_gradients(F, rows, D, W, dtype):
    ConvCase(D, W, dtype, rows=rows).check(F)


@pytest.mark.parametrize('off', ['state', 'bias', 'act', 'all'])
def test_conv_without_its_optional_parts(F, off):
    names = ['state', 'bias', 'act'] if off == 'all' else [off]
    ConvCase(48, 4, torch.float32, rows=(2, 19), **{k: False for k in names}).check(F)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('D', [64, 13])
@pytest.mark.parametrize('lengths,tail', [([5, 0, 3, 1, 16, 0], 0), ([0, 0, 7], 3), ([1] * 19, 0), ([2, 1, 2, 40, 9], 11),
                                          ([0], 4), ([16, 16, 0, 32, 64, 1], 70), ([15, 17, 31, 33], 0)])
def test_conv_packed(F, lengths, tail, D, dtype):
    ConvCase(D, 4, dtype, lengths=lengths, tail=tail).check(F)


def test_conv_reads_strided_views(F):
    for start in (8, 3):                               # rows on 16 bytes, and not
        c = ConvCase(64, 4, torch.bfloat16, rows=(2, 21), seed=3)
        want, wstate = c.call(F, c.gpu)
        both = torch.full((c.T, 200), 7.0, dtype=c.dtype, device='cuda')
        both[:, start:start + 64] = c.gpu['x']
        out, state = c.call(F, dict(c.gpu, x=both[:, start:start + 64]))
        assert torch.equal(out, want) and torch.equal(state, wstate)
        swapped = c.gpu['x'].unflatten(0, (2, 21)).transpose(0, 1).contiguous().transpose(0, 1)      # length-major
        out = F.short_conv(swapped, c.gpu['weight'], c.gpu['bias'], silu=True, state=c.gpu['state'])
        assert torch.equal(out, want)


def test_conv_sequences_do_not_see_each_other_or_the_tail(F):
    c = ConvCase(24, 4, torch.float32, lengths=[9, 13, 8], tail=6, seed=5)
    want, _ = c.call(F, c.gpu)
    v = {k: t.clone() for k, t in c.gpu.items()}
    v['x'][30:] = float('nan')
    leaf = {k: t.clone().requires_grad_() for k, t in v.items()}
    out = c.call(F, leaf, False)
    assert torch.equal(out, want) and not out[30:].any()
    d = torch.ones_like(out)
    d[30:] = float('nan')
    for k, g in zip(leaf, torch.autograd.grad(out, list(leaf.values()), d)):
        assert torch.isfinite(g).all(), k
    v['x'][8] = float('inf')
    out, _ = c.call(F, v)
    assert torch.equal(out[:8], want[:8]) and torch.equal(out[9:30], want[9:30])


def test_conv_of_nothing(F):
    for shape in ((0, 5), (3, 0)):
        c = ConvCase(16, 3, torch.float32, rows=shape)
        v = {k: t.clone().requires_grad_() for k, t in c.gpu.items()}
        out, state = c.call(F, v)
        assert out.shape == (*shape, 16) and torch.equal(state, v['state'])
        g = torch.autograd.grad((out, state), list(v.values()), (torch.ones_like(out), torch.ones_like(state)))
        assert not g[1].any() and not g[2].any() and torch.equal(g[3], torch.ones_like(state))


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('rows,D,W', [(1, 1, 2), (3, 64, 4), (5, 70, 3), (33, 512, 4)])
def test_conv_steps_follow_the_convolution(F, rows, D, W, dtype):
    c = ConvCase(D, W, dtype, rows=(rows, 6), seed=7)
    r, m = c.ref(), c.ref(True)
    state = c.gpu['state'].clone()
    x = c.gpu['x'].unflatten(0, c.rows)
    outs = [F.short_conv_step(state, x[:, t], c.gpu['weight'], c.gpu['bias'], silu=True) for t in range(6)]
    close('out', torch.stack(outs, 1).flatten(0, 1), r['out'], m['out'], 32, HALF[dtype])
    assert np.array_equal(f64(state), r['state'])


# ------------------------------------------------------------------------------------------------ norm
NORM_SHAPES = [(1, 1), (3, 8), (5, 130), (7, 512), (2, 1001), (33, 2048), (4, 4096), (3, 4104), (2, 5000), (130, 64)]
MIXES = [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32)]


@pytest.mark.parametrize('dtype,rtype', MIXES)
@pytest.mark.parametrize('rows,D', NORM_SHAPES)
def test_norm_and_gradients(F, rows, D, dtype, rtype):
    g = gen(rows + D)
    x, r = rnd(g, rows, D).to(dtype), rnd(g, rows, D, scale=3).to(rtype)
    w, eps = 1 + rnd(g, D, scale=0.3), 1e-5
    dy, ds = rnd(g, rows, D).to(dtype), rnd(g, rows, D).to(rtype)
    total = (x.float() + r.float()).to(rtype)                                         # one rounding: exact to compare
    ref, size = (R.norm(f64(total), f64(w), eps, f64(dy), f64(ds), s) for s in (False, True))
    xg, rg, wg = (t.cuda().requires_grad_() for t in (x, r, w))
    y, s = F.add_rms_norm(xg, rg, wg, eps)
    assert y.dtype == dtype and s.dtype == rtype and torch.equal(s.detach().cpu(), total)
    count = 16 + D + rows                                                             # one rounding per summed term
    close('y', y, ref['y'], size['y'], count, HALF[dtype])
    dx, dr, dw = torch.autograd.grad((y, s), (xg, rg, wg), (dy.cuda(), ds.cuda()))
    assert dx.dtype == dtype and dr.dtype == rtype
    close('dx', dx, ref['x'], size['x'], count, HALF[dtype])
    close('dresidual', dr, ref['x'], size['x'], count, HALF[rtype])
    close('dweight', dw, ref['weight'], size['weight'], count, U32)
    with torch.no_grad():
        y2, s2 = F.add_rms_norm(xg, rg, wg, eps)
    assert torch.equal(y, y2) and torch.equal(s, s2)
    # only the norm's output used; no residual
    ref0 = R.norm(f64(x), f64(w), eps, f64(dy))
    size0 = R.norm(f64(x), f64(w), eps, f64(dy), size=True)
    y3, s3 = F.add_rms_norm(xg, None, wg, eps)
    assert s3 is xg
    close('y without residual', y3, ref0['y'], size0['y'], count, HALF[dtype])
    (dx,) = torch.autograd.grad(y3, (xg,), dy.cuda())
    close('dx without residual', dx, ref0['x'], size0['x'], count, HALF[dtype])


def test_norm_gradients_of_the_leaves_do_not_share_memory(F):
    x, r = (torch.randn(4, 64, device='cuda').requires_grad_() for _ in range(2))
    w = torch.ones(64, device='cuda', requires_grad=True)
    for _ in range(2):                                                                # the second adds to the first
        y, s = F.add_rms_norm(x, r, w)
        (y.sum() + (s * 2).sum()).backward()
    assert x.grad.data_ptr() != r.grad.data_ptr()
    torch.testing.assert_close(x.grad, r.grad, rtol=0, atol=0)


def test_norm_of_a_tensor_with_itself_as_residual(F):
    x = torch.randn(5, 64, device='cuda', requires_grad=True)
    y0 = x.detach().clone().requires_grad_()
    w = torch.rand(64, device='cuda') + 0.5
    y, s = F.add_rms_norm(x, x, w)
    dy, ds = torch.randn_like(y), torch.randn_like(y)
    (g,) = torch.autograd.grad((y, s), (x,), (dy, ds))
    a, b = F.add_rms_norm(y0, x.detach(), w)
    (h,) = torch.autograd.grad((a, b), (y0,), (dy, ds))
    assert torch.equal(g, h + h)


def test_norm_reads_strided_rows_and_any_leading_shape(F):
    g = gen(1)
    big = rnd(g, 6, 5, 200).cuda()
    r = rnd(g, 6, 5, 64).cuda()
    w = (1 + rnd(g, 64)).cuda()
    for start in (64, 3):
        y, s = F.add_rms_norm(big[..., start:start + 64], r, w)
        y0, s0 = F.add_rms_norm(big[..., start:start + 64].contiguous(), r, w)
        torch.testing.assert_close(y, y0, rtol=1e-6, atol=1e-6)
        assert torch.equal(s, s0) and y.shape == (6, 5, 64)
    y, s = F.add_rms_norm(r[:0], r[:0], w)
    assert y.shape == (0, 5, 64) and s.shape == (0, 5, 64)


@pytest.mark.parametrize('dtype,rtype', MIXES)
@pytest.mark.parametrize('rows,D', [(1, 1), (3, 8), (5, 130), (2, 1001), (33, 2048), (3, 4104)])
def test_norm_in_8_bits(F, rows, D, dtype, rtype):
    g = gen(rows * D)
    x, r = rnd(g, rows, D).to(dtype), rnd(g, rows, D).to(rtype)
    w = 1 + rnd(g, D, scale=0.3)
    if rows > 2:
        x[1], r[1] = 0, 0
    q, scale, s = F.add_rms_norm_q8(x.cuda(), r.cuda(), w.cuda(), 1e-5)
    total = (x.float() + r.float()).to(rtype)
    assert torch.equal(s.cpu(), total) and q.dtype == torch.float8_e4m3fn and scale.shape == (rows,)
    y = R.norm(f64(total), f64(w), 1e-5)['y']
    most = np.abs(y).max(1)
    want = np.where(most > 0, most / 448, 1.0)
    assert np.all(np.abs(f64(scale) - want) <= (D + 16) * U32 * want)
    # half a step of e4m3 (2^-4 of the value; 2^-10 below its smallest normal 2^-6), after the fp32 roundings before it
    val = y / want[:, None]
    err = np.abs(f64(q.float()) - val)
    assert np.all(err <= 2.0 ** -4 * np.abs(val) * (1 + 1e-3) + 2.0 ** -10 + (D + 32) * U32 * 448)
    if rows > 2:
        assert not q[1].float().any() and scale[1] == 1


@pytest.mark.parametrize('rows,D', [((1 << 23) + 5, 3), ((1 << 25) + 6, 4)])
def test_norm_of_more_rows_than_one_launch_takes(F, rows, D):
    """the last rows, and those on both sides of the border between launches, as they are alone; dw against 64 bits"""
    x, w = torch.randn(rows, D, device='cuda').requires_grad_(), (torch.rand(D, device='cuda') + 0.5).requires_grad_()
    r = torch.randn(rows, D, device='cuda')
    border = 1 << rows.bit_length() - 1
    pick = torch.cat([torch.arange(9), torch.arange(border - 4, rows)]).cuda()
    y, s = F.add_rms_norm(x, r, w)
    dy = torch.randn(rows, D, device='cuda')
    dx, dw = torch.autograd.grad((y, s), (x, w), (dy, dy))
    x1 = x.detach()[pick].requires_grad_()
    y1, s1 = F.add_rms_norm(x1, r[pick], w)
    (dx1,) = torch.autograd.grad((y1, s1), (x1,), (dy[pick], dy[pick]))
    assert torch.equal(y[pick], y1) and torch.equal(s[pick], s1) and torch.equal(dx[pick], dx1)
    v = s.detach().double()
    terms = dy.double() * v * torch.rsqrt((v * v).mean(1, keepdim=True) + 1e-6)
    # D + 16 roundings per term; a term is then added at most rows / 2048 times within a wave (or 64 times, and to less than
    # rows / 8192 partial sums before its own), and the partial sums of that less than a thousand times more
    count = D + 16 + rows // 2048 + 4096
    assert ((dw.double() - terms.sum(0)).abs() <= count * U32 * terms.abs().sum(0)).all()
    q, scale, _ = F.add_rms_norm_q8(x.detach(), r, w.detach())
    q1, scale1, _ = F.add_rms_norm_q8(x1.detach(), r[pick], w.detach())
    assert torch.equal(q[pick].view(torch.uint8), q1.view(torch.uint8)) and torch.equal(scale[pick], scale1)


@pytest.mark.parametrize('D', [64, 13])
def test_norm_in_8_bits_of_the_smallest_numbers(F, D):
    """rows whose largest value, over 448, is below the smallest normal number"""
    g = gen(D)
    sizes = 2.0 ** -torch.arange(110, 149).float()
    x, w = torch.rand(39, D, generator=g) + 0.5, torch.ones(D)
    for i, s in enumerate(sizes):
        q, scale, _ = F.add_rms_norm_q8(x[i:i + 1].cuda(), None, (w * s).cuda(), 1e-5)
        y = R.norm(f64(x[i:i + 1]), f64(w * s), 1e-5)['y']
        got = f64(q.float()) * f64(scale)[:, None]
        # half a step of e4m3, relative or of its smallest numbers (2^-10 of the scale); y itself has a step of 2^-149
        bound = 2.0 ** -4 * np.abs(y) * (1 + 1e-3) + 2.0 ** -10 * f64(scale)[:, None] + 2.0 ** -149
        assert np.all(np.abs(got - y) <= bound) and scale.item() >= 2.0 ** -126, float(s)


def test_norm_rows_with_what_is_not_a_number(F):
    g = gen(9)
    x, w = rnd(g, 4, 256).cuda(), torch.ones(256, device='cuda')
    x[1, 3], x[2, 5] = float('nan'), float('inf')
    y, _ = F.add_rms_norm(x, torch.zeros_like(x), w)
    assert y[1].isnan().all() and y[2, 5].isnan() and not y[2, :5].any() and torch.isfinite(y[[0, 3]]).all()
    q, scale, _ = F.add_rms_norm_q8(x, torch.zeros_like(x), w)
    assert q[1].float().isnan().all() and scale[1].isnan() and torch.isfinite(q[[0, 3]].float()).all()


# ------------------------------------------------------------------------------------------------ together, and elsewhere
def test_on_another_stream(F):
    c = ScanCase(64, 16, 1, torch.float32, rows=(2, 40), seed=11)
    want, wstate = c.call(F, c.gpu)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        v = {k: t * 1.0 for k, t in c.gpu.items()}
        out, state = c.call(F, v)
        y, total = F.add_rms_norm(out, out, torch.ones(64, device='cuda'))
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(out, want) and torch.equal(state, wstate)
    assert torch.equal(total, want + want)


def _block(F, v, c, w):
    x = F.short_conv(c.lead(v['u']), w['conv'], None, silu=True, offsets=c.offsets)
    out = F.selective_scan(x, c.lead(v['delta']), v['A'], c.lead(v['B']), c.lead(v['C']), D=v['D'], z=c.lead(v['z']),
                           delta_bias=v['bias'], delta_softplus=True, offsets=c.offsets)
    return F.add_rms_norm(out, x, w['norm'])


@pytest.mark.parametrize('lengths', [None, [7, 0, 900, 4]])
def test_captured_and_replayed_beside_a_second_graph(F, lengths):
    """forward and backward of the three operators in a row, captured twice on different data and replayed in turn, with
    eager work between: every replay equals the eager result, bit for bit"""
    from hipvae import graph
    cases = [ScanCase(48, 16, 1, torch.float32, rows=None if lengths else (2, 300), lengths=lengths, seed=s, state=False)
             for s in (21, 22)]
    w = {'conv': torch.randn(48, 4, device='cuda'), 'norm': torch.rand(48, device='cuda') + 0.5}

    def step(c):
        leaf = {k: t.detach().requires_grad_() for k, t in c.gpu.items() if t is not None}
        leaf['state'] = None
        ww = {k: t.detach().requires_grad_() for k, t in w.items()}
        y, s = _block(F, leaf, c, ww)
        ins = [t for t in (*leaf.values(), *ww.values()) if t is not None]
        return [y.detach(), s.detach(), *torch.autograd.grad((y, s), ins, (torch.ones_like(y), torch.ones_like(s)))]

    want = [[t.clone() for t in step(c)] for c in cases]
    graphs, outs = [], []
    side = graph.capture_stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for c in cases:
            step(c)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with graph.quiet_collector(), torch.cuda.graph(g, stream=side):
            outs.append(step(c))
        graphs.append(g)
        graph._keep(g)
    for _ in range(3):
        for g, o, e, c in zip(graphs, outs, want, cases):
            for t in o:
                t.fill_(-3.0)
            g.replay()
            step(cases[0])
            torch.cuda.synchronize()
            for i, (a, b) in enumerate(zip(o, e)):
                assert torch.equal(a, b), i
    del graphs


def test_tensors_of_more_than_2_to_the_31_elements(F):
    """the last tokens of a packed batch whose tensors pass 2^31 elements: as those tokens alone"""
    D, T, n = 32768, 66000, 40                                                        # 2.16e9 elements, 4.3 GB each
    off = torch.tensor([0, 7, T - n, T], dtype=torch.int32, device='cuda')
    x = torch.zeros(T, D, dtype=torch.bfloat16, device='cuda')
    x[T - n:] = torch.randn(n, D, device='cuda').bfloat16()
    tail = x[T - n:]
    w, b = torch.randn(D, 4, device='cuda'), torch.randn(D, device='cuda')
    out, st = F.short_conv(x, w, b, silu=True, offsets=off, return_state=True)
    alone, st1 = F.short_conv(tail[None], w, b, silu=True, return_state=True)
    assert torch.equal(out[T - n:], alone[0]) and torch.equal(st[2], st1[0])
    del out
    y, s = F.add_rms_norm(x, x, b)
    y1, s1 = F.add_rms_norm(tail, tail, b)
    assert torch.equal(y[T - n:], y1) and torch.equal(s[T - n:], s1)
    del y, s
    A = -torch.rand(D, 4, device='cuda') - 0.5
    B = torch.randn(T, 4, device='cuda').bfloat16()
    leaf = x.requires_grad_()
    out, st = F.selective_scan(leaf, leaf, A, B, B, delta_softplus=True, offsets=off, return_state=True)
    t1 = tail.detach()[None].requires_grad_()
    alone, st1 = F.selective_scan(t1, t1, A, B[None, T - n:], B[None, T - n:], delta_softplus=True, return_state=True)
    bound = 2 * HALF[torch.bfloat16]                                                  # two roundings, and fp32's below
    assert ((out[T - n:] - alone[0]).abs() <= bound * alone[0].abs() + 1e-4).all()
    assert ((st[2] - st1[0]).abs() <= 1e-4).all()
    d = torch.zeros_like(out)
    d[T - n:] = 1
    (g,) = torch.autograd.grad(out, (leaf,), d)
    (g1,) = torch.autograd.grad(alone, (t1,), torch.ones_like(alone))
    # u and delta are one tensor: its gradient is the sum of two rounded ones
    assert ((g[T - n:] - g1[0]).abs() <= 3 * bound * (g1[0].abs() + g1[0].abs().max() * 0.05) + 1e-3).all()
    assert not g[:T - n].any()


@pytest.mark.parametrize('how', ['offloaded', 'recomputed', 'turned'])
def test_backward_from_tensors_that_hooks_put_in_place_of_the_kept_ones(F, how):
    """saved-tensor hooks hand back other memory, or other strides, than the forward pass read: same gradients, also with
    what the forward pass read overwritten by then"""
    from torch.utils.checkpoint import checkpoint
    c = ScanCase(48, 16, 1, torch.float32, lengths=[70, 0, 230], tail=4, seed=41, state=False)
    w = {'conv': torch.randn(48, 4, device='cuda'), 'norm': torch.rand(48, device='cuda') + 0.5}

    def run(hooked):
        leaf = {k: t.clone().requires_grad_() for k, t in c.gpu.items() if t is not None}
        ww = {k: t.clone().requires_grad_() for k, t in w.items()}
        body = lambda: _block(F, {k: t * 1.0 for k, t in leaf.items()}, c, ww)           # noqa: E731

        def turned(t):                                                                  # the same values, column by column
            return t.t().contiguous().t() if t.dim() == 2 else t.clone()

        if not hooked:
            y, s = body()
        elif how == 'offloaded':
            with torch.autograd.graph.save_on_cpu():
                y, s = body()
        elif how == 'turned':
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t, turned):
                y, s = body()
        else:
            y, s = checkpoint(body, use_reentrant=False)
        junk = [torch.full((c.gpu['u'].numel(),), float('nan'), device='cuda') for _ in range(64)]   # (in what is free by now)
        ins = [*leaf.values(), *ww.values()]
        got = torch.autograd.grad((y, s), ins, (torch.ones_like(y), torch.ones_like(s)))
        del junk
        return got

    for a, b in zip(run(False), run(True)):
        assert torch.equal(a, b)


def test_a_state_that_a_step_has_changed_is_refused_by_the_backward_pass(F):
    c = ScanCase(16, 4, 1, torch.float32, rows=(2, 6), seed=43)
    v = dict(c.gpu, u=c.gpu['u'].clone().requires_grad_())
    x, w = v['u'], torch.randn(16, 4, device='cuda')
    state, last = v['state'].clone(), torch.randn(2, 3, 16, device='cuda')
    out = c.call(F, dict(v, state=state), False)
    conv = F.short_conv(c.lead(x), w, state=last)
    with torch.no_grad():
        F.selective_scan_step(state, x[:2], v['delta'][:2], v['A'], v['B'][:2], v['C'][:2])
        F.short_conv_step(last, x[:2], w)
    for y in (out, conv):
        with pytest.raises(RuntimeError, match='modified by an inplace operation'):
            torch.autograd.grad(y, (x,), torch.ones_like(y))
    with torch.inference_mode():
        i = state.clone()
        F.selective_scan_step(i, x[:2], v['delta'][:2], v['A'], v['B'][:2], v['C'][:2])


def test_scan_of_more_sequences_than_a_grid_has_rows(F):
    """70000 sequences of two chunks each, the ones at the ends and on both sides of 65536 against the reference"""
    n, L, D, N = 70000, 256, 8, 2
    v = dict(u=torch.randn(n, L, D, device='cuda'), delta=torch.randn(n, L, D, device='cuda') - 1,
             B=torch.randn(n, L, 1, N, device='cuda'), C=torch.randn(n, L, 1, N, device='cuda'))
    v = {k: t.requires_grad_() for k, t in v.items()}
    A = -torch.rand(D, N, device='cuda') - 0.1
    out, state = F.selective_scan(v['u'], v['delta'], A, v['B'], v['C'], delta_softplus=True, return_state=True)
    got = dict(zip(v, torch.autograd.grad((out, state), list(v.values()), (torch.ones_like(out), torch.ones_like(state)))))
    for i in (0, 1, 65535, 65536, n - 1):
        one = np.ones
        r, m = (R.scan(f64(v['u'][i]), f64(v['delta'][i]), f64(A), f64(v['B'][i]), f64(v['C'][i]), [0, L], None, None, None,
                       True, None, one((L, D)), one((1, D, N)), size) for size in (False, True))
        count = 12 * L + L + D + 64
        close('out', out[i], r['out'], m['out'], count, U32)
        close('state', state[i:i + 1], r['state'], m['state'], count, U32)
        for k, t in got.items():
            close('d' + k, t[i], r[k], m[k], count, U32)


def test_scan_of_one_token_takes_any_token_stride(F):
    c = ScanCase(16, 4, 1, torch.float32, rows=(3, 1), seed=44)
    want = c.call(F, c.gpu)
    odd = lambda t: t.as_strided((3, 1, 16), (16, 1 << 27, 1))                            # noqa: E731
    v = c.gpu
    out, state = F.selective_scan(odd(v['u']), odd(v['delta']), v['A'], c.lead(v['B']), c.lead(v['C']), D=v['D'],
                                  z=odd(v['z']), delta_bias=v['bias'], delta_softplus=True, state=v['state'],
                                  return_state=True)
    assert torch.equal(out, want[0]) and torch.equal(state, want[1])


@pytest.mark.parametrize('S', [63, 64, 65, 200, 4096, 4097, 9000])
def test_many_packed_sequences(F, S):
    """searches over one, two and three rounds of 64 ends, with empty sequences between"""
    lens = torch.randint(0, 4, (S,), generator=gen(S)).tolist()
    c = ScanCase(5, 3, 1, torch.float32, lengths=lens, tail=3, seed=S)
    c.check(F, grads=False)
    x, w, st = rnd(gen(S + 1), c.T, 5), rnd(gen(S + 2), 5, 3), rnd(gen(S + 3), S, 2, 5)
    out, last = F.short_conv(x.cuda(), w.cuda(), state=st.cuda(), offsets=c.offsets, return_state=True)
    want, ends, off = torch.zeros(c.T, 5, dtype=torch.float64), st.double(), c.off
    for s in range(S):
        h = torch.cat([st[s], x[off[s]:off[s + 1]]]).double()
        ends[s] = h[len(h) - 2:]
        for t in range(off[s], off[s + 1]):
            want[t] = (h[t - off[s]:t - off[s] + 3] * w.t().double()).sum(0)
    assert torch.equal(last.cpu().double(), ends)
    assert ((out.cpu().double() - want).abs() <= 8 * U32 * 3 * x.abs().max() * w.abs().max()).all()


def test_results_repeat_bit_for_bit(F):
    c = ScanCase(200, 16, 2, torch.bfloat16, rows=(3, 150), seed=31, state=False)
    runs = []
    for _ in range(2):
        v = {k: None if t is None else t.clone().requires_grad_() for k, t in c.gpu.items()}
        out = c.call(F, v, False)
        runs.append([out] + list(torch.autograd.grad(out, [t for t in v.values() if t is not None], torch.ones_like(out))))
    assert all(torch.equal(a, b) for a, b in zip(*runs))


# ------------------------------------------------------------------------------------------------ refusals
def test_refusals(F):
    c = ScanCase(16, 4, 2, torch.float32, rows=(2, 6))
    v = c.gpu
    bad = [dict(u=v['u'].half()), dict(delta=v['delta'].bfloat16()), dict(delta=v['delta'][:, :8]),
           dict(A=v['A'][:8]), dict(A=v['A'].double()), dict(B=v['B'][:, :1]), dict(C=v['C'][..., :3]),
           dict(D=v['D'][:3]), dict(state=v['state'][:1]), dict(state=v['state'].bfloat16()), dict(u=v['u'].cpu()),
           dict(A=torch.zeros(16, 17, device='cuda'), B=torch.zeros(12, 2, 17, device='cuda'),
                C=torch.zeros(12, 2, 17, device='cuda'), state=torch.zeros(2, 16, 17, device='cuda')),
           dict(B=torch.zeros(12, 3, 4, device='cuda'), C=torch.zeros(12, 3, 4, device='cuda'))]
    for change in bad:
        with pytest.raises(RuntimeError):
            c.call(F, dict(v, **change))
    with pytest.raises(RuntimeError):
        F.selective_scan(v['u'], v['delta'], v['A'], v['B'], v['C'])                   # [tokens, channels], no offsets
    for off in (torch.tensor([0, 12], device='cuda'), torch.tensor([0], dtype=torch.int32, device='cuda'),
                torch.tensor([0, 12], dtype=torch.int32)):
        with pytest.raises(RuntimeError):
            F.selective_scan(v['u'], v['delta'], v['A'], v['B'], v['C'], offsets=off)
    st = v['state'].clone()
    step = lambda s, **k: F.selective_scan_step(s, v['u'][:2], v['delta'][:2], v['A'], v['B'][:2], v['C'][:2], **k)  # noqa: E731
    for s in (st[:1], st.transpose(1, 2).contiguous().transpose(1, 2), st.double()):
        with pytest.raises(RuntimeError):
            step(s)
    with pytest.raises(RuntimeError):
        step(st.requires_grad_())                                                      # no gradients through a step
    x, w = torch.randn(2, 5, 8, device='cuda'), torch.randn(8, 4, device='cuda')
    for args in ((x, w[:, :1]), (x, torch.randn(8, 5, device='cuda')), (x, w[:4]), (x[0], w), (x.half(), w),
                 (x, w.double()), (x.cpu(), w)):
        with pytest.raises(RuntimeError):
            F.short_conv(*args)
    with pytest.raises(RuntimeError):
        F.short_conv(x, w, state=torch.zeros(2, 4, 8, device='cuda'))
    with pytest.raises(RuntimeError):
        F.short_conv_step(torch.zeros(2, 3, 8, device='cuda', dtype=torch.bfloat16), x[:, 0], w)
    n = torch.ones(8, device='cuda')
    for args in ((x, x[:1], n), (x, x.bfloat16(), n), (x, x, n[:4]), (x, x, n.bfloat16()), (x.half(), x.half(), n)):
        with pytest.raises(RuntimeError):
            F.add_rms_norm(*args)
        with pytest.raises(RuntimeError):
            F.add_rms_norm_q8(*args)
