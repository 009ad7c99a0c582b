"""What of the sequence operators can be checked without a GPU: the references' gradients against differences, and that
the library refuses what its kernels do not take before it launches anything."""
import numpy as np
import pytest
import torch

import seq_reference as R


def _differences(f, v, key, eps=1e-6):
    x = v[key]
    g = np.zeros_like(x)
    for i in np.ndindex(x.shape):
        keep = x[i]
        x[i] = keep + eps
        hi = f(v)
        x[i] = keep - eps
        lo = f(v)
        x[i] = keep
        g[i] = (hi - lo) / (2 * eps)
    return g


@pytest.mark.parametrize('plus', [True, False])
def test_scan_formulas_against_differences(plus):
    r = np.random.RandomState(0)
    off, D, N, G = [0, 3, 3, 4], 4, 3, 2
    T = 5
    v = dict(u=r.randn(T, D), delta=np.abs(r.randn(T, D)), A=-np.exp(r.randn(D, N)), B=r.randn(T, G, N), C=r.randn(T, G, N),
             D=r.randn(D), z=r.randn(T, D), bias=r.rand(D), state=r.randn(3, D, N))
    dout, dst = r.randn(T, D), r.randn(3, D, N)
    dout_live = dout.copy()
    dout_live[4:] = 0                                                                 # the last token is in no sequence

    def f(v):
        o = R.scan(offsets=off, plus=plus, **v)
        return (o['out'] * dout_live).sum() + (o['state'] * dst).sum()

    got = R.scan(offsets=off, plus=plus, dout=dout, dstate=dst, **v)
    for k in v:
        want = _differences(f, v, k)
        np.testing.assert_allclose(got['state_in' if k == 'state' else k], want, rtol=1e-6, atol=1e-7, err_msg=k)


@pytest.mark.parametrize('W', [2, 3, 4])
@pytest.mark.parametrize('act', [True, False])
def test_conv_formulas_against_differences(W, act):
    r = np.random.RandomState(1)
    off, D, T = [0, 4, 4, 5, 7], 3, 8
    v = dict(x=r.randn(T, D), w=r.randn(D, W), bias=r.randn(D), state=r.randn(4, W - 1, D))
    dout, dst = r.randn(T, D), r.randn(4, W - 1, D)

    def f(v):
        o = R.conv(offsets=off, act=act, **v)
        return (o['out'][:7] * dout[:7]).sum() + (o['state'] * dst).sum()

    got = R.conv(offsets=off, act=act, dout=dout, dstate=dst, **v)
    for k, name in (('x', 'x'), ('w', 'weight'), ('bias', 'bias'), ('state', 'state_in')):
        np.testing.assert_allclose(got[name], _differences(f, v, k), rtol=1e-6, atol=1e-7, err_msg=k)


def test_norm_formulas_against_differences():
    r = np.random.RandomState(2)
    v = dict(v=r.randn(3, 6), w=r.randn(6))
    dy, ds = r.randn(3, 6), r.randn(3, 6)
    got = R.norm(eps=1e-3, dy=dy, dsum=ds, **v)
    f = lambda v: (R.norm(eps=1e-3, **v)['y'] * dy).sum() + (v['v'] * ds).sum()        # noqa: E731
    np.testing.assert_allclose(got['x'], _differences(f, v, 'v'), rtol=1e-6, atol=1e-7)
    np.testing.assert_allclose(got['weight'], _differences(f, v, 'w'), rtol=1e-6, atol=1e-7)


def _lib():
    from hipvae import _lib
    return _lib.lib


def _scan_fwd(rows=2, L=8, D=16, G=1, N=16, S=2, dtype=0, offsets=None):
    lib = _lib()
    n = None
    return lib.dvae_selective_scan_fwd(n, 0, 0, n, 0, 0, n, n, 0, 0, 0, n, 0, 0, 0, n, n, 0, 0, n, 1, n, n, offsets, n, n,
                                       rows, L, D, G, N, S, dtype, n, n)


@pytest.mark.parametrize('bad,text', [
    (dict(N=17), b'1 to 16 states'), (dict(N=0), b'states'), (dict(G=3), b'multiple of G'), (dict(dtype=2), b'dtype'),
    (dict(rows=1 << 20, L=1 << 12), b'too large'), (dict(offsets=64, rows=2), b'one row'),
])
def test_scan_refuses_before_any_launch(bad, text):
    assert _scan_fwd(**bad) != 0
    assert text in _lib().dvae_last_error()


@pytest.mark.parametrize('rows,L,D,text', [
    (1, (1 << 31) - (1 << 16), 1, b'too large'), (1 << 30, 2, 1, b'too large'),            # positions are 32 bits
    (1 << 24, 1, 64, b'one launch'), (1 << 23, 1, 300, b'one launch'),                     # 2^32 threads are too many
])
def test_scan_sizes_that_no_launch_takes(rows, L, D, text):
    assert _scan_fwd(rows=rows, L=L, D=D, S=rows) != 0
    assert text in _lib().dvae_last_error()


def test_conv_sizes_that_no_launch_takes():
    lib, n = _lib(), None
    for rows, L in ((1, (1 << 31) - (1 << 16)), (1 << 30, 2)):
        assert lib.dvae_short_conv_fwd(n, 0, 0, n, n, 0, n, n, n, n, rows, L, 16, 4, rows, 0, n) != 0
        assert b'too many tokens' in lib.dvae_last_error()
    assert lib.dvae_short_conv_step(n, n, 0, n, n, 0, n, 1 << 24, 256, 4, 0, n) != 0
    assert b'one launch' in lib.dvae_last_error()
    assert lib.dvae_selective_scan_step(n, n, 0, n, 0, n, n, 0, 0, n, 0, 0, n, n, 0, n, 1, n, 1 << 24, 256, 1, 16, 0, n) != 0
    assert b'one launch' in lib.dvae_last_error()


def test_calls_without_tokens_launch_nothing():
    assert _scan_fwd(rows=0) == 0 and _scan_fwd(L=0) == 0
    lib, n = _lib(), None
    assert lib.dvae_short_conv_fwd(n, 0, 0, n, n, 0, n, n, n, n, 0, 5, 16, 4, 0, 0, n) == 0
    assert lib.dvae_short_conv_step(n, n, 0, n, n, 0, n, 0, 16, 4, 0, n) == 0
    assert lib.dvae_selective_scan_step(n, n, 0, n, 0, n, n, 0, 0, n, 0, 0, n, n, 0, n, 1, n, 0, 16, 1, 16, 0, n) == 0
    assert lib.dvae_add_rms_norm_fwd(n, 0, n, 0, n, 1e-6, n, n, n, 0, 16, 0, 0, n) == 0


def test_conv_and_norm_refuse_before_any_launch():
    lib, n = _lib(), None
    for W, dtype, text in ((1, 0, b'taps'), (5, 0, b'taps'), (4, 2, b'dtype')):
        assert lib.dvae_short_conv_fwd(n, 0, 0, n, n, 0, n, n, n, n, 2, 5, 16, W, 2, dtype, n) != 0
        assert text in lib.dvae_last_error()
    assert lib.dvae_add_rms_norm_fwd(n, 0, n, 0, n, 1e-6, n, n, n, 4, 16, 0, 1, n) != 0
    assert b"residual's type" in lib.dvae_last_error()
    assert lib.dvae_add_rms_norm_bwd(n, 0, n, 0, n, 0, n, n, n, n, n, 0, 16, 0, 0, n, n) != 0
    assert b'no rows' in lib.dvae_last_error()


def test_cpu_tensors_are_refused():
    from hipvae import functional as F
    x, w = torch.zeros(2, 5, 8), torch.zeros(8, 4)
    for call in (lambda: F.short_conv(x, w), lambda: F.add_rms_norm(x, x, w[:, 0]),
                 lambda: F.add_rms_norm_q8(x, x, w[:, 0]), lambda: F.selective_scan(x, x, w, x, x),
                 lambda: F.short_conv_step(torch.zeros(2, 3, 8), x[:, 0], w),
                 lambda: F.selective_scan_step(torch.zeros(2, 8, 4), x[:, 0], x[:, 0], w, x[:, 0, :4], x[:, 0, :4])):
        with pytest.raises(RuntimeError, match='GPU'):
            call()
