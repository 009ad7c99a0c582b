"""Refusals of the sequence operators that come before a tensor's device is looked at."""
import pytest
import torch
import torch.autograd.forward_ad as fwd


def _calls(dual):
    """every entry point with one dual tensor among its arguments"""
    from hipvae import functional as F
    x, w, n = torch.randn(2, 5, 8), torch.randn(8, 4), torch.randn(8)
    bc = torch.randn(2, 5, 4)
    return {
        'selective_scan': [lambda: F.selective_scan(dual(x), x, w, bc, bc), lambda: F.selective_scan(x, x, w, bc, bc, D=dual(n)),
                           lambda: F.selective_scan(x, x, w, bc, bc, state=dual(torch.randn(2, 8, 4)))],
        'selective_scan_step': [lambda: F.selective_scan_step(torch.zeros(2, 8, 4), x[:, 0], dual(x[:, 0]), w, bc[:, 0],
                                                              bc[:, 0])],
        'short_conv': [lambda: F.short_conv(x, dual(w))],
        'short_conv_step': [lambda: F.short_conv_step(dual(torch.zeros(2, 3, 8)), x[:, 0], w)],
        'add_rms_norm': [lambda: F.add_rms_norm(dual(x), x, n), lambda: F.add_rms_norm(x, None, dual(n))],
        'add_rms_norm_q8': [lambda: F.add_rms_norm_q8(x, dual(x), n)],
    }


@pytest.mark.parametrize('grad', [True, False])
def test_forward_mode_is_refused(grad):
    """a dual tensor does not require gradients: the operators must not return outputs without its tangent"""
    with fwd.dual_level(), torch.set_grad_enabled(grad):
        for what, calls in _calls(lambda t: fwd.make_dual(t, torch.ones_like(t))).items():
            for call in calls:
                with pytest.raises(RuntimeError, match=f'{what}: forward-mode'):
                    call()
        for calls in _calls(lambda t: t).values():                  # a dual level alone changes nothing
            for call in calls:
                with pytest.raises(RuntimeError, match='GPU'):
                    call()


def test_forward_mode_transforms_are_refused():
    from hipvae import functional as F
    x, n = torch.randn(2, 5, 8), torch.randn(8)
    for f in (torch.func.jvp, lambda f, a, b: torch.func.jacfwd(f)(*a)):
        with pytest.raises(RuntimeError, match='forward-mode'):
            f(lambda t: F.add_rms_norm(t, None, n)[0], (x,), (x,))


@pytest.mark.parametrize('rows,L,D,G,N,split', [
    (1, 4096, 2048, 1, 16, True), (8, 2048, 2048, 1, 16, True), (16, 1024, 2048, 1, 16, True), (1, 31, 64, 1, 16, False),
    (1, 1, 64, 1, 16, False), (28, 2048, 2048, 1, 8, True), (32, 512, 2048, 1, 5, True), (1, 8192, 49152, 1, 16, True),
    # a wave for most SIMDs, and many for each: the passes that chunks need cost more than they gain
    (24, 512, 2048, 1, 16, False), (32, 1024, 2048, 1, 16, False), (96, 512, 2048, 1, 16, False),
    (256, 512, 2048, 1, 16, False), (4096, 4096, 64, 1, 16, False), (512, 512, 256, 4, 16, False),
    (64, 512, 2048, 1, 8, False), (64, 4096, 2048, 1, 5, False), (1, 1024, 131072, 1, 16, False),
])
def test_the_scan_splits_the_time_axis_where_there_are_few_rows(rows, L, D, G, N, split):
    """scratch is what tells from outside: without chunks the forward pass needs none"""
    from hipvae._lib import lib
    for keep in (0, 1):
        assert (lib.dvae_selective_scan_fwd_ws_floats(rows, L, D, G, N, keep) > 0) == split
