"""models.SSMEncoder: the sequence operators together, in their sequence form, packed form and step form, against a plain
torch restatement in fp64 on the CPU (values and gradients).

fp32 products and sums of at most a few hundred terms: the bar of 2e-5 (relative L2) that the GEMM-shaped kernels are held
to, twice per layer and once at each end, and 1e-4 for gradients, as for the models."""
import pytest
import torch

pytestmark = pytest.mark.gpu
CFG = dict(input_dim=24, hidden_dim=32, num_layers=2, state_dim=8, conv_width=4)


def norm(x, w, eps=1e-6):
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w


def plain(p, x, states, cfg, groups=1):
    """one sequence [T, input] token by token -> [T, hidden], states"""
    N, W = cfg['state_dim'], cfg['conv_width']
    outs = []
    for t in range(x.shape[0]):
        h, r = x[t] @ p['proj.weight'].t() + p['proj.bias'], None
        new = []
        for i in range(cfg['num_layers']):
            q = lambda k: p[f'layers.{i}.{k}']                                        # noqa: E731
            conv, scan = states[i]
            r = h if r is None else h + r
            u, z = (norm(r, q('norm')) @ q('in_proj.weight').t()).chunk(2)
            win = torch.cat([conv, u[None]])
            u = torch.nn.functional.silu((win.t() * q('conv_weight')).sum(1) + q('conv_bias'))
            pr = u @ q('x_proj.weight').t()
            R = pr.numel() - 2 * groups * N
            per = u.numel() // groups
            B, C = (pr[R + k * groups * N:R + (k + 1) * groups * N].view(groups, N).repeat_interleave(per, 0) for k in (0, 1))
            dt = torch.nn.functional.softplus(pr[:R] @ q('dt_proj.weight').t() + q('dt_bias'))
            scan = torch.exp(dt[:, None] * -torch.exp(q('A_log'))) * scan + (dt * u)[:, None] * B
            y = ((scan * C).sum(1) + q('D') * u) * torch.nn.functional.silu(z)
            h = y @ q('out_proj.weight').t()
            new.append((win[1:], scan))
        states = new
        outs.append(norm(h + r, p['norm']))
    return torch.stack(outs) if outs else x.new_zeros(0, cfg['hidden_dim']), states


def rel(a, b):
    return float((a.detach().double().cpu() - b.detach()).norm() / b.detach().norm().clamp_min(1e-30))


def make(seed=0, **more):
    import models
    torch.manual_seed(seed)
    m = models.SSMEncoder(**{**CFG, **more})
    p64 = {k: v.detach().double().requires_grad_() for k, v in m.state_dict().items()}
    return m.cuda(), p64


def zeros64(m, n):
    return [[(a[k].double().cpu(), b[k].double().cpu()) for a, b in m.init_states(n)] for k in range(n)]


@pytest.mark.parametrize('groups', [1, 2])
def test_sequences_and_gradients(groups):
    m, p = make(groups=groups)
    cfg = CFG
    B, T = 3, 13
    x = torch.randn(B, T, cfg['input_dim'])
    x64 = x.double().requires_grad_()
    ref = [plain(p, x64[b], s, cfg, groups) for b, s in enumerate(zeros64(m, B))]
    seq = torch.stack([r[0] for r in ref])
    xg = x.cuda().requires_grad_()
    y, states = m(xg, return_sequence=True)
    assert rel(y, seq) < 1e-4
    for i in range(cfg['num_layers']):
        for k in (0, 1):
            assert rel(states[i][k], torch.stack([r[1][i][k] for r in ref])) < 1e-4
    w = torch.randn(B, T, cfg['hidden_dim'])
    names = list(p)
    want = torch.autograd.grad((seq * w.double()).sum(), [x64] + [p[k] for k in names], retain_graph=True)
    named = dict(m.named_parameters())
    got = torch.autograd.grad((y * w.cuda()).sum(), [xg] + [named[k] for k in names])
    for k, a, b in zip(['x'] + names, got, want):
        assert rel(a, b) < 1e-4, (k, rel(a, b))
    last, _ = m(xg)
    assert torch.equal(last, y[:, -1])


def test_packed_sequences_are_the_sequences():
    m, p = make(1)
    lengths = [5, 0, 17, 1]
    off = torch.tensor([0, 5, 5, 22, 23], dtype=torch.int32, device='cuda')
    x = torch.randn(23, CFG['input_dim'], device='cuda')
    seq, states = m(x, return_sequence=True, offsets=off)
    last, _ = m(x, offsets=off)
    for s, n in enumerate(lengths):
        b = int(off[s])
        if n == 0:
            assert not last[s].any()
            assert all(not states[i][k][s].any() for i in range(2) for k in (0, 1))
            continue
        alone, st = m(x[None, b:b + n], return_sequence=True)
        # rows of a matrix product may be computed in other tiles: equal up to its rounding
        torch.testing.assert_close(seq[b:b + n], alone[0], rtol=1e-4, atol=1e-5)
        torch.testing.assert_close(last[s], seq[b + n - 1], rtol=0, atol=0)
        for i in range(2):
            for k in (0, 1):
                torch.testing.assert_close(states[i][k][s], st[i][k][0], rtol=1e-4, atol=1e-5)


def test_steps_go_on_where_a_prompt_ended():
    m, p = make(2)
    B, T, more = 4, 9, 6
    x = torch.randn(B, T + more, CFG['input_dim'], device='cuda')
    with torch.no_grad():
        whole, _ = m(x, return_sequence=True)
        head, states = m(x[:, :T], return_sequence=True)
        outs = [m.step(x[:, t], states) for t in range(T, T + more)]
        tail, _ = m(x[:, T:], return_sequence=True, states=m(x[:, :T])[1])
    torch.testing.assert_close(head, whole[:, :T], rtol=1e-4, atol=1e-5)
    torch.testing.assert_close(torch.stack(outs, 1), whole[:, T:], rtol=1e-4, atol=1e-5)
    torch.testing.assert_close(tail, whole[:, T:], rtol=1e-4, atol=1e-5)


def test_captured_step():
    """frame-by-frame serving from one captured graph: the states move on with every replay"""
    from hipvae import graph
    m, _ = make(3)
    B, T = 2, 6
    x = torch.randn(B, T, CFG['input_dim'], device='cuda')
    with torch.no_grad():
        states = m.init_states(B)
        want = [m.step(x[:, t], states).clone() for t in range(T)]
        live = m.init_states(B)
        frame = x[:, 0].clone()
        side = graph.capture_stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            m.step(frame, m.init_states(B))
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with graph.quiet_collector(), torch.cuda.graph(g, stream=side):
            out = m.step(frame, live)
        graph._keep(g)
        for a, b in live:
            a.zero_()
            b.zero_()
        for t in range(T):
            frame.copy_(x[:, t])
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want[t]), t
