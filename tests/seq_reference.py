"""The sequence operators in 64 bits, token by token, with their gradients by formula (numpy, on the CPU).

With `size=True` every factor enters by its absolute value (decays and gates excepted, which are factors between terms):
what comes out is the sum of the sizes of the terms, the quantity that rounding errors are proportional to."""
import numpy as np


def softplus(x):
    return np.maximum(x, 0) + np.log1p(np.exp(-np.abs(x)))


def sigmoid(x):
    return 1 / (1 + np.exp(-x))


def silu(x):
    return x * sigmoid(x)


def silu_grad(x):
    s = sigmoid(x)
    return s * (1 + x * (1 - s))


def scan(u, delta, A, B, C, offsets, D=None, z=None, bias=None, plus=True, state=None, dout=None, dstate=None, size=False):
    """u, delta, z [T, D]; A [D, N]; B, C [T, G, N]; offsets: list.  -> dict of outputs and, with dout, gradients"""
    f = np.abs if size else (lambda v: v)
    T, ch = u.shape
    N, G, S = A.shape[1], B.shape[1], len(offsets) - 1
    group = np.arange(ch) // (ch // G)
    pre = delta + (0 if bias is None else bias)
    dt = softplus(pre) if plus else pre
    gate = np.ones_like(u) if z is None else silu(z)
    y, hs = np.zeros((T, ch)), np.zeros((T, ch, N))
    final = np.zeros((S, ch, N)) if state is None else f(state).copy()
    before = np.zeros((T, ch, N))
    for s in range(S):
        h = final[s].copy()
        for t in range(offsets[s], offsets[s + 1]):
            before[t] = h
            h = np.exp(dt[t][:, None] * A) * h + f(dt[t] * u[t])[:, None] * f(B[t][group])
            hs[t] = h
            y[t] = (f(C[t][group]) * h).sum(1) + (0 if D is None else f(D * u[t]))
        final[s] = h
    r = {'out': y * f(gate), 'state': final}
    if dout is None:
        return r
    live = np.zeros(T, bool)
    live[offsets[0]:offsets[-1]] = True
    g = f(dout) * f(gate) * live[:, None]
    r.update(u=np.zeros_like(u), delta=np.zeros_like(u), A=np.zeros_like(A), B=np.zeros_like(B), C=np.zeros_like(C),
             D=(g * f(u)).sum(0), state_in=np.zeros((S, ch, N)))
    if z is not None:
        # silu'(z) = s (1 + z (1 - s)) is a sum of two terms that cancel near z = -1.28: rounding the product z (1 - s)
        # (to half a step of |z| (1 - s), near 1 there) leaves an error of that size however small the sum is, so its
        # size, like every other sum's, is that of its terms
        slope = sigmoid(z) * (1 + np.abs(z) * sigmoid(-z)) if size else silu_grad(z)
        r['z'] = f(dout) * y * slope * live[:, None]
    for s in range(S):
        carry = np.zeros((ch, N)) if dstate is None else f(dstate[s]).copy()
        for t in range(offsets[s + 1] - 1, offsets[s] - 1, -1):
            Bt, Ct = f(B[t][group]), f(C[t][group])
            d = carry + Ct * g[t][:, None]
            carry = d * np.exp(dt[t][:, None] * A)
            k = carry * before[t]
            r['A'] += k * f(dt[t])[:, None]
            through = (d * Bt).sum(1)
            r['u'][t] = through * f(dt[t]) + (0 if D is None else f(D) * g[t])
            dd = (k * f(A)).sum(1) + through * f(u[t])
            r['delta'][t] = dd * sigmoid(pre[t]) if plus else dd
            for q in range(G):
                m = group == q
                r['B'][t, q] = (d[m] * f(dt[t] * u[t])[m, None]).sum(0)
                r['C'][t, q] = (hs[t][m] * g[t][m, None]).sum(0)
        r['state_in'][s] = carry
    r['bias'] = r['delta'].sum(0)
    return r


def conv(x, w, offsets, bias=None, act=True, state=None, dout=None, dstate=None, size=False):
    """x [T, D], w [D, W]"""
    f = np.abs if size else (lambda v: v)
    T, ch = x.shape
    W, S = w.shape[1], len(offsets) - 1
    out, dx = np.zeros((T, ch)), np.zeros((T, ch))
    final, dst = np.zeros((S, W - 1, ch)), np.zeros((S, W - 1, ch))
    dw, db = np.zeros_like(w), np.zeros(ch)
    for s in range(S):
        lo, hi = offsets[s], offsets[s + 1]
        line = np.concatenate([np.zeros((W - 1, ch)) if state is None else state[s], x[lo:hi]])
        n = hi - lo
        pre = np.stack([line[t:t + W].T for t in range(n)]) if n else np.zeros((0, ch, W))      # [n, ch, W]
        true = (pre * w).sum(2) + (0 if bias is None else bias)
        big = (f(pre) * f(w)).sum(2) + (0 if bias is None else f(bias))
        # silu is at most 1.1-Lipschitz and |silu(x)| <= |x|: the terms' sizes carry over
        out[lo:hi] = (1.1 * big if size else silu(true)) if act else big
        final[s] = line[n:]
        if dout is None:
            continue
        d = f(dout[lo:hi])
        if act:
            d = d * (1.1 + 0.5 * big if size else silu_grad(true))      # |silu'| <= 1.1, and it is 0.5-Lipschitz
        dline = np.zeros_like(line)
        for k in range(W):
            dline[k:k + n] += d * f(w[:, k])
            dw[:, k] += (d * f(line[k:k + n])).sum(0)
        if dstate is not None:
            dline[n:] += f(dstate[s])
        db += d.sum(0)
        dx[lo:hi], dst[s] = dline[W - 1:], dline[:W - 1]
    return {'out': out, 'state': final, 'x': dx, 'weight': dw, 'bias': db, 'state_in': dst}


def norm(v, w, eps, dy=None, dsum=None, size=False):
    """v [R, D]: the stored sum"""
    f = np.abs if size else (lambda a: a)
    r = 1 / np.sqrt((v * v).mean(1, keepdims=True) + eps)
    hat = v * r
    out = {'y': f(hat * w)}
    if dy is not None:
        gw = f(dy * w)
        m = (gw * f(hat)).mean(1, keepdims=True)
        out['x'] = r * (gw + f(hat) * m if size else gw - hat * m) + (0 if dsum is None else f(dsum))
        out['weight'] = (f(dy) * f(hat)).sum(0)
    return out
