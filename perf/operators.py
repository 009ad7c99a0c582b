"""The sequence operators of hipvae.functional, as cases that can be measured.

Three operators that work together in a selective state-space block, the time-mixing layer that stands beside the LSTM
recurrences: the short causal convolution over time (`short_conv`), the selective scan (`selective_scan`) and the
root-mean-square norm with the residual's addition (`add_rms_norm`).  Each is measured as a prompt or an evaluation
runs it ("forward"), as training runs it ("train": forward and backward) and, where it has such forms, as
frame-by-frame serving runs it ("step": one token per sequence, the state updated in place) and with an 8-bit output
("q8").

Tensors are channels-last: [tokens, channels] with the tokens of all sequences one after the other.  A batch of equal
clips reaches the operators as [batch, length, channels]; sequences of different lengths are packed and come with
`offsets`.  The plain forms work on tokens and their sequences' borders and are the same for both.
"""
import math
import os
import sys

import torch

own = False

#: what `own` runs: hipvae.functional, looked up on the first call that needs it
_functional = None

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
EPS = 1e-6


def _case(name, op, mode, dtype, rows, length, channels, states=0, groups=1, width=0, sequences=0):
    """`sequences` > 0: rows * length tokens are shared out over that many packed sequences of different lengths."""
    return dict(name=name, op=op, mode=mode, dtype=dtype, rows=rows, length=length, channels=channels, states=states,
                groups=groups, width=width, sequences=sequences)


def listed():
    return [
        # one clip's next frame through a layer with the width of the configurations' frame features: latency
        _case("scan step 1 x 512", "scan", "step", "fp32", 1, 1, 512, states=16),
        # the next frame of a full evaluation batch
        _case("scan step 256 x 2048", "scan", "step", "bf16", 256, 1, 2048, states=16),
        # one long sequence at once, its final state kept for the steps that follow: few rows, a long time axis
        _case("scan prompt 1 x 4096", "scan", "forward", "bf16", 1, 4096, 2048, states=16),
        # a training batch of 20-frame clips, inner width twice the 512 frame features
        _case("scan train 256 x 20", "scan", "train", "fp32", 256, 20, 1024, states=16),
        # a training batch of long sequences
        _case("scan train 8 x 2048", "scan", "train", "bf16", 8, 2048, 2048, states=16),
        # sequences of different lengths in one packed batch, an odd number of channels per group
        _case("scan packed 37", "scan", "train", "bf16", 1, 5003, 1002, states=16, groups=2, sequences=37),
        # the convolution's next frame of an evaluation batch
        _case("conv step 32 x 1024", "conv", "step", "fp32", 32, 1, 1024, width=4),
        # the convolution of a training batch of long sequences
        _case("conv train 8 x 2048", "conv", "train", "bf16", 8, 2048, 2048, width=4),
        # packed sequences, three taps, rows that are not a multiple of 16 bytes
        _case("conv packed 37", "conv", "forward", "fp32", 1, 5003, 1001, width=3, sequences=37),
        # the norm before one frame's layer: latency
        _case("norm 1 x 512", "norm", "forward", "fp32", 1, 1, 512),
        # the norm of a training batch of long sequences
        _case("norm train 16384 x 2048", "norm", "train", "bf16", 8, 2048, 2048),
        # activations kept in 8 bits between layers, an odd number of rows
        _case("norm q8 4099 x 2560", "norm", "q8", "bf16", 1, 4099, 2560),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["scan", "scan", "conv", "norm"])
    mode = rng.choice({"scan": ["forward", "train", "step"], "conv": ["forward", "train", "step"],
                       "norm": ["forward", "train", "q8"]}[op])
    dtype = rng.choice(["fp32", "bf16"])
    groups = rng.choice([1, 1, 1, 2, 4]) if op == "scan" else 1
    # widths: multiples of 64, and any number
    per_group = _log_int(rng, 24, 2048 // groups)
    if rng.random() < 0.6:
        per_group = max(64, per_group // 64 * 64) if groups < 4 else max(16, per_group // 16 * 16)
    channels = per_group * groups
    states = rng.choice([5, 8, 16, 16, 16]) if op == "scan" else 0
    width = rng.choice([2, 3, 4, 4]) if op == "conv" else 0
    sequences = 0
    if mode == "step":
        rows, length = _log_int(rng, 1, 256), 1
    else:
        length = _log_int(rng, 1, 8192)
        rows = _log_int(rng, 1, max(1, min(256, 16384 // length)))
        if op != "norm" and rng.random() < 0.35:
            length, rows = rows * length, 1
            sequences = _log_int(rng, 1, min(64, length))
    return {k: v for k, v in _case("", op, mode, dtype, rows, length, channels, states, groups, width, sequences).items()
            if k != "name"}


# ------------------------------------------------------------------------------------------------ inputs
def _lengths(case):
    """the lengths of the case's sequences, the same for every seed: ragged, with an empty one where there are several"""
    total = case["rows"] * case["length"]
    n = case["sequences"]
    if not n:
        return [case["length"]] * case["rows"]
    g = torch.Generator().manual_seed(7 * total + n)
    share = torch.rand(n, generator=g).pow(2) + 0.02
    if n > 3:
        share[n // 2] = 0.0
    ends = (share.cumsum(0) / share.sum() * total).round().long().tolist()
    ends[-1] = total
    return [e - b for b, e in zip([0] + ends[:-1], ends)]


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    t = TYPES[case["dtype"]]
    T, D = case["rows"] * case["length"], case["channels"]

    def randn(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device=dev) * scale

    s = {"case": dict(case), "dtype": t}
    if case["op"] == "norm":
        s["x"], s["residual"] = randn(T, D).to(t), randn(T, D, scale=2.0).to(t)
        s["weight"] = 1 + 0.2 * randn(D)
        if case["mode"] == "train":
            s["dy"], s["dsum"] = randn(T, D).to(t), randn(T, D).to(t)
        return s
    lengths = _lengths(case)
    s["sequences"] = len(lengths)
    s["longest"] = max(lengths)
    s["offsets"] = torch.tensor([0] + lengths, device=dev).cumsum(0).to(torch.int32)
    # the layer's input projection writes both halves side by side: the operators read them as strided views
    both = randn(T, 2 * D).to(t)
    if case["op"] == "conv":
        W = case["width"]
        s["x"] = both[:, :D]
        s["weight"], s["bias"] = randn(D, W, scale=W ** -0.5), randn(D, scale=0.1)
        if case["mode"] != "train":                      # serving: the last inputs of each sequence are carried along
            s["state"] = randn(len(lengths), W - 1, D).to(t)
        else:
            s["dout"] = randn(T, D).to(t)
        return s
    N, G, R = case["states"], case["groups"], max(4, D // 16 // 4 * 4)
    s["z"] = both[:, D:]
    s["u"] = torch.nn.functional.silu(randn(T, D)).to(t)
    s["delta"] = randn(T, D, scale=0.7).to(t)
    proj = randn(T, R + 2 * G * N).to(t)
    s["B"] = proj[:, R:R + G * N].view(T, G, N)
    s["C"] = proj[:, R + G * N:].view(T, G, N)
    # decay rates 1 .. N per channel; step sizes from 1e-3 to 1e-1, spread over the channels
    s["A"] = -torch.arange(1, N + 1, device=dev, dtype=torch.float32).repeat(D, 1) * torch.exp(0.1 * randn(D, N))
    dt = torch.exp(torch.rand(D, generator=g, device=dev) * math.log(100.0) + math.log(1e-3))
    s["delta_bias"] = dt + torch.log(-torch.expm1(-dt))
    s["D"] = 1 + 0.1 * randn(D)
    if case["mode"] != "train":
        s["state"] = randn(len(lengths), D, N, scale=0.3)
    else:
        s["dout"] = randn(T, D).to(t)
    return s


# ------------------------------------------------------------------------------------------------ the framework's calls
def _calls():
    global _functional
    if _functional is None:
        pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "disentangled-vae_amd")
        if pkg not in sys.path:
            sys.path.insert(1, pkg)
        from hipvae import functional
        _functional = functional
    return _functional


def _batched(s, *tensors):
    """[tokens, ...] as [batch, length, ...], the form of a batch of equal clips; packed sequences stay as they are"""
    c = s["case"]
    if c["sequences"]:
        return tensors
    return tuple(t.unflatten(0, (c["rows"], c["length"])) for t in tensors)


def _run_own(s):
    F = _calls()
    c = s["case"]
    if c["op"] == "norm":
        if c["mode"] == "forward":
            y, total = F.add_rms_norm(s["x"], s["residual"], s["weight"], EPS)
            return {"y": y, "sum": total}
        if c["mode"] == "q8":
            q, scale, total = F.add_rms_norm_q8(s["x"], s["residual"], s["weight"], EPS)
            return {"q": q, "scale": scale, "sum": total}
        x, r, w = (s[k].detach().requires_grad_() for k in ("x", "residual", "weight"))
        y, total = F.add_rms_norm(x, r, w, EPS)
        dx, dr, dw = torch.autograd.grad((y, total), (x, r, w), (s["dy"], s["dsum"]))
        return {"y": y, "sum": total, "dx": dx, "dresidual": dr, "dweight": dw}
    offsets = s["offsets"] if c["sequences"] else None
    if c["op"] == "conv":
        if c["mode"] == "step":
            out = F.short_conv_step(s["state"], s["x"], s["weight"], s["bias"], silu=True)
            return {"out": out, "state": s["state"]}
        if c["mode"] == "forward":
            (x,) = _batched(s, s["x"])
            out, state = F.short_conv(x, s["weight"], s["bias"], silu=True, state=s["state"], offsets=offsets,
                                      return_state=True)
            return {"out": out.flatten(0, -2), "state": state}
        x, w, b = (s[k].detach().requires_grad_() for k in ("x", "weight", "bias"))
        xb, dout = _batched(s, x, s["dout"])
        out = F.short_conv(xb, w, b, silu=True, offsets=offsets)
        dx, dw, db = torch.autograd.grad(out, (x, w, b), dout)
        return {"out": out.flatten(0, -2), "dx": dx, "dweight": dw, "dbias": db}
    if c["mode"] == "step":
        out = F.selective_scan_step(s["state"], s["u"], s["delta"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"],
                                    delta_bias=s["delta_bias"], delta_softplus=True)
        return {"out": out, "state": s["state"]}
    if c["mode"] == "forward":
        u, delta, B, C, z = _batched(s, s["u"], s["delta"], s["B"], s["C"], s["z"])
        out, state = F.selective_scan(u, delta, s["A"], B, C, D=s["D"], z=z, delta_bias=s["delta_bias"],
                                      delta_softplus=True, state=s["state"], offsets=offsets, return_state=True)
        return {"out": out.flatten(0, -2), "state": state}
    names = ("u", "delta", "A", "B", "C", "D", "z", "delta_bias")
    v = {k: s[k].detach().requires_grad_() for k in names}
    u, delta, B, C, z, dout = _batched(s, v["u"], v["delta"], v["B"], v["C"], v["z"], s["dout"])
    out = F.selective_scan(u, delta, v["A"], B, C, D=v["D"], z=z, delta_bias=v["delta_bias"], delta_softplus=True,
                           offsets=offsets)
    grads = torch.autograd.grad(out, [v[k] for k in names], dout)
    return {"out": out.flatten(0, -2), **{"d" + k: g for k, g in zip(names, grads)}}


# ------------------------------------------------------------------------------------------------ the plain forms
def _norm_plain(s):
    c, t = s["case"], s["dtype"]
    total = (s["x"].float() + s["residual"].float()).to(t)
    v, w = total.float(), s["weight"]
    rstd = (v.square().mean(-1, keepdim=True) + EPS).rsqrt()
    y = v * rstd * w
    if c["mode"] == "forward":
        return {"y": y.to(t), "sum": total}
    if c["mode"] == "q8":
        most = y.abs().amax(-1, keepdim=True)
        scale = torch.where(most > 0, most / 448.0, torch.ones_like(most))
        return {"q": (y / scale).to(torch.float8_e4m3fn), "scale": scale.squeeze(-1), "sum": total}
    dy, hat = s["dy"].float(), v * rstd
    gw = dy * w
    dv = rstd * (gw - hat * (gw * hat).mean(-1, keepdim=True)) + s["dsum"].float()
    dx = dv.to(t)
    return {"y": y.to(t), "sum": total, "dx": dx, "dresidual": dx, "dweight": (dy * hat).sum(0)}


def _tokens(s):
    """per token: its sequence and its place in it; per sequence: first token and length"""
    off = s["offsets"].long()
    lengths = off[1:] - off[:-1]
    T = s["case"]["rows"] * s["case"]["length"]
    seq = torch.repeat_interleave(torch.arange(len(lengths), device=off.device), lengths, output_size=T)
    place = torch.arange(T, device=off.device) - off[seq]
    return seq, place, off[:-1], lengths


def _conv_plain(s):
    c, t = s["case"], s["dtype"]
    W, D = c["width"], c["channels"]
    x, w, b = s["x"].float(), s["weight"], s["bias"]
    state = s.get("state")
    if c["mode"] == "step":
        window = torch.cat([state.float(), x[:, None]], 1)                       # [rows, W, channels]
        pre = (window * w.t()).sum(1) + b
        state.copy_(window[:, 1:])
        return {"out": (pre * torch.sigmoid(pre)).to(t), "state": state}
    seq, place, first, lengths = _tokens(s)
    T = x.shape[0]
    taps = torch.arange(W, device=x.device) - (W - 1)                            # -(W-1) .. 0
    inside = (place[:, None] + taps) >= 0
    source = (torch.arange(T, device=x.device)[:, None] + taps).clamp_min(0)
    window = x[source] * inside[..., None]                                       # [tokens, W, channels]
    if state is not None:                                                        # what lies before a sequence's start
        before = state.float()[seq[:, None], (place[:, None] + taps + W - 1).clamp_max(W - 2)]
        window = torch.where(inside[..., None], window, before)
    pre = (window * w.t()).sum(1) + b
    sig = torch.sigmoid(pre)
    out = (pre * sig).to(t)
    if c["mode"] == "forward":
        # the last W-1 inputs of each sequence, what was carried in among them where it is shorter
        back = torch.arange(W - 1, device=x.device) - (W - 1) + lengths[:, None]   # place in the sequence
        new = torch.where((back >= 0)[..., None], x[(first[:, None] + back).clamp(0, T - 1)],
                          state.float().gather(1, (back + W - 1).clamp(0, W - 2)[..., None].expand(-1, -1, D)))
        return {"out": out, "state": new.to(t)}
    dpre = s["dout"].float() * (sig * (1 + pre * (1 - sig)))
    dw = (dpre[:, None] * window).sum(0).t()
    ahead = torch.arange(T, device=x.device)[:, None] - taps                     # the tokens that read this one
    reads = place[:, None] - taps < lengths[seq][:, None]
    dx = (dpre[ahead.clamp_max(T - 1)] * reads[..., None] * w.t()).sum(1)
    return {"out": out, "dx": dx.to(t), "dweight": dw, "dbias": dpre.sum(0)}


def _linear_recurrence(a, b, longest):
    """h[t] = a[t] h[t-1] + b[t] along the first axis by doubling: after k rounds h[t] holds the last 2^k terms.
    Overwrites both; a is 0 where a sequence starts."""
    reach = 1
    while reach < longest:
        b[reach:] += a[reach:] * b[:-reach]
        a[reach:] = a[reach:] * a[:-reach]
        reach *= 2
    return b


def _scan_plain(s):
    c, t = s["case"], s["dtype"]
    G, N, D = c["groups"], c["states"], c["channels"]
    u, z, A, state = s["u"].float(), s["z"].float(), s["A"], s.get("state")
    pre = s["delta"].float() + s["delta_bias"]
    dt = torch.nn.functional.softplus(pre)
    per = D // G
    B = s["B"].float().repeat_interleave(per, 1)                                 # [tokens, channels, states]
    C = s["C"].float().repeat_interleave(per, 1)
    sig = torch.sigmoid(z)
    a = torch.exp(dt[..., None] * A)
    b = (dt * u)[..., None] * B
    if c["mode"] == "step":
        state.copy_(a * state + b)
        y = (state * C).sum(-1) + s["D"] * u
        return {"out": (y * z * sig).to(t), "state": state}
    seq, place, first, lengths = _tokens(s)
    starts = place == 0
    if state is not None:
        b[starts] += a[starts] * state[seq[starts]]
    link = a.masked_fill(starts[:, None, None], 0.0)
    h = _linear_recurrence(link.clone(), b, s["longest"])
    y = (h * C).sum(-1) + s["D"] * u
    out = (y * z * sig).to(t)
    if c["mode"] == "forward":
        last = h[(first + lengths - 1).clamp_min(0)]
        return {"out": out, "state": torch.where((lengths > 0)[:, None, None], last, state)}
    dout = s["dout"].float()
    dz = dout * y * (sig * (1 + z * (1 - sig)))
    g = dout * z * sig
    # the adjoint runs the other way: dh[t] = C[t] g[t] + a[t+1] dh[t+1]
    ahead = torch.cat([link[1:], torch.zeros_like(link[:1])])
    dh = _linear_recurrence(ahead.flip(0), (C * g[..., None]).flip(0), s["longest"]).flip(0)
    dC = (h * g[..., None]).unflatten(1, (G, per)).sum(2)
    before = torch.cat([torch.zeros_like(h[:1]), h[:-1]]).masked_fill_(starts[:, None, None], 0.0)
    da = dh * before * a
    dA = (da * dt[..., None]).sum(0)
    through = (dh * B).sum(-1)
    ddelta = ((da * A).sum(-1) + through * u) * torch.sigmoid(pre)
    dB = (dh * (dt * u)[..., None]).unflatten(1, (G, per)).sum(2)
    du = through * dt + s["D"] * g
    return {"out": out, "du": du.to(t), "ddelta": ddelta.to(t), "dA": dA, "dB": dB.to(t), "dC": dC.to(t),
            "dD": (g * u).sum(0), "dz": dz.to(t), "ddelta_bias": ddelta.sum(0)}


def run(state):
    if own:
        return _run_own(state)
    return {"norm": _norm_plain, "conv": _conv_plain, "scan": _scan_plain}[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------------------ work
def work(case):
    T, D, N, W, G = (case["rows"] * case["length"], case["channels"], case["states"], case["width"], case["groups"])
    e = 4 if case["dtype"] == "fp32" else 2
    n = case["sequences"] or case["rows"]
    mode = case["mode"]
    if case["op"] == "norm":
        if mode == "train":       # forward: x, residual, weight -> y, sum; backward: dy, dsum, sum -> dx (= dresidual), dw
            return {"bytes": T * D * e * 8 + 8 * D, "flops": T * D * 13}
        out = e if mode == "forward" else 1
        return {"bytes": T * D * (3 * e + out) + 4 * D + (4 * T if mode == "q8" else 0), "flops": T * D * 5}
    if case["op"] == "conv":
        if mode == "train":       # x -> out; x, dout -> dx and the weights' gradients
            return {"bytes": T * D * e * 5 + D * (W + 1) * 8, "flops": T * D * (2 * W + 4) + T * D * (6 * W + 10)}
        return {"bytes": T * D * e * 2 + 2 * n * (W - 1) * D * e + D * (W + 1) * 4, "flops": T * D * (2 * W + 4)}
    params = D * (N + 2) * 4
    per_token = D * (7 * N + 12)
    if mode == "train":           # u, delta, z, B, C -> out; the same and dout -> du, ddelta, dz, dB, dC, dA, dD, dbias
        return {"bytes": T * e * (4 * D + 2 * G * N) + T * e * (7 * D + 4 * G * N) + 3 * params,
                "flops": T * (per_token + D * (18 * N + 24))}
    return {"bytes": T * e * (4 * D + 2 * G * N) + 2 * n * D * N * 4 + params, "flops": T * per_token}


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def _padded(s):
    """token indices [sequences, longest], and which of them exist"""
    off = s["offsets"].long()
    place = torch.arange(max(s["longest"], 1), device=off.device)
    there = place < (off[1:] - off[:-1])[:, None]
    return torch.where(there, off[:-1, None] + place, torch.zeros_like(off[:-1, None])), there


def _exact_scan(s):
    c = s["case"]
    G, N, D = c["groups"], c["states"], c["channels"]
    per, dev = D // G, s["u"].device
    train = c["mode"] == "train"
    T = s["u"].shape[0]
    idx, there = _padded(s)
    S, L = idx.shape
    A, skip = s["A"].double(), s["D"].double()
    pre = s["delta"].double() + s["delta_bias"].double()
    dt = torch.where(pre > 0, pre, torch.zeros_like(pre)) + torch.log1p(torch.exp(-pre.abs()))
    u, z = s["u"].double(), s["z"].double()
    gate = z / (1 + torch.exp(-z))
    channel_group = torch.arange(D, device=dev) // per
    Bm, Cm = s["B"].double(), s["C"].double()
    h = s["state"].double().clone() if "state" in s else torch.zeros(S, D, N, device=dev, dtype=torch.float64)
    y = torch.zeros(T, D, device=dev, dtype=torch.float64)
    kept = torch.empty(L, S, D, N, device=dev, dtype=torch.float64) if train else None
    for i in range(L):
        rows, ok = idx[:, i], there[:, i]
        if train:
            kept[i] = h                                                          # the state before this token
        new = torch.exp(dt[rows][..., None] * A) * h + (dt[rows] * u[rows])[..., None] * Bm[rows][:, channel_group]
        h = torch.where(ok[:, None, None], new, h)
        y[rows[ok]] = ((h * Cm[rows][:, channel_group]).sum(-1) + skip * u[rows])[ok]
    out = y * gate
    if not train:
        return {"out": out, "state": h}
    dout = s["dout"].double()
    sg = 1 / (1 + torch.exp(-z))
    g = dout * gate
    res = {"out": out, "du": skip * g, "ddelta": torch.zeros_like(u), "dA": torch.zeros_like(A),
           "dB": torch.zeros_like(Bm), "dC": torch.zeros_like(Cm), "dD": (g * u).sum(0),
           "dz": dout * y * sg * (1 + z * (1 - sg)), "ddelta_bias": None}
    carry = torch.zeros(S, D, N, device=dev, dtype=torch.float64)
    for i in range(L - 1, -1, -1):
        ok = there[:, i]
        rows = idx[ok, i]
        before, d, uu, gg = kept[i][ok], dt[rows], u[rows], g[rows]
        Bx, Cx = Bm[rows][:, channel_group], Cm[rows][:, channel_group]
        a = torch.exp(d[..., None] * A)
        now = a * before + (d * uu)[..., None] * Bx
        dh = carry[ok] + Cx * gg[..., None]
        res["dC"][rows] = (now * gg[..., None]).view(-1, G, per, N).sum(2)
        res["dB"][rows] = (dh * (d * uu)[..., None]).view(-1, G, per, N).sum(2)
        into = dh * a
        res["dA"] += (into * before * d[..., None]).sum(0)
        hit = (dh * Bx).sum(-1)
        res["du"][rows] += hit * d
        res["ddelta"][rows] = ((into * before * A).sum(-1) + hit * uu) / (1 + torch.exp(-pre[rows]))
        carry[ok] = into
    res["ddelta_bias"] = res["ddelta"].sum(0)
    return res


def _exact_conv(s):
    c = s["case"]
    W, D = c["width"], c["channels"]
    x, w, b = s["x"].double(), s["weight"].double(), s["bias"].double()
    off = s["offsets"].tolist()
    outs, states, dxs = [], [], []
    dw, db = torch.zeros_like(w), torch.zeros_like(b)
    for i, (lo, hi) in enumerate(zip(off[:-1], off[1:])):
        head = s["state"][i].double() if "state" in s else torch.zeros(W - 1, D, device=x.device, dtype=torch.float64)
        line = torch.cat([head, x[lo:hi]])                                       # [W-1+length, channels]
        n = hi - lo
        pre = b.expand(n, D).clone()
        for k in range(W):
            pre += line[k:k + n] * w[:, k]
        sg = 1 / (1 + torch.exp(-pre))
        outs.append(pre * sg)
        states.append(line[n:])
        if c["mode"] == "train":
            d = s["dout"][lo:hi].double() * sg * (1 + pre * (1 - sg))
            dline = torch.zeros_like(line)
            for k in range(W):
                dline[k:k + n] += d * w[:, k]
                dw[:, k] += (d * line[k:k + n]).sum(0)
            db += d.sum(0)
            dxs.append(dline[W - 1:])
    if c["mode"] == "train":
        return {"out": torch.cat(outs), "dx": torch.cat(dxs), "dweight": dw, "dbias": db}
    return {"out": torch.cat(outs), "state": torch.stack(states)}


def _exact_norm(s):
    c = s["case"]
    total = s["x"].double() + s["residual"].double()
    v = total.to(s["dtype"]).double()                     # the norm is that of the stored sum
    w, D = s["weight"].double(), c["channels"]
    r = 1 / torch.sqrt((v * v).sum(-1, keepdim=True) / D + EPS)
    y = w * (v * r)
    if c["mode"] == "forward":
        return {"y": y, "sum": total}
    if c["mode"] == "q8":
        scale = y.abs().max(-1, keepdim=True)[0] / 448.0
        scale = scale + (scale == 0).double()
        return {"q": y / scale, "scale": scale[:, 0], "sum": total}
    dy = s["dy"].double()
    inner = (dy * w * v).sum(-1, keepdim=True)
    dv = r * dy * w - v * inner * r ** 3 / D + s["dsum"].double()
    return {"y": y, "sum": total, "dx": dv, "dresidual": dv, "dweight": (dy * v * r).sum(0)}


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "conv": _exact_conv, "scan": _exact_scan}[case["op"]](s)
