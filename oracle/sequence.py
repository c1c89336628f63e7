"""64-bit CPU definitions of the sequence operators (fastdeepqlearning_amd/sequence.py): outputs and hand-written adjoints, step by step.
With ``mag`` every term enters with its absolute value, so each result bounds the sum of its terms' magnitudes: what a rounding
error bound of a float32 evaluation is proportional to."""
import math

import torch


def _f64(t):
    return None if t is None else t.detach().cpu().double()


def _abs(t, mag):
    return t.abs() if mag and t is not None else t


def causal_conv(x, weight, bias=None, state=None, reset=None, silu=True, dy=None, dstate=None, mag=False):
    """dict of y, state and - with dy - dx, dweight, dbias, dstate.  [T, R, D] tensors; mag: |weight|, |x|, |dy| throughout."""
    x0, w0, b0, s0 = _f64(x), _f64(weight), _f64(bias), _f64(state)
    T, R, D = x0.shape
    K = w0.shape[1]
    s0 = torch.zeros(R, K - 1, D, dtype=torch.float64) if s0 is None else s0
    b0 = torch.zeros(D, dtype=torch.float64) if b0 is None else b0
    rst = torch.zeros(T, R, dtype=torch.bool) if reset is None else reset.cpu().bool()

    def forward(xx, ww, bb, ss):
        win = torch.cat([torch.zeros(R, 1, D, dtype=torch.float64), ss], 1)
        pre, wins = [], []
        for t in range(T):
            old = torch.where(rst[t][:, None, None], torch.zeros((), dtype=torch.float64), win[:, 1:])
            win = torch.cat([old, xx[t][:, None]], 1)
            wins.append(win)
            pre.append((win * ww.t()).sum(1) + bb)
        return pre, wins, win[:, 1:]

    pre, wins, last = forward(x0, w0, b0, s0)
    out = {"state": last}
    if mag:
        mpre, mwins, _ = forward(x0.abs(), w0.abs(), b0.abs(), s0.abs())
        out["y"] = torch.stack(mpre) * 1.1 if T else torch.zeros(0, R, D, dtype=torch.float64)   # |SiLU'| <= 1.1
    else:
        out["y"] = torch.stack([p * torch.sigmoid(p) if silu else p for p in pre]) if T else torch.zeros(0, R, D, dtype=torch.float64)
    if dy is None:
        return out
    g0, ds = _abs(_f64(dy), mag), _abs(_f64(dstate), mag)
    dx = torch.zeros(K - 1 + T, R, D, dtype=torch.float64)
    dw, db = torch.zeros(D, K, dtype=torch.float64), torch.zeros(D, dtype=torch.float64)
    ww = _abs(w0, mag)
    if ds is not None:
        for k in range(K - 1):
            t = T - (K - 1) + k
            gone = rst[max(t, -1) + 1:].any(0)
            dx[t + K - 1] += torch.where(gone[:, None], 0.0, ds[:, k])
    for t in range(T):
        if mag:      # |SiLU'| <= 1.1, and its own error is that of pre: |SiLU''| <= 0.5
            d = g0[t] * (1.1 + 0.5 * mpre[t]) if silu else g0[t]
            win = mwins[t]
        else:
            s = torch.sigmoid(pre[t])
            d = g0[t] * s * (1 + pre[t] * (1 - s)) if silu else g0[t]
            win = wins[t]
        db += d.sum(0)
        dw += (d[:, None] * win).sum(0).t()
        cut = torch.zeros(R, dtype=torch.bool)
        for j in range(K):
            dx[t - j + K - 1] += torch.where(cut[:, None], 0.0, d * ww[:, K - 1 - j])
            if t - j >= 0:
                cut = cut | rst[t - j]
    out.update(dx=dx[K - 1:], dweight=dw, dbias=db, dstate=dx[:K - 1].transpose(0, 1))
    return out


def selective_scan(x, dt, A, B, C, skip=None, z=None, dt_bias=None, softplus=True, state=None, reset=None, dy=None, dstate=None, mag=False):
    """dict of y, state and - with dy - every gradient.  [T, R, D] tensors, B and C [T, R, G, N]; mag: absolute values of all factors but
    the decays."""
    x, dt, A, B, C, skip, z, dt_bias = (_f64(t) for t in (x, dt, A, B, C, skip, z, dt_bias))
    T, R, D = x.shape
    G, N = B.shape[-2:]
    h = torch.zeros(R, D, N, dtype=torch.float64) if state is None else _f64(state)
    rst = torch.zeros(T, R, dtype=torch.bool) if reset is None else reset.cpu().bool()
    raw = dt if dt_bias is None else dt + dt_bias
    delta = torch.logaddexp(raw, torch.zeros((), dtype=torch.float64)) if softplus else raw
    slope = torch.sigmoid(raw) if softplus else torch.ones_like(raw)
    sg = None if z is None else torch.sigmoid(z)
    gate = torch.ones_like(x) if z is None else z * sg
    decay = torch.exp(delta[..., None] * A)
    x, B, C, skip, gate, h = (_abs(t, mag) for t in (x, B, C, skip, gate, h))
    direct = lambda m: 0.0 if skip is None else skip * m  # noqa: E731
    step = _abs(delta, mag)
    wide = lambda m: m.repeat_interleave(D // G, 1)  # noqa: E731
    fold = lambda m: m.view(R, G, D // G, N).sum(2)  # noqa: E731
    zero = torch.zeros((), dtype=torch.float64)
    hs, core = [h], []
    for t in range(T):
        h = torch.where(rst[t][:, None, None], zero, decay[t] * h) + (step[t] * x[t])[..., None] * wide(B[t])
        hs.append(h)
        core.append((h * wide(C[t])).sum(-1) + direct(x[t]))
    core = torch.stack(core) if T else torch.zeros_like(x)
    out = {"y": core * gate, "state": h}
    if dy is None:
        return out
    dout = _abs(_f64(dy), mag)
    g_core = dout * gate
    carry = torch.zeros(R, D, N, dtype=torch.float64) if dstate is None else _abs(_f64(dstate), mag)
    Am = _abs(A, mag)
    dx, ddt, dB, dC, dA = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(B), torch.zeros_like(C), torch.zeros_like(A)
    for t in reversed(range(T)):
        g = carry + g_core[t][..., None] * wide(C[t])
        carry = torch.where(rst[t][:, None, None], zero, g * decay[t])
        past = torch.where(rst[t][:, None, None], zero, g * decay[t] * hs[t])
        gb = (g * wide(B[t])).sum(-1)
        dx[t] = direct(g_core[t]) + step[t] * gb
        ddt[t] = ((past * Am).sum(-1) + gb * x[t]) * slope[t]
        dA += (past * step[t][..., None]).sum(0)
        dB[t] = fold(g * (step[t] * x[t])[..., None])
        dC[t] = fold(hs[t + 1] * g_core[t][..., None])
    out.update(dx=dx, ddt=ddt, dA=dA, dB=dB, dC=dC, dskip=(g_core * x).sum((0, 1)), ddt_bias=ddt.sum((0, 1)), dstate=carry)
    if z is not None:
        out["dz"] = dout * core * (1.1 if mag else sg * (1 + z * (1 - sg)))
    return out


def activation(kind, g):
    """f(g), f'(g)"""
    s = torch.sigmoid(g)
    if kind == "silu":
        return g * s, s * (1 + g * (1 - s))
    if kind == "sigmoid":
        return s, s * (1 - s)
    cdf = 0.5 * torch.erfc(-g / math.sqrt(2))
    return g * cdf, cdf + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)


def gated_linear(x, w_gate, w_up, b_gate=None, b_up=None, kind="silu", dy=None):
    """dict of y, the magnitudes mg, mu of the two products' terms, and - with dy - every gradient and its terms' magnitude (m_*)."""
    x, w_gate, w_up, b_gate, b_up = (_f64(t) for t in (x, w_gate, w_up, b_gate, b_up))
    g, u = x @ w_gate.t(), x @ w_up.t()
    mg, mu = x.abs() @ w_gate.abs().t(), x.abs() @ w_up.abs().t()
    if b_gate is not None:
        g, u, mg, mu = g + b_gate, u + b_up, mg + b_gate.abs(), mu + b_up.abs()
    f, df = activation(kind, g)
    out = {"y": f * u, "m_y": 1.2 * mg * u.abs() + f.abs() * mu}        # |f'| <= 1.13 for all three
    if dy is None:
        return out
    dy = _f64(dy)
    dg, du = dy * u * df, dy * f
    out.update(dx=dg @ w_gate + du @ w_up, dw_gate=dg.t() @ x, dw_up=du.t() @ x, db_gate=dg.sum(0), db_up=du.sum(0))
    out.update(r_dx=dg.abs() @ w_gate.abs() + du.abs() @ w_up.abs(), r_dw_gate=dg.abs().t() @ x.abs(), r_dw_up=du.abs().t() @ x.abs(),
               r_db_gate=dg.abs().sum(0), r_db_up=du.abs().sum(0))
    eg, eu = dy.abs() * (1.2 * mu + u.abs() * mg), dy.abs() * 1.2 * mg  # what the products' errors do to dg, du (|f''| <= 1)
    out.update(e_dx=eg @ w_gate.abs() + eu @ w_up.abs(), e_dw_gate=eg.t() @ x.abs(), e_dw_up=eu.t() @ x.abs(), e_db_gate=eg.sum(0), e_db_up=eu.sum(0))
    return out
