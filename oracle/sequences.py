"""The sequence operators from their formulas in float64, one sequence at a time, and the magnitudes
that bound the rounding errors of any float32 evaluation.

``magnitude=True`` evaluates the same formulas with every factor replaced by its absolute value and every
difference by a sum: a float32 result is then off by at most (roundings along the longest chain) * 2^-24
times that."""

import numpy as np


def sigmoid(v):
    return 0.5 * (1 + np.tanh(0.5 * v))


def silu(v):
    return v * sigmoid(v)


def silu_slope(v, magnitude=False):
    s = sigmoid(v)
    return s * (1 + (np.abs(v) if magnitude else v) * (1 - s))


def _abs(magnitude, *arrays):
    return [None if a is None else np.abs(a) if magnitude else np.asarray(a, dtype=np.float64) for a in arrays]


# ---- short causal convolution ----------------------------------------------------------------
def causal_conv(x, w, bias=None, state=None, silu_=False, magnitude=False):
    """(y, new_state); ``magnitude``: of the sum before the activation (silu never enlarges an error by
    more than 1.1)."""
    x, w, bias, state = _abs(magnitude, x, w, bias, state)
    taps = w.shape[1]
    rows, chan = x.shape
    line = np.concatenate([np.zeros((taps - 1, chan)) if state is None else state, x])
    pre = np.zeros((rows, chan)) + (0 if bias is None else bias)
    for j in range(taps):
        pre = pre + w[:, j] * line[j:j + rows]
    return (silu(pre) if silu_ and not magnitude else pre), line[rows:]


def causal_conv_grad(x, w, dy, bias=None, state=None, dnew_state=None, silu_=False, magnitude=False):
    """dict of dx, dw, dbias, dstate"""
    pre, _ = causal_conv(x, w, bias, state)
    x, w, dy, state, dnew_state = _abs(magnitude, x, w, dy, state, dnew_state)
    taps = w.shape[1]
    rows, chan = x.shape
    line = np.concatenate([np.zeros((taps - 1, chan)) if state is None else state, x])
    if silu_:
        # (the slope's own error comes from that of `pre`: |silu''| <= 1/2)
        dy = dy * (silu_slope(pre, True) + np.abs(pre) + 1 if magnitude else silu_slope(pre))
    dline = np.zeros_like(line)
    dw = np.zeros_like(w)
    for j in range(taps):
        dline[j:j + rows] += w[:, j] * dy
        dw[:, j] = (dy * line[j:j + rows]).sum(0)
    if dnew_state is not None:
        dline[rows:] += dnew_state
    return dict(dx=dline[taps - 1:], dw=dw, dbias=dy.sum(0), dstate=dline[:taps - 1])


# ---- selective state space scan --------------------------------------------------------------
def scan_steps(dt, dt_bias=None, softplus=False):
    raw = np.asarray(dt, dtype=np.float64) + (0 if dt_bias is None else np.asarray(dt_bias, dtype=np.float64))
    return raw, (np.logaddexp(0, raw) if softplus else raw)


def _heads(v, groups, chan):
    rows = v.shape[0]
    return np.repeat(v.reshape(rows, groups, v.shape[1] // groups), chan // groups, axis=1)


def selective_scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, softplus=False, state=None, magnitude=False,
                   history=False):
    """(y, new_state) [, states before every row, sum before the gate]"""
    _, s = scan_steps(dt, dt_bias, softplus)
    A = np.asarray(A, dtype=np.float64)
    rows, chan = x.shape
    n = A.shape[1]
    groups = B.shape[1] // n
    gate = None if z is None else silu(np.asarray(z, dtype=np.float64))
    x, B, C, D, gate, state, sm = _abs(magnitude, x, B, C, D, gate, state, s)
    h = np.zeros((chan, n)) if state is None else state.copy()
    B, C = _heads(B, groups, chan), _heads(C, groups, chan)
    before, p = np.zeros((rows, chan, n)), np.zeros((rows, chan))
    for t in range(rows):
        before[t] = h
        h = np.exp(s[t][:, None] * A) * h + (sm[t] * x[t])[:, None] * B[t]
        p[t] = (C[t] * h).sum(1) + (0 if D is None else D * x[t])
    y = p if gate is None else p * gate
    return (y, h, before, p) if history else (y, h)


def selective_scan_grad(x, dt, A, B, C, dy, D=None, z=None, dt_bias=None, softplus=False, state=None, dnew_state=None,
                        magnitude=False):
    """dict of dx, ddt, dA, dB, dC, dD, dz, ddt_bias, dstate"""
    _, _, before, p = selective_scan(x, dt, A, B, C, D, None, dt_bias, softplus, state, magnitude, history=True)
    raw, s = scan_steps(dt, dt_bias, softplus)
    A = np.asarray(A, dtype=np.float64)
    rows, chan = x.shape
    n = A.shape[1]
    groups = B.shape[1] // n
    z = None if z is None else np.asarray(z, dtype=np.float64)
    gate = None if z is None else silu(z)
    x, B, C, D, gate, dy, dnew_state, Am, sm = _abs(magnitude, x, B, C, D, gate, dy, dnew_state, A, s)
    B, C = _heads(B, groups, chan), _heads(C, groups, chan)
    dp = dy if gate is None else dy * gate
    carry = np.zeros((chan, n)) if dnew_state is None else dnew_state.copy()
    dx, ds, dA = np.zeros((rows, chan)), np.zeros((rows, chan)), np.zeros((chan, n))
    dB, dC = np.zeros((rows, groups, n)), np.zeros((rows, groups, n))
    over = lambda v: v.reshape(groups, chan // groups, n).sum(1)
    for t in range(rows - 1, -1, -1):
        a = np.exp(s[t][:, None] * A)
        h = a * before[t] + (sm[t] * x[t])[:, None] * B[t]
        g = C[t] * dp[t][:, None] + carry
        carry = g * a
        q = carry * before[t]
        u = (g * B[t]).sum(1)
        dx[t] = (0 if D is None else D * dp[t]) + sm[t] * u
        ds[t] = x[t] * u + (q * Am).sum(1)
        dA += q * sm[t][:, None]
        dB[t], dC[t] = over(g * (sm[t] * x[t])[:, None]), over(dp[t][:, None] * h)
    if softplus:
        ds = ds * sigmoid(raw)
    out = dict(dx=dx, ddt=ds, dA=dA, dB=dB.reshape(rows, groups * n), dC=dC.reshape(rows, groups * n), dD=(dp * x).sum(0),
               ddt_bias=ds.sum(0), dstate=carry)
    if z is not None:
        out["dz"] = dy * p * silu_slope(z, magnitude)
    return out


# ---- norms around a block --------------------------------------------------------------------
def residual_norm(x, gate=None, gate_first=True, residual=None, weight=None, scale=1.0, norm_weight=None, groups=1,
                  eps=1e-5, parts=False):
    """(y, h) [, intermediate values]"""
    x, gate, residual, weight, norm_weight, scale = _abs(False, x, gate, residual, weight, norm_weight, scale)
    rows, chan = x.shape
    sg = 1.0 if gate is None else silu(gate)
    u = x * sg if gate_first else x
    if weight is not None:
        lead = u.reshape(rows, groups, chan // groups)
        inv = np.repeat(1 / np.sqrt((lead ** 2).mean(-1) + eps), chan // groups, axis=1)
        hat = u * inv
        v = hat * weight
    else:
        inv, hat, v = np.ones_like(u), u, u
    o = v if gate_first else v * sg
    y = scale * o + (0 if residual is None else residual)
    rinv = 1 / np.sqrt((y ** 2).mean(-1, keepdims=True) + eps)
    h = y * rinv * (1 if norm_weight is None else norm_weight)
    return (y, h, (sg, u, inv, hat, o, rinv)) if parts else (y, h)


def residual_norm_grad(x, dy=None, dh=None, gate=None, gate_first=True, residual=None, weight=None, scale=1.0,
                       norm_weight=None, groups=1, eps=1e-5):
    """dict of dx, dgate, dresidual, dweight, dscale, dnorm_weight"""
    y, _, (sg, u, inv, hat, o, rinv) = residual_norm(x, gate, gate_first, residual, weight, scale, norm_weight, groups,
                                                     eps, parts=True)
    x, gate, weight, norm_weight, dy, dh = _abs(False, x, gate, weight, norm_weight, dy, dh)
    rows, chan = x.shape
    dr = np.zeros((rows, chan)) if dy is None else dy.copy()
    out = {}
    if dh is not None:
        yhat = y * rinv
        e = dh * (1 if norm_weight is None else norm_weight)
        dr = dr + rinv * (e - yhat * (e * yhat).mean(-1, keepdims=True))
        out["dnorm_weight"] = (dh * yhat).sum(0)
    out["dresidual"], out["dscale"] = dr, (dr * o).sum(0)
    do = dr * scale
    dv = do if gate_first else do * sg
    out["dweight"] = (dv * hat).sum(0)
    if weight is not None:
        e = (dv * weight).reshape(rows, groups, chan // groups)
        hat3 = hat.reshape(rows, groups, chan // groups)
        du = inv * (e - hat3 * (e * hat3).mean(-1, keepdims=True)).reshape(rows, chan)
    else:
        du = dv
    out["dx"] = du * sg if gate_first else du
    if gate is not None:
        v = hat * (1 if weight is None else weight)
        out["dgate"] = (du * x if gate_first else do * v) * silu_slope(gate)
    return out
