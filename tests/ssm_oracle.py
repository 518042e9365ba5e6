"""The sequence filters in 64 bits, token after token (numpy), and how far
32-bit results may be from them.

Each function also evaluates its formula with every term's magnitude
(``magnitude=True``): no term can cancel another, so the result M bounds what
rounding errors are relative to.  A result of n rounded operations in a row,
each within u = 2^-24 of its value, is within n u M; ``rounds`` counts them.
"""

from __future__ import annotations

import numpy as np

U32 = 2.0 ** -24
# Half the distance between neighbours of the result's type, relative to it:
# 24, 8 and 11 significant bits.
U_OUT = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}
# Results below the type's smallest normal number: half of its smallest step.
TINY = {"float32": 2.0 ** -126, "bfloat16": 2.0 ** -126, "float16": 2.0 ** -25}


def sigmoid(x):
    return 0.5 * (1.0 + np.tanh(0.5 * x))


def softplus(x):
    return np.maximum(x, 0.0) + np.log1p(np.exp(-np.abs(x)))


def _m(x, magnitude):
    return None if x is None else np.abs(x) if magnitude else x


def conv(x, w, bias=None, initial=None, silu=True, grad=None, grad_final=None, magnitude=False):
    """One sequence: x (tokens, channels), w (channels, width).  Returns a dict
    with out, final and, where grad is given, the gradients."""
    t, d = x.shape
    k = w.shape[1]
    x, w, bias, initial = (_m(v, magnitude) for v in (x, w, bias, initial))
    ext = np.concatenate([np.zeros((k - 1, d), dtype=x.dtype) if initial is None else initial, x])
    p = np.zeros((t, d)) + (0 if bias is None else bias)
    for j in range(k):
        p = p + ext[j:j + t] * w[:, j]
    out = p * sigmoid(p) if silu else p
    if magnitude and silu:
        out = p  # |p sigmoid(p)| and its slope times p's error are within 1.1 |p|
    r = {"out": out, "final": ext[t:]}
    if grad is not None:
        s = sigmoid(p)
        dp = grad * s * (1 + p * (1 - s)) if silu else grad
        if magnitude:
            # the slope's own error follows p's: |act''| <= 0.5, |act'| <= 1.1
            dp = np.abs(grad) * (1.1 + 0.5 * p) if silu else np.abs(grad)
        dext = np.zeros_like(ext)
        dw = np.zeros_like(w)
        for j in range(k):
            dext[j:j + t] += dp * w[:, j]
            dw[:, j] = (dp * ext[j:j + t]).sum(0)
        if grad_final is not None:
            dext[t:] += _m(grad_final, magnitude)
        r.update(x=dext[k - 1:], initial=dext[:k - 1], weight=dw, bias=dp.sum(0))
    return r


def scan(u, delta, A, B, C, D=None, z=None, bias=None, initial=None, use_softplus=True, grad=None, grad_final=None,
         magnitude=False):
    """One sequence: u, delta, z (tokens, channels), A (channels, states), B and
    C (tokens, groups, states)."""
    t, d = u.shape
    n = A.shape[1]
    rep = d // B.shape[1]
    raw = delta + (0 if bias is None else bias)
    dt = softplus(raw) if use_softplus else raw
    slope = sigmoid(raw) if use_softplus else np.ones_like(raw)
    a = np.exp(dt[:, :, None] * A)
    gate = np.ones_like(u) if z is None else z * sigmoid(z)
    gslope = np.zeros_like(u) if z is None else sigmoid(z) * (1 + z * (1 - sigmoid(z)))
    D = np.zeros(d) if D is None else D
    if magnitude:
        gslope = sigmoid(z) * (1 + np.abs(z) * (1 - sigmoid(z))) if z is not None else gslope
        u, dt, A, B, C, D, gate, gslope, initial, grad, grad_final = (
            _m(v, True) for v in (u, dt, A, B, C, D, gate, gslope, initial, grad, grad_final))
    Bd, Cd = (np.repeat(v, rep, axis=1) for v in (B, C))  # (tokens, channels, states)
    h = np.zeros((d, n)) if initial is None else initial.copy()
    hs, s = [h], np.zeros((t, d))
    for i in range(t):
        h = a[i] * h + (dt[i] * u[i])[:, None] * Bd[i]
        hs.append(h)
        s[i] = (Cd[i] * h).sum(-1) + D * u[i]
    r = {"out": s * gate, "final": h}
    if grad is not None:
        ds = grad * gate
        g = np.zeros((d, n)) if grad_final is None else grad_final.copy()
        gu, gd, gA = np.zeros((t, d)), np.zeros((t, d)), np.zeros((d, n))
        gB, gC = np.zeros_like(B), np.zeros_like(C)
        for i in range(t - 1, -1, -1):
            g = g + ds[i][:, None] * Cd[i]
            gb = (g * Bd[i]).sum(-1)
            held = a[i] * hs[i]
            gu[i] = D * ds[i] + dt[i] * gb
            gd[i] = (u[i] * gb + (g * held * A).sum(-1)) * slope[i]
            gA += g * held * dt[i][:, None]
            gB[i] = (g * (dt[i] * u[i])[:, None]).reshape(-1, rep, n).sum(1)
            gC[i] = (ds[i][:, None] * hs[i + 1]).reshape(-1, rep, n).sum(1)
            g = a[i] * g
        r.update(u=gu, delta=gd, A=gA, B=gB, C=gC, D=(ds * u).sum(0), z=grad * s * gslope, bias=gd.sum(0), initial=g)
    return r


def scan_rounds(t, A, dt_most, n, summed=1):
    """Roundings that a result of a t-token scan went through: each token's
    decay has its argument's (the product, A's factor log2(e), and dt's own
    within 2 |delta| + 8 of them) and the exponential's, a few more for the
    update; n states and `summed` values are added up; activations take a few."""
    x = float(np.max(np.abs(A))) * dt_most
    return (t + 2) * (12.0 * x + 6.0) + n + summed + 32


def within(got, want, m, rounds, dtype, what=""):
    """Whether got is within the bound of want everywhere, with the worst place."""
    got, want, m = (np.asarray(v, dtype=np.float64) for v in (got, want, m))
    assert got.shape == want.shape, (what, got.shape, want.shape)
    if not got.size:
        return
    assert np.isfinite(want).all() and np.isfinite(got).all(), what
    most = U_OUT[dtype] * np.abs(want) + (1 + U_OUT[dtype]) * rounds * U32 * m + TINY[dtype]
    over = np.abs(got - want) - most
    at = np.unravel_index(np.argmax(over), over.shape)
    assert over[at] <= 0, f"{what} at {at}: got {got[at]}, want {want[at]}, bound {most[at]}"
