"""The gated linear recurrence token after token in 64 bits, and its gradients
by the formulas; sequences apart, in plain torch on the CPU."""

from __future__ import annotations

import torch


def softplus(x):
    return torch.where(x > 30, x, torch.log1p(torch.exp(x.clamp(max=30))))


def terms(x, ga, gx, decay, ba, bx, rate):
    """r, i, log a, a, m of tokens [n, channels]."""
    r, i = torch.sigmoid(ga + ba), torch.sigmoid(gx + bx)
    log_a = -rate * softplus(decay) * r
    return r, i, log_a, torch.exp(log_a), torch.sqrt(-torch.expm1(2 * log_a))


def forward(x, ga, gx, decay, ba, bx, rate, initial):
    """One sequence [n, channels]: its outputs, the states before its tokens, the last state."""
    _, i, _, a, m = terms(x, ga, gx, decay, ba, bx, rate)
    h, before, out = initial.clone(), torch.empty_like(x), torch.empty_like(x)
    for t in range(x.shape[0]):
        before[t] = h
        h = a[t] * h + m[t] * i[t] * x[t]
        out[t] = h
    return out, before, h


def backward(x, ga, gx, decay, ba, bx, rate, initial, grad, grad_final):
    """Gradients of one sequence, and of each what its rounding errors go by: sums of absolute values."""
    r, i, log_a, a, m = terms(x, ga, gx, decay, ba, bx, rate)
    _, before, _ = forward(x, ga, gx, decay, ba, bx, rate, initial)
    d, dh, size, sizes = grad_final.clone(), torch.empty_like(x), grad_final.abs(), torch.empty_like(x)
    for t in range(x.shape[0] - 1, -1, -1):
        dh[t], sizes[t] = grad[t] + d, grad[t].abs() + size
        d, size = a[t] * dh[t], a[t] * sizes[t]
    closed = m == 0
    over = torch.where(closed, 0, a * a / torch.where(closed, 1, m))
    log = dh * (a * before - i * x * over)
    log_size = sizes * (a * before.abs() + (i * x).abs() * over)
    k = -rate * softplus(decay)
    slope = -rate * torch.sigmoid(decay)
    gate_a, gate_x = log * k * r * (1 - r), dh * m * x * i * (1 - i)
    got = {"x": dh * m * i, "gate_a": gate_a, "gate_x": gate_x, "decay": (log * r).sum(0) * slope,
           "bias_a": gate_a.sum(0), "bias_x": gate_x.sum(0), "initial": d}
    a_size, x_size = log_size * k.abs() * r, sizes * m * x.abs() * i
    by = {"x": sizes * m * i, "gate_a": a_size, "gate_x": x_size, "decay": (log_size * r).sum(0) * slope.abs(),
          "bias_a": a_size.sum(0), "bias_x": x_size.sum(0), "initial": size}
    return got, by
