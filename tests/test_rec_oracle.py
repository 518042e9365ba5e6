"""The recurrence's oracle against automatic differentiation in 64 bits, on the CPU."""

import torch

import rec_oracle as oracle


def test_gradients_are_those_of_the_definition():
    torch.manual_seed(0)
    n, ch = 9, 5
    v = [torch.randn(n, ch).double().requires_grad_() for _ in range(3)]
    p = [torch.randn(ch).double().requires_grad_() for _ in range(3)]
    h0 = torch.randn(ch).double().requires_grad_()
    grad, last = torch.randn(n, ch).double(), torch.randn(ch).double()
    r, i = torch.sigmoid(v[1] + p[1]), torch.sigmoid(v[2] + p[2])
    a = torch.exp(-8.0 * torch.nn.functional.softplus(p[0]) * r)
    h, outs = h0, []
    for t in range(n):
        h = a[t] * h + torch.sqrt(1 - a[t] ** 2) * i[t] * v[0][t]
        outs.append(h)
    ((torch.stack(outs) * grad).sum() + (h * last).sum()).backward()
    with torch.no_grad():
        out, _, end = oracle.forward(*v, *p, 8.0, h0)
        got, by = oracle.backward(*v, *p, 8.0, h0, grad, last)
    assert torch.allclose(out, torch.stack(outs)) and torch.allclose(end, h)
    for k, x in zip(("x", "gate_a", "gate_x", "decay", "bias_a", "bias_x", "initial"), (*v, *p, h0)):
        assert torch.allclose(got[k], x.grad, rtol=1e-9, atol=1e-12), k
        assert (got[k].abs() <= by[k] + 1e-12).all(), k
