"""The 64-bit oracle of the sequence filters (tests/ssm_oracle.py) on its own:
its gradients against central differences, its scan against the convolution
that a constant filter is, and its bound against 32-bit evaluations."""

from __future__ import annotations

import numpy as np
import pytest

import ssm_oracle as o


def _conv_case(rng, t, d, k):
    return dict(x=rng.standard_normal((t, d)), w=rng.standard_normal((d, k)), bias=rng.standard_normal(d),
                initial=rng.standard_normal((k - 1, d)))


def _scan_case(rng, t, d, n, groups):
    return dict(u=rng.standard_normal((t, d)), delta=rng.standard_normal((t, d)),
                A=-rng.uniform(0.1, 2.0, (d, n)), B=rng.standard_normal((t, groups, n)),
                C=rng.standard_normal((t, groups, n)), D=rng.standard_normal(d), z=rng.standard_normal((t, d)),
                bias=rng.standard_normal(d), initial=rng.standard_normal((d, n)))


# Five-point differences in extended precision with step h: the fifth
# derivative's term h^4 and rounding 2^-64 / h, also of losses of some 10^4 (a
# scan without softplus grows where delta is negative), stay below 1e-7 at
# h = 1e-5.
H, TOL = 1e-5, 1e-6


def _differences(f, args, name, rng):
    """The derivative of f along a random direction of one argument."""
    v = rng.standard_normal(args[name].shape)

    def at(k):
        return f({n: x.astype(np.longdouble) + (k * H * v if n == name else 0) if x is not None else None
                  for n, x in args.items()})

    return float((8 * (at(1) - at(-1)) - (at(2) - at(-2))) / (12 * np.longdouble(H))), v


@pytest.mark.parametrize("t,d,k,silu", [(7, 3, 4, True), (1, 2, 3, True), (2, 2, 5, False), (0, 2, 3, True)])
def test_conv_gradients_are_differences(t, d, k, silu):
    rng = np.random.default_rng(10 * t + k)
    args = _conv_case(rng, t, d, k)
    gy, gf = rng.standard_normal((t, d)), rng.standard_normal((k - 1, d))

    def loss(a):
        r = o.conv(**a, silu=silu)
        return (r["out"] * gy).sum() + (r["final"] * gf).sum()

    g = o.conv(**args, silu=silu, grad=gy, grad_final=gf)
    for name, of in (("x", "x"), ("w", "weight"), ("bias", "bias"), ("initial", "initial")):
        want, v = _differences(loss, args, name, rng)
        assert abs((g[of] * v).sum() - want) <= TOL * (1 + abs(want)), name


@pytest.mark.parametrize("t,d,n,groups,use_softplus", [(6, 4, 3, 2, True), (1, 2, 1, 1, True), (5, 3, 2, 1, False),
                                                       (0, 2, 2, 1, True)])
def test_scan_gradients_are_differences(t, d, n, groups, use_softplus):
    rng = np.random.default_rng(100 * t + n)
    args = _scan_case(rng, t, d, n, groups)
    gy, gf = rng.standard_normal((t, d)), rng.standard_normal((d, n))

    def loss(a):
        r = o.scan(**a, use_softplus=use_softplus)
        return (r["out"] * gy).sum() + (r["final"] * gf).sum()

    g = o.scan(**args, use_softplus=use_softplus, grad=gy, grad_final=gf)
    for name in args:
        want, v = _differences(loss, args, name, rng)
        assert abs((g[name] * v).sum() - want) <= TOL * (1 + abs(want)), name


def test_constant_scan_is_a_convolution():
    rng = np.random.default_rng(3)
    t, d, n = 40, 3, 4
    c = _scan_case(rng, t, d, n, 1)
    c.update(delta=np.zeros((t, d)), B=np.tile(c["B"][:1], (t, 1, 1)), C=np.tile(c["C"][:1], (t, 1, 1)), z=None,
             initial=None)
    dt = o.softplus(c["bias"])
    i = np.arange(t)
    kernel = np.einsum("n,tdn,n,d->td", c["C"][0, 0], np.exp(i[:, None, None] * dt[:, None] * c["A"]), c["B"][0, 0],
                       dt)
    want = np.stack([np.convolve(c["u"][:, j], kernel[:, j])[:t] for j in range(d)], 1) + c["D"] * c["u"]
    assert np.allclose(o.scan(**c)["out"], want, rtol=1e-12, atol=1e-12)


@pytest.mark.parametrize("seed", range(4))
def test_bound_holds_for_32_bit_arithmetic(seed):
    """The recurrence in float32 stays within the bound of the 64-bit one."""
    rng = np.random.default_rng(seed)
    t, d, n = 150, 8, 5
    c = _scan_case(rng, t, d, n, 1)
    c = {k: v.astype(np.float32).astype(np.float64) for k, v in c.items()}
    f = {k: v.astype(np.float32) for k, v in c.items()}
    raw = f["delta"] + f["bias"]
    dt = np.maximum(raw, 0) + np.log1p(np.exp(-np.abs(raw)))
    h, out = f["initial"], []
    for i in range(t):
        h = np.exp(dt[i][:, None] * f["A"]) * h + (dt[i] * f["u"][i])[:, None] * f["B"][i]
        y = (f["C"][i] * h).sum(-1) + f["D"] * f["u"][i]
        out.append(y * f["z"][i] * (1 / (1 + np.exp(-f["z"][i]))))
    assert out[0].dtype == np.float32
    want, m = o.scan(**c), o.scan(**c, magnitude=True)
    rounds = o.scan_rounds(t, c["A"], dt.max(), n)
    o.within(np.stack(out), want["out"], m["out"], rounds, "float32", "out")
    o.within(h, want["final"], m["final"], rounds, "float32", "final")


def test_bound_sees_a_wrong_term():
    """A scan whose oracle forgets one token's input is outside the bound."""
    rng = np.random.default_rng(9)
    c = _scan_case(rng, 60, 4, 4, 1)
    want, m = o.scan(**c), o.scan(**c, magnitude=True)
    bad = dict(c, B=c["B"].copy())
    bad["B"][30] = 0
    rounds = o.scan_rounds(60, c["A"], 5.0, 4)
    with pytest.raises(AssertionError, match="out at"):
        o.within(o.scan(**bad)["out"], want["out"], m["out"], rounds, "float32", "out")
