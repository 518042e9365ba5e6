"""The sequence filters as a model uses them: a block that mixes a sequence's
tokens with a short causal convolution and a selective scan, run over a prompt,
then token by token with its states in a cache, and trained.

    python ferrum-gpu_amd/examples/sequence_filters.py

The block's projections are torch products, and the filters run on torch's current
stream between them, so the host waits for nothing.  torch is imported before
the package, as it has to be.
"""

from __future__ import annotations

import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__)))))
import ferrum_gpu  # noqa: E402
from ferrum_gpu import ssm  # noqa: E402


class Block:
    """x -> conv -> silu -> (delta, B, C) -> scan, gated by z."""

    def __init__(self, device: ferrum_gpu.hip.Device, channels=256, states=16, width=4, rank=16, dtype=torch.float32,
                 seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        rand = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
        self.device, self.channels, self.states, self.width, self.rank = device, channels, states, width, rank
        self.dtype, self.name, self.plans = dtype, str(dtype).rpartition(".")[2], {}
        self.weight, self.bias = 0.5 * rand(channels, width), 0.1 * rand(channels)
        self.project = (rand(channels, rank + 2 * states) / channels ** 0.5).to(dtype)
        self.widen = (rand(rank, channels) / rank ** 0.5).to(dtype)
        self.A = -torch.arange(1, states + 1, device="cuda", dtype=torch.float32).repeat(channels, 1)
        self.D, self.delta_bias = torch.ones(channels, device="cuda"), torch.full((channels,), -3.0, device="cuda")

    def _plans(self, batch, length):
        """Both filters' plans for sequences of this shape, made once."""
        if (batch, length) not in self.plans:
            self.plans[batch, length] = (
                ssm.ConvPlan(batch, length, self.channels, self.width, self.device, dtype=self.name),
                ssm.ScanPlan(batch, length, self.channels, self.states, self.device, dtype=self.name))
        return self.plans[batch, length]

    def _split(self, u):
        p = u @ self.project
        r, n = self.rank, self.states
        return p[..., :r] @ self.widen, p[..., r:r + n], p[..., r + n:]

    def prompt(self, x, z, conv_state, scan_state):
        """Outputs for whole sequences; the states are left for what follows."""
        u, out = torch.empty_like(x), torch.empty_like(x)
        conv, scan = self._plans(*x.shape[:2])
        here = torch.cuda.current_stream()
        conv.forward(x, self.weight, u, bias=self.bias, initial=conv_state, final=conv_state, stream=here)
        delta, b, c = self._split(u)
        scan.forward(u, delta, self.A, b, c, out, D=self.D, z=z, delta_bias=self.delta_bias, initial=scan_state,
                     final=scan_state, stream=here)
        return out

    def token(self, x, z, conv_state, scan_state, slots):
        """Outputs for one token of each row, whose states lie in cache slots."""
        u, out = torch.empty_like(x), torch.empty_like(x)
        here = torch.cuda.current_stream()
        ssm.conv_step(self.device, x, self.weight, conv_state, u, bias=self.bias, slots=slots, stream=here)
        delta, b, c = self._split(u)
        ssm.scan_step(self.device, u, delta, self.A, b, c, scan_state, out, D=self.D, z=z,
                      delta_bias=self.delta_bias, slots=slots, stream=here)
        return out

    def gradients(self, x, z, grad):
        """Gradients of the convolution's and the scan's parameters and of x and z."""
        u, out = torch.empty_like(x), torch.empty_like(x)
        conv, scan = self._plans(*x.shape[:2])
        check = torch.empty(scan.checkpoint_bytes, dtype=torch.uint8, device="cuda")
        here = torch.cuda.current_stream()
        conv.forward(x, self.weight, u, bias=self.bias, stream=here)
        delta, b, c = self._split(u)
        g = {k: torch.empty_like(v) for k, v in dict(u=u, delta=delta, A=self.A, B=b, C=c, D=self.D, z=z,
                                                     delta_bias=self.delta_bias).items()}
        scan.forward(u, delta, self.A, b, c, out, D=self.D, z=z, delta_bias=self.delta_bias, checkpoints=check,
                     stream=here)
        scan.backward(u, delta, self.A, b, c, grad, check, D=self.D, z=z, delta_bias=self.delta_bias,
                      **{"grad_" + k: v for k, v in g.items()}, stream=here)
        r, n = self.rank, self.states
        p = torch.cat([g["delta"] @ self.widen.t().contiguous(), g["B"], g["C"]], -1)
        g["u"] += p @ self.project.t().contiguous()
        g["x"], g["weight"], g["bias"] = torch.empty_like(x), torch.empty_like(self.weight), torch.empty_like(self.bias)
        conv.backward(x, self.weight, g["u"], grad_x=g["x"], grad_weight=g["weight"], grad_bias=g["bias"],
                      bias=self.bias, stream=here)
        return out, g


def main(device=None) -> dict:
    """Runs the block all three ways and returns how far they are apart."""
    device = device or ferrum_gpu.hip.Device(0)
    torch.manual_seed(0)
    block = Block(device)
    batch, length, more, rows = 3, 50, 8, 5
    x = torch.randn(batch, length + more, block.channels, device="cuda")
    z = torch.randn_like(x)
    states = lambda n: (torch.zeros(n, block.width - 1, block.channels, device="cuda"),  # noqa: E731
                        torch.zeros(n, block.channels, block.states, device="cuda"))
    whole = block.prompt(x, z, *states(batch))
    # the prompt's states go to slots of a larger cache, where the tokens find them
    conv_state, scan_state = states(batch)
    block.prompt(x[:, :length], z[:, :length], conv_state, scan_state)
    slots = torch.tensor([4, 0, 2], dtype=torch.int32, device="cuda")
    conv_cache, scan_cache = states(rows)
    conv_cache[slots.long()], scan_cache[slots.long()] = conv_state, scan_state
    apart = 0.0
    for t in range(length, length + more):
        y = block.token(x[:, t], z[:, t], conv_cache, scan_cache, slots)
        apart = max(apart, ((y - whole[:, t]).abs().max() / whole.abs().max()).item())
    # a step along the gradient's direction changes the loss by its length
    grad = torch.randn_like(x)
    out, g = block.gradients(x, z, grad)
    step = 1e-2 / g["x"].norm()
    loss = [(block.prompt(x + s * step * g["x"], z, *states(batch)).double() * grad).sum().item() for s in (1, -1)]
    slope = (loss[0] - loss[1]) / (2 * 1e-2)
    got = {"tokens against the whole": apart, "same block forward": ((out - whole).abs().max()).item(),
           "slope against the gradient": abs(slope / g["x"].double().norm().item() - 1)}
    for k, v in got.items():
        print(f"{k}: {v:.2e}", flush=True)
    return got


if __name__ == "__main__":
    main()
