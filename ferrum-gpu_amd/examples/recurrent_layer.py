"""A layer of a recurrent language model on its residual stream: dropout, the
stream's addition and norm, a short causal convolution and the gated linear
recurrence; run over a prompt, then token by token with its states in a cache,
and trained.

    python ferrum-gpu_amd/examples/recurrent_layer.py

The layer's projections are torch products, and the package's operators run on
torch's current stream between them.  torch is imported before the package, as it
has to be.
"""

from __future__ import annotations

import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__)))))
import ferrum_gpu  # noqa: E402
from ferrum_gpu import ssm  # noqa: E402
from ferrum_gpu.norm import NormPlan  # noqa: E402


class Layer:
    """y, stream -> stream + dropout(y), normed -> (u, gate) -> conv -> recurrence, times silu(gate) -> out."""

    def __init__(self, device: ferrum_gpu.hip.Device, width=256, channels=384, taps=4, rows=4096, dtype=torch.float32,
                 seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        rand = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
        self.device, self.width, self.channels, self.taps = device, width, channels, taps
        self.dtype, self.name, self.plans = dtype, str(dtype).rpartition(".")[2], {}
        self.norm_weight = 1 + 0.1 * rand(width)
        self.norm = NormPlan(rows, width, device, dtype=self.name)
        self.norm8 = NormPlan(rows, width, device, dtype=self.name, group=128)
        self.into = (rand(width, 2 * channels) / width ** 0.5).to(dtype)
        self.gates = (rand(channels, 2 * channels) / channels ** 0.5).to(dtype)
        self.out = (rand(channels, width) / channels ** 0.5).to(dtype)
        self.taps_weight, self.taps_bias = 0.5 * rand(channels, taps), 0.1 * rand(channels)
        self.decay, self.bias_a, self.bias_x = rand(channels) - 4, 0.1 * rand(channels), 0.1 * rand(channels)

    def _plans(self, batch, length):
        """Both filters' plans for sequences of this shape, made once."""
        if (batch, length) not in self.plans:
            self.plans[batch, length] = (
                ssm.ConvPlan(batch, length, self.channels, self.taps, self.device, dtype=self.name),
                ssm.RecurrencePlan(batch, length, self.channels, self.device, dtype=self.name))
        return self.plans[batch, length]

    def _normed(self, y, stream, drop):
        """The normed rows and the stream behind the addition, of y's shape."""
        x, total = torch.empty_like(y), torch.empty_like(y)
        rows = [t.view(-1, self.width) for t in (y, x, stream, total)]
        self.norm.forward(rows[0], rows[1], weight=self.norm_weight, residual=rows[2], sum_out=rows[3],
                          stream=torch.cuda.current_stream(), **drop)
        return x, total

    def normed_in_8_bits(self, y, stream):
        """What a product in 8 bits takes of the same rows, (rows, width) and its scales."""
        y, stream = y.reshape(-1, self.width), stream.reshape(-1, self.width)
        x = torch.empty(y.shape, dtype=torch.float8_e4m3fn, device="cuda")
        scales = torch.empty(y.shape[0], -(-self.width // 128), device="cuda")
        self.norm8.forward(y, x, weight=self.norm_weight, residual=stream, scales=scales,
                           stream=torch.cuda.current_stream())
        return x, scales

    def prompt(self, y, stream, window=None, state=None, keep=None, drop={}):
        """Outputs and stream of whole sequences; the states are left for what follows.  keep: a dict for backward()."""
        x, total = self._normed(y, stream, drop)
        p = x @ self.into
        u, gate = p[..., :self.channels], p[..., self.channels:]
        conv, rec = self._plans(*y.shape[:2])
        here, c, h = torch.cuda.current_stream(), torch.empty_like(u), torch.empty_like(u)
        conv.forward(u, self.taps_weight, c, bias=self.taps_bias, initial=window, final=window, stream=here)
        q = c @ self.gates
        a, i = q[..., :self.channels], q[..., self.channels:]
        check = None if keep is None else torch.empty(rec.checkpoint_bytes, dtype=torch.uint8, device="cuda")
        rec.forward(c, a, i, self.decay, h, bias_a=self.bias_a, bias_x=self.bias_x, initial=state, final=state,
                    checkpoints=check, stream=here)
        if keep is not None:
            keep.update(total=total, x=x, u=u, gate=gate, c=c, a=a, i=i, h=h, check=check, drop=drop)
        return (h * torch.nn.functional.silu(gate)) @ self.out, total

    def token(self, y, stream, window, state, slots):
        """Outputs and stream of one token of each row, whose states lie in cache slots."""
        x, total = self._normed(y, stream, {})
        p = x @ self.into
        u, gate = p[:, :self.channels], p[:, self.channels:]
        here, c, h = torch.cuda.current_stream(), torch.empty_like(u), torch.empty_like(u)
        ssm.conv_step(self.device, u, self.taps_weight, window, c, bias=self.taps_bias, slots=slots, stream=here)
        q = c @ self.gates
        ssm.recurrence_step(self.device, c, q[:, :self.channels], q[:, self.channels:], self.decay, state, h,
                            bias_a=self.bias_a, bias_x=self.bias_x, slots=slots, stream=here)
        return (h * torch.nn.functional.silu(gate)) @ self.out, total

    def backward(self, k, grad, grad_total):
        """Gradients of y, of the stream and of the parameters of the package's operators."""
        here, g = torch.cuda.current_stream(), {}
        conv, rec = self._plans(*k["u"].shape[:2])
        dm = grad @ self.out.t().contiguous()
        s = torch.sigmoid(k["gate"])
        dgate = dm * k["h"] * s * (1 + k["gate"] * (1 - s))
        dh = dm * k["gate"] * s
        c, a, i = (torch.empty_like(k["c"]) for _ in range(3))
        for n in ("decay", "bias_a", "bias_x"):
            g[n] = torch.empty_like(self.decay)
        rec.backward(k["c"], k["a"], k["i"], self.decay, dh, k["check"], grad_x=c, grad_gate_a=a, grad_gate_x=i,
                     bias_a=self.bias_a, bias_x=self.bias_x, grad_decay=g["decay"], grad_bias_a=g["bias_a"],
                     grad_bias_x=g["bias_x"], stream=here)
        c += torch.cat([a, i], -1) @ self.gates.t().contiguous()
        u, g["taps"] = torch.empty_like(k["c"]), torch.empty_like(self.taps_weight)
        conv.backward(k["u"], self.taps_weight, c, grad_x=u, grad_weight=g["taps"], bias=self.taps_bias, stream=here)
        dx = (torch.cat([u, dgate], -1) @ self.into.t().contiguous()).view(-1, self.width)
        g["y"], g["stream"], g["norm"] = torch.empty_like(grad), torch.empty_like(grad), torch.empty_like(self.norm_weight)
        self.norm.backward(k["total"].view(-1, self.width), dx, weight=self.norm_weight,
                           grad_sum=grad_total.view(-1, self.width), grad_x=g["y"].view(-1, self.width),
                           grad_residual=g["stream"].view(-1, self.width), grad_weight=g["norm"], stream=here,
                           **k["drop"])
        return g


def main(device=None) -> dict:
    """Runs the layer all three ways and returns how far they are apart."""
    device = device or ferrum_gpu.hip.Device(0)
    torch.manual_seed(0)
    layer = Layer(device)
    batch, length, more, rows = 3, 50, 8, 5
    y, stream = (torch.randn(batch, length + more, layer.width, device="cuda") for _ in range(2))
    states = lambda n: (torch.zeros(n, layer.taps - 1, layer.channels, device="cuda"),  # noqa: E731
                        torch.zeros(n, layer.channels, device="cuda"))
    whole, total = layer.prompt(y, stream, *states(batch))
    # the prompt's states go to slots of a larger cache, where the tokens find them
    window, state = states(batch)
    layer.prompt(y[:, :length].contiguous(), stream[:, :length].contiguous(), window, state)
    slots = torch.tensor([4, 0, 2], dtype=torch.int32, device="cuda")
    windows, cache = states(rows)
    windows[slots.long()], cache[slots.long()] = window, state
    apart = 0.0
    for t in range(length, length + more):
        out, _ = layer.token(y[:, t].contiguous(), stream[:, t].contiguous(), windows, cache, slots)
        apart = max(apart, ((out - whole[:, t]).abs().max() / whole.abs().max()).item())
    x8, scales = layer.normed_in_8_bits(y, stream)
    x, _ = layer._normed(y, stream, {})
    x8 = x8.float() * scales.repeat_interleave(128, 1)[:, :layer.width]
    eight = ((x8 - x.view_as(x8)).norm() / x.norm()).item()
    # a step along the gradient's direction, with dropout, changes the loss by its length
    drop = {"dropout": 0.2, "seed": 7, "offset": 1000}
    grad, grad_total, keep = torch.randn_like(y), torch.randn_like(y), {}
    layer.prompt(y, stream, keep=keep, drop=drop)
    g = layer.backward(keep, grad, grad_total)
    loss = lambda o: ((o[0].double() * grad).sum() + (o[1].double() * grad_total).sum()).item()  # noqa: E731
    got = {"tokens against the whole": apart, "8 bits against the rows' type": eight}
    for name, inputs in (("y", lambda s: (y + s, stream)), ("stream", lambda s: (y, stream + s))):
        step = 1e-2 * g[name] / g[name].norm()
        slope = (loss(layer.prompt(*inputs(step), drop=drop)) - loss(layer.prompt(*inputs(-step), drop=drop))) / 2e-2
        got[f"slope against the gradient of {name}"] = abs(slope / g[name].double().norm().item() - 1)
    for k, v in got.items():
        print(f"{k}: {v:.2e}", flush=True)
    return got


if __name__ == "__main__":
    main()
