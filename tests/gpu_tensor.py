"""Arrays on the GPU that the package takes as it takes torch's: a DeviceBuffer
behind a CPU tensor's type, shape and strides.

torch's own GPU tensors would do, but torch finds no GPU in a process that
loaded the package, and with it the system's HIP runtime, before torch; that is
so where these tests run together with the others.
"""

from __future__ import annotations

import numpy as np
import torch

from ferrum_gpu import _native as N
from ferrum_gpu.hip import DeviceBuffer

_device = None
_kept: list = []  # buffers of the running test: none is freed under a call in flight


def use(device):
    """For a fixture: arrays are on `device` while a test runs."""
    global _device
    _device = device
    torch.manual_seed(0)
    yield
    device.sync()
    _kept.clear()


class Gpu:
    """A CPU tensor's copy on the GPU, with its strides; views share it."""

    def __init__(self, cpu: torch.Tensor, buf=None):
        if buf is None:
            s = cpu.untyped_storage()
            at = cpu.storage_offset(), cpu.shape, cpu.stride()
            cpu = torch.empty(0, dtype=cpu.dtype).set_(s.clone(), *at)
            buf = DeviceBuffer(_device, max(16, s.nbytes()))
            _kept.append(buf)
            self.cpu, self.buf = cpu, buf
            self._push()
        self.cpu, self.buf = cpu, buf

    def _push(self) -> None:
        s = self.cpu.untyped_storage()
        if s.nbytes():
            N.check(N.lib.fg_copy_h2d(_device.handle, self.buf.ptr, s.data_ptr(), s.nbytes()))

    def get(self) -> torch.Tensor:
        """The GPU's values on the CPU, after the work on the default stream."""
        s = self.cpu.untyped_storage()
        if s.nbytes():
            N.check(N.lib.fg_copy_d2h(_device.handle, s.data_ptr(), self.buf.ptr, s.nbytes()))
        return self.cpu.clone()

    def copy_(self, values) -> "Gpu":
        self.get()
        self.cpu.copy_(values.get() if isinstance(values, Gpu) else values)
        self._push()
        return self

    def fill_(self, value) -> "Gpu":
        return self.copy_(torch.full_like(self.cpu, value))

    def normal_(self) -> "Gpu":
        return self.copy_(torch.randn(self.cpu.shape))

    def clone(self) -> "Gpu":
        return Gpu(self.get())

    def _view(self, cpu: torch.Tensor) -> "Gpu":
        assert cpu.untyped_storage().data_ptr() == self.cpu.untyped_storage().data_ptr()
        return Gpu(cpu, self.buf)

    def __getitem__(self, at) -> "Gpu":
        return self._view(self.cpu[at])

    def __setitem__(self, at, values) -> None:
        self[at].copy_(values if isinstance(values, Gpu) else torch.as_tensor(values))

    def view(self, *shape) -> "Gpu":
        return self._view(self.cpu.view(*shape))

    def expand(self, *shape) -> "Gpu":
        return self._view(self.cpu.expand(*shape))

    def __eq__(self, value):
        return self.get() == value

    __hash__ = None
    dtype = property(lambda self: self.cpu.dtype)
    shape = property(lambda self: self.cpu.shape)
    device = property(lambda self: f"cuda:{_device.ordinal}")

    def data_ptr(self) -> int:
        return self.buf.ptr + self.cpu.storage_offset() * self.cpu.element_size()

    def get_device(self) -> int:
        return _device.ordinal

    def stride(self):
        return self.cpu.stride()

    def dim(self):
        return self.cpu.dim()

    def numel(self):
        return self.cpu.numel()

    def element_size(self):
        return self.cpu.element_size()

    def is_contiguous(self):
        return self.cpu.is_contiguous()


class Far:
    """Rows of a [1, length, ...] tensor `row` elements apart, from element `at`
    of a buffer too large for a copy on the host."""

    def __init__(self, buf: DeviceBuffer, cpu: torch.Tensor, row: int, at: int):
        self.buf, self.row, self.at, self.dtype, self.shape = buf, row, at, cpu.dtype, cpu.shape
        for t in range(cpu.shape[1]):
            line = cpu[0, t].contiguous()
            N.check(N.lib.fg_copy_h2d(_device.handle, self._line(t), line.data_ptr(), line.nbytes))

    def _line(self, t: int) -> int:
        return self.buf.ptr + (self.at + t * self.row) * self.dtype.itemsize

    def get(self) -> torch.Tensor:
        out = torch.empty(self.shape, dtype=self.dtype)
        for t in range(self.shape[1]):
            line = out[0, t]
            N.check(N.lib.fg_copy_d2h(_device.handle, line.data_ptr(), self._line(t), line.nbytes))
        return out

    def data_ptr(self) -> int:
        return self._line(0)

    def get_device(self) -> int:
        return _device.ordinal

    def stride(self):
        return (0, self.row, 1) if len(self.shape) == 3 else (0, self.row, self.shape[3], 1)


def up(x) -> Gpu | None:
    return None if x is None else Gpu(x)


def fill(shape, dtype="float32", value=7.0) -> Gpu:
    """An array that a call has to overwrite."""
    return Gpu(torch.full(tuple(shape), value, dtype=getattr(torch, dtype)))


def like(x) -> Gpu:
    """An array of x's type and shape that a call has to overwrite."""
    return Gpu(torch.full(x.shape, 7, dtype=x.dtype))


def room(nbytes: int) -> Gpu:
    return Gpu(torch.zeros(nbytes, dtype=torch.uint8))


def values(x) -> np.ndarray:
    """In 64 bits, of an array on either side."""
    return (x.get() if isinstance(x, (Gpu, Far)) else x).detach().double().numpy()


def same(a, b) -> bool:
    return torch.equal(*(x.get() if isinstance(x, (Gpu, Far)) else x for x in (a, b)))
