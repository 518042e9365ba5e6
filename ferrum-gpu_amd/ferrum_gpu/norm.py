"""ferrum_gpu.norm -- the root-mean-square norm of a residual stream, with what
stands before it and an output in 8 bits for products that take one.

It stands between the blocks of ``ferrum_gpu.ssm``'s filters and takes arrays of
rows, types and streams as they do: GPU torch tensors of shape ``(rows, width)``
with any stride between rows, DeviceBuffers and raw addresses as contiguous.
Import torch before this package.
"""

from __future__ import annotations

import ctypes
import struct

from ferrum_gpu import _native as _n
from ferrum_gpu.hip import Device
from ferrum_gpu.ssm import _DTYPES, _Plan, _address, _check_dtype, _dtype_of, _flat, _rows, _stream, _torch_types

__all__ = ["NormPlan"]

_shape_pack = struct.Struct("=4qd").pack
_forward_pack = struct.Struct("=q" + "Qqq" * 4 + "QQdQQQ").pack
_backward_pack = struct.Struct("=q" + "Qqq" * 5 + "QQdQQQ").pack
_MASK = 2**64 - 1


class NormPlan(_Plan):
    """Norm of up to ``rows`` rows of ``width`` elements::

        v = dropout(x) + residual
        out = v / sqrt(mean(v^2) + eps) * weight

    ``group``: of an output in 8 bits, how many elements of a row share a scale:
    32, 64 or 128, or 0, a scale for each row.

    Calls take as many rows as ``x`` has, or ``rows`` where it is no tensor (None:
    the plan's).  Dropout's bits are those of ``ferrum_gpu.pointwise.dropout``, of
    element ``row * width + column``; ``dropout`` is its probability, and the
    backward pass takes the same ``dropout``, ``seed``, ``offset`` and ``counter``.
    """

    _destroy, _get_info = _n.lib.fg_norm_plan_destroy, _n.lib.fg_norm_plan_get_info
    _info = ("row_threads", "workspace_bytes")

    def __init__(self, rows: int, width: int, device: Device, dtype="bfloat16", eps: float = 1e-6, group: int = 0):
        self.device, self.rows, self.width = device, int(rows), int(width)
        self.dtype, self.eps, self.group = _check_dtype(dtype), float(eps), int(group)
        self._at, self._p = device.ordinal, ctypes.c_void_p()
        shape = _shape_pack(self.rows, self.width, _DTYPES[self.dtype], self.group, self.eps)
        _n.check(_n.lib.fg_norm_plan_create(device.handle, shape, ctypes.byref(self._p)))
        self._groups = -(-self.width // self.group) if self.group else 1

    def _of(self, x, n: int, what: str) -> tuple:
        if x is None:
            return 0, 0, 0
        try:  # what a tensor passes in most calls, which may be bound by the host
            if x.shape == (n, self.width) and x.dtype is _torch_types[self.dtype] and x.get_device() == self._at:
                if x.is_contiguous():
                    return x.data_ptr(), 0, self.width
                row, element = x.stride()
                if element == 1:
                    return x.data_ptr(), 0, row
        except (AttributeError, KeyError):  # no tensor, or the first one
            pass
        return _rows(x, (n,), self.width, (), self.dtype, self.device.ordinal, what)

    def _out8(self, x, n: int) -> tuple:
        """Rows of e4m3: float8_e4m3fn or uint8."""
        if hasattr(x, "data_ptr"):
            if _dtype_of(x) not in ("float8_e4m3fn", "uint8"):
                raise ValueError(f"out: {_dtype_of(x)}, expected float8_e4m3fn or uint8 where there are scales")
            if x.shape != (n, self.width):
                raise ValueError(f"out: shape {tuple(x.shape)}, expected {(n, self.width)}")
            if x.get_device() != self.device.ordinal:
                raise ValueError(f"out: tensor on {x.device}, the call runs on GPU {self.device.ordinal}")
            row, element = x.stride()
            if element != 1 and self.width > 1:
                raise ValueError(f"out: the elements of a row must be adjacent (strides {tuple(x.stride())})")
            return x.data_ptr(), 0, row
        return _address(x, n * self.width, "out"), 0, self.width

    def _count(self, x, rows) -> int:
        if rows is not None:
            return int(rows)
        try:
            return x.shape[0]
        except (AttributeError, IndexError):  # no tensor, or one that the checks refuse
            return self.rows

    def _weight(self, x, what: str) -> int:
        return _flat(x, (self.width,), "float32", 4 * self.width, self.device.ordinal, what)

    def _counter(self, x) -> int:
        return _flat(x, (1,), "int64", 8, self.device.ordinal, "counter")

    def forward(self, x, out, weight=None, residual=None, sum_out=None, scales=None, dropout: float = 0.0,
                seed: int = 0, offset: int = 0, counter=None, rows=None, stream=0) -> None:
        """``weight`` (width) float32 (None: ones).  ``sum_out``: room for v in the
        rows' type, which backward() takes; may be ``residual``, and ``out`` may be
        ``x``.  With ``scales``, (rows, groups) float32, ``out`` is float8_e4m3fn
        (or uint8): the normed row over its scale, max |out| / 448 of a group; NaN,
        like all scales of a row, where the row's sum of squares is not finite."""
        n, at = self._count(x, rows), self.device.ordinal
        args = _forward_pack(n, *self._of(x, n, "x"), *self._of(residual, n, "residual"),
                             *(self._of(out, n, "out") if scales is None else self._out8(out, n)),
                             *self._of(sum_out, n, "sum_out"), self._weight(weight, "weight"),
                             _flat(scales, (n, self._groups), "float32", 4 * n * self._groups, at, "scales"), dropout,
                             seed & _MASK, offset & _MASK, self._counter(counter))
        rc = _n.lib.fg_norm_forward(self._handle(), args, _stream(stream, at))
        if rc:
            _n.check(rc)

    def backward(self, sum_in, grad_out, weight=None, grad_sum=None, grad_x=None, grad_residual=None,
                 grad_weight=None, dropout: float = 0.0, seed: int = 0, offset: int = 0, counter=None, rows=None,
                 stream=0) -> None:
        """Gradients from ``grad_out``, that of ``out``, and ``grad_sum``, that of
        ``sum_out`` (None: zeros), given the ``sum_in`` that forward() stored (x
        itself where it had neither dropout nor a residual); each is written where
        room for it is given.  ``grad_residual`` may be ``grad_sum`` and ``grad_x``
        may be ``grad_out``."""
        n = self._count(sum_in, rows)
        args = _backward_pack(n, *self._of(sum_in, n, "sum_in"), *self._of(grad_out, n, "grad_out"),
                              *self._of(grad_sum, n, "grad_sum"), *self._of(grad_x, n, "grad_x"),
                              *self._of(grad_residual, n, "grad_residual"), self._weight(weight, "weight"),
                              self._weight(grad_weight, "grad_weight"), dropout, seed & _MASK, offset & _MASK,
                              self._counter(counter))
        rc = _n.lib.fg_norm_backward(self._handle(), args, _stream(stream, self.device.ordinal))
        if rc:
            _n.check(rc)
