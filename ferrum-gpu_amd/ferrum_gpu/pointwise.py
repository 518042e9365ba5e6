"""ferrum_gpu.pointwise -- elementwise complex kernels on device arrays.

The reference's cmul_interleaved, cmul_split, deinterleave and interleave
(crates/ferrum-gpu-fft-kernels/src/kernels_body.rs:1612-1672).  ``n`` counts
complex elements; arguments are DeviceBuffers, GPU torch tensors or raw device
addresses, and a DeviceBuffer or tensor smaller than what the call reads or
writes (8 bytes per element interleaved, 4 per f32 part) is refused with a
ValueError before anything is launched.  Products are f32 ``re = ar*br - ai*bi``, ``im = ar*bi + ai*br``
without fused multiply-add, as in the reference.  All calls are stream-ordered
and asynchronous.

``dropout`` is for real elements, beside the row operators of ``ferrum_gpu.ssm``
and ``ferrum_gpu.norm``, and takes its arguments as they do.
"""

from __future__ import annotations

import ctypes
import struct

from ferrum_gpu import _native as _n
from ferrum_gpu.fft import _ptr_sized as _p
from ferrum_gpu.hip import Device
from ferrum_gpu.ssm import _BYTES, _DTYPES, _bytes, _check_dtype, _dtype_of, _flat, _stream

__all__ = ["cmul", "cmul_split", "deinterleave", "interleave", "dropout"]

_dropout_pack = struct.Struct("=QQqqdQQQ").pack


def _s(stream: int) -> ctypes.c_void_p:
    return ctypes.c_void_p(stream or None)


def cmul(device: Device, a, b, out, n: int, stream: int = 0) -> None:
    """out[i] = a[i] * b[i] over n interleaved complex64 elements (out may be a or b)."""
    n = int(n)
    _n.check(_n.lib.fg_cmul_c64(device.handle, _p(a, 8 * n, "a"), _p(b, 8 * n, "b"), _p(out, 8 * n, "out"), n,
                                _s(stream)))


def cmul_split(device: Device, a_re, a_im, b_re, b_im, o_re, o_im, n: int, stream: int = 0) -> None:
    """(o_re, o_im)[i] = (a_re, a_im)[i] * (b_re, b_im)[i] over n elements of float32 arrays."""
    n = int(n)
    parts = [_p(x, 4 * n, name) for x, name in
             ((a_re, "a_re"), (a_im, "a_im"), (b_re, "b_re"), (b_im, "b_im"), (o_re, "o_re"), (o_im, "o_im"))]
    _n.check(_n.lib.fg_cmul_split(device.handle, *parts, n, _s(stream)))


def deinterleave(device: Device, src, re, im, n: int, stream: int = 0) -> None:
    """re[i], im[i] = src[i] for n complex64 elements."""
    n = int(n)
    _n.check(_n.lib.fg_deinterleave_c64(device.handle, _p(src, 8 * n, "src"), _p(re, 4 * n, "re"),
                                        _p(im, 4 * n, "im"), n, _s(stream)))


def interleave(device: Device, re, im, out, n: int, stream: int = 0) -> None:
    """out[i] = (re[i], im[i]) for n elements."""
    n = int(n)
    _n.check(_n.lib.fg_interleave_c64(device.handle, _p(re, 4 * n, "re"), _p(im, 4 * n, "im"),
                                      _p(out, 8 * n, "out"), n, _s(stream)))


def dropout(device: Device, x, out, n: int, p: float, seed: int, offset: int = 0, counter=None, dtype=None,
            stream=0) -> None:
    """out[e] = x[e] / (1 - p) where element e is kept, else 0, over n elements
    of float32, bfloat16 or float16 (out may be x).

    An element is kept where 32 bits are at least ``p`` 2^32: half ``e % 2`` (the
    lower one first) of the splitmix64 number ``offset + e // 2`` of ``seed``, the
    generator of ``ferrum_gpu.synthetic``.  No mask is stored: a gradient takes the
    same call with the same p, seed and offset.  A call uses ``(n + 1) // 2``
    numbers; the next one's offset lies behind them.  ``counter``: an int64 on the GPU
    that is added to ``offset``, for calls captured into a graph.  ``dtype``
    comes from a tensor, it is given where x is a DeviceBuffer or an address;
    ``stream`` as for ``ferrum_gpu.ssm``."""
    n, at = int(n), device.ordinal
    dtype = _check_dtype(dtype or (_dtype_of(x) if hasattr(x, "data_ptr") else "bfloat16"))
    for v, what in ((x, "x"), (out, "out")):
        if hasattr(v, "data_ptr") and _dtype_of(v) != dtype:
            raise ValueError(f"{what}: {_dtype_of(v)}, expected {dtype}")
    nbytes = n * _BYTES[dtype]
    args = _dropout_pack(_bytes(x, nbytes, at, "x"), _bytes(out, nbytes, at, "out"), n, _DTYPES[dtype], p,
                         seed & (2**64 - 1), offset & (2**64 - 1), _flat(counter, (1,), "int64", 8, at, "counter"))
    rc = _n.lib.fg_dropout(device.handle, args, _stream(stream, at))
    if rc:
        _n.check(rc)
