"""ferrum_gpu.ssm -- sequence filters: the short causal convolution and the
selective state space scan.

They stand beside the FFT's filters (``fft`` -> ``pointwise.cmul`` -> inverse),
which cover long filters that stay the same over time: the convolution is for
a few taps per channel, the scan for filters whose coefficients change from
token to token.  With a constant time step, B and C the scan is the
convolution with ``k[t, d] = sum_n C[n] exp(t dt A[d, n]) dt B[n]``, which the
FFT computes too.

=====================  =====================================================
``ConvPlan``           causal convolution of whole sequences, and its gradients
``conv_step``          one token of each row, windows in a cache of slots
``ScanPlan``           selective scan of whole sequences, and its gradients
``scan_step``          one token of each row, states in a cache of slots
=====================  =====================================================

Arrays of rows (one row of ``channels``, for B and C ``groups * states``
elements a token) are GPU torch tensors of shape ``(batch, length, n)``, packed
``(tokens, n)``, and for a step ``(batch, n)``, of the plan's ``dtype``, with
any strides but 1 between the elements of a row: slices of a projection's
output need no copy.  DeviceBuffers and raw device addresses are taken as
contiguous.  Everything else is contiguous: parameters and their gradients,
scan states (float32), convolution states (``dtype``), ``offsets`` and
``slots`` (int32).  A tensor of another shape, type or device and a DeviceBuffer
that is too small raise ValueError before anything is launched; a raw address
cannot be checked.

Packed sequences lie one after another in ``tokens`` rows: rows ``offsets[s]``
up to ``offsets[s + 1]`` are sequence ``s``, at most ``length`` of them;
``offsets`` holds ``batch + 1`` int32 on the GPU that do not fall (outputs are
undefined where they do); values beyond the rows are taken as the nearest.  Rows
outside every sequence are not written.

Arithmetic is float32 whatever the type of the rows.  Results do not depend on
timing: sums over channels and tokens are added in a fixed order.

All calls are stream-ordered and asynchronous.  ``stream`` takes a
``torch.cuda.Stream``, and with torch tensors it should: ``stream=
torch.cuda.current_stream()`` runs the call behind the torch operations that made
its tensors and ahead of those that take its outputs or get their memory.  The
default, ``stream=0``, is the device's own default stream, which waits for none
of torch's and none of them for it: there the caller synchronizes both, or
passes arrays that nothing else is working on.  Stream handles are taken too.  A
plan's workspaces serve one call at a time; its first ``backward`` allocates, so
it cannot be captured into a graph, later calls can.

Import torch before this package: torch finds no GPU in a process that loaded
the package, and with it the system's HIP runtime, first.
"""

from __future__ import annotations

import ctypes
import struct

from ferrum_gpu import _native as _n
from ferrum_gpu.hip import Device, DeviceBuffer, _release

__all__ = ["ConvPlan", "ScanPlan", "conv_step", "scan_step", "MAX_STATES", "MAX_WIDTH"]

MAX_STATES, MAX_WIDTH = 64, 8

_DTYPES = {"float32": 0, "bfloat16": 1, "float16": 2}
_BYTES = {"float32": 4, "bfloat16": 2, "float16": 2}
_ACTIVATIONS = {"silu": 1, None: 0}
_torch_types: dict = {}  # name -> torch dtype, filled when the first tensor comes
_type_names: dict = {}  # the other way round


def _torch_type(dtype: str):
    t = _torch_types.get(dtype)
    if t is None:
        import torch  # a tensor has come, so it is there

        for name in (*_DTYPES, "int32"):
            _torch_types[name] = getattr(torch, name)
            _type_names[_torch_types[name]] = name
        t = _torch_types[dtype]
    return t


def _dtype_of(x) -> str:
    d = x.dtype
    return _type_names.get(d) or str(d).rpartition(".")[2]


def _check_dtype(dtype) -> str:
    if dtype in _DTYPES:
        return dtype
    name = dtype if isinstance(dtype, str) else str(dtype).rpartition(".")[2]
    if name not in _DTYPES:
        raise ValueError(f"dtype must be one of {list(_DTYPES)}, got {dtype}")
    return name


def _check_activation(activation) -> int:
    if activation not in _ACTIVATIONS:
        raise ValueError(f"activation must be 'silu' or None, got {activation!r}")
    return _ACTIVATIONS[activation]


def _address(x, nbytes: int, what: str) -> int:
    """The address of a DeviceBuffer of at least nbytes, or of a raw pointer."""
    if isinstance(x, DeviceBuffer):
        if x.nbytes < nbytes:
            raise ValueError(f"{what}: buffer of {x.nbytes} bytes, the call reads or writes {nbytes}")
        return x.ptr
    return int(x)


_NULL_STREAM = 1  # FG_STREAM_NULL: torch's default stream, whose handle is 0


def _stream(stream, ordinal: int):
    """What the library takes as its stream: a handle, or None for the device's default stream."""
    if stream.__class__ is int or stream is None:
        return stream or None
    handle = getattr(stream, "cuda_stream", None)
    if handle is None:
        return int(stream) or None
    if stream.device_index != ordinal:
        raise ValueError(f"stream: of GPU {stream.device_index}, the call runs on GPU {ordinal}")
    return handle or _NULL_STREAM


def _wrong(x, what: str, shapes, dtype, ordinal: int):
    """Why a tensor is refused; called when one of the checks has failed."""
    if shapes is not None and x.shape not in shapes:
        return ValueError(f"{what}: shape {tuple(x.shape)}, expected {shapes[0]}")
    if dtype is not None and _dtype_of(x) != dtype:
        return ValueError(f"{what}: {_dtype_of(x)}, expected {dtype}")
    if x.get_device() != ordinal:
        hint = "; torch finds no GPU where this package was imported first" if x.get_device() < 0 else ""
        return ValueError(f"{what}: tensor on {x.device}, the call runs on GPU {ordinal}{hint}")
    return None


def _flat(x, shape: tuple, dtype: str, nbytes: int, ordinal: int, what: str) -> int:
    """The address of a contiguous array, 0 for None."""
    if x is None:
        return 0
    # What a tensor passes in most calls; a one-token call is bound by the host.
    try:
        if x.shape == shape and x.dtype is _torch_types[dtype] and x.get_device() == ordinal and x.is_contiguous():
            return x.data_ptr()
    except (AttributeError, KeyError):  # no tensor, or the first one
        pass
    if hasattr(x, "data_ptr"):
        if x.shape != shape or x.dtype is not _torch_type(dtype) or x.get_device() != ordinal:
            raise _wrong(x, what, (shape,), dtype, ordinal)
        if not x.is_contiguous():
            raise ValueError(f"{what}: tensor is not contiguous")
        return x.data_ptr()
    return _address(x, nbytes, what)


def _bytes(x, nbytes: int, ordinal: int, what: str) -> int:
    """The address of at least nbytes, 0 for None."""
    if x is None:
        return 0
    if hasattr(x, "data_ptr"):
        if x.numel() * x.element_size() < nbytes or not x.is_contiguous():
            raise ValueError(f"{what}: tensor of {x.numel() * x.element_size()} bytes (contiguous: "
                             f"{x.is_contiguous()}), the call reads or writes {nbytes} contiguous bytes")
        if x.get_device() != ordinal:
            raise _wrong(x, what, None, None, ordinal)
        return x.data_ptr()
    return _address(x, nbytes, what)


def _rows(x, lead: tuple, width: int, inner: tuple, dtype: str, ordinal: int, what: str) -> tuple:
    """(address, sequence stride, row stride) of an array of rows of ``width``
    elements, or of shape ``inner`` (B and C: groups, states)."""
    if x is None:
        return 0, 0, 0
    n = len(lead)
    if hasattr(x, "data_ptr"):
        st = x.stride()
        if x.dtype is not _torch_type(dtype) or x.get_device() != ordinal:
            fine = None
        elif x.shape == (*lead, width):
            fine = st[n] == 1 or width == 1
        elif inner and x.shape == lead + inner:
            fine = (inner[1] == 1 or st[n + 1] == 1) and (inner[0] == 1 or st[n] == inner[1])
        else:
            fine = None
        if fine is None:
            raise _wrong(x, what, (lead + (width,), lead + inner) if inner else (lead + (width,),), dtype, ordinal)
        if not fine:
            raise ValueError(f"{what}: the elements of a row must be adjacent (strides {tuple(st)})")
        return (x.data_ptr(), st[0], st[1]) if n == 2 else (x.data_ptr(), 0, st[0])
    rows = lead[0] * lead[1] if n == 2 else lead[0]
    p = _address(x, rows * width * _BYTES[dtype], what)
    return (p, lead[1] * width, width) if n == 2 else (p, 0, width)


_conv_forward_pack = struct.Struct("=QqqQqqQQQQQ").pack
_conv_backward_pack = struct.Struct("=" + "Qqq" * 3 + "Q" * 8).pack
_conv_step_pack = struct.Struct("=6q" + "Qqq" * 2 + "Q" * 5).pack
_scan_forward_pack = struct.Struct("=" + "Qqq" * 5 + "Q" * 5 + "Qqq" + "QQ").pack
_scan_backward_pack = struct.Struct("=" + "Qqq" * 5 + "Q" * 5 + "Qqq" + "QQ" + "Qqq" * 5 + "Q" * 4).pack
_scan_step_pack = struct.Struct("=7q" + "Qqq" * 6 + "Q" * 6).pack
_shape_pack = struct.Struct("=8q").pack
_scan_shape_pack = struct.Struct("=9q").pack


class _Plan:
    _destroy = None

    def _setup(self, batch, length, tokens, channels, device: Device, dtype) -> None:
        self.device = device
        self.batch, self.length, self.channels = int(batch), int(length), int(channels)
        self.dtype = _check_dtype(dtype)
        self.packed = tokens is not None
        self.tokens = int(tokens) if self.packed else self.batch * self.length
        self._lead = (self.tokens,) if self.packed else (self.batch, self.length)
        self._p = ctypes.c_void_p()

    def _row(self, x, what: str) -> tuple:
        return _rows(x, self._lead, self.channels, (), self.dtype, self.device.ordinal, what)

    def _param(self, x, shape: tuple, what: str) -> int:
        n = 4
        for k in shape:
            n *= k
        return _flat(x, shape, "float32", n, self.device.ordinal, what)

    def _offsets(self, x) -> int:
        if (x is not None) != self.packed:
            raise ValueError("offsets: packed sequences need them" if self.packed
                             else "offsets: only packed sequences (a plan with tokens=) have them")
        return _flat(x, (self.batch + 1,), "int32", 4 * (self.batch + 1), self.device.ordinal, "offsets")

    def _handle(self):
        if not self._p.value:
            raise ValueError("plan is destroyed")
        return self._p

    def describe(self) -> dict:
        """How the calls run, and the GPU memory that the plan holds (the
        backward pass's from its first call on)."""
        out = (ctypes.c_int64 * len(self._info))()
        _n.check(self._get_info(self._handle(), out))
        return dict(zip(self._info, out))

    def destroy(self) -> None:
        """Free the plan and its workspaces; no call of it may be in flight."""
        if getattr(self, "_p", None) is not None and self._p.value:
            _n.check(type(self)._destroy(self._p))
            self._p = ctypes.c_void_p()

    def __del__(self):  # pragma: no cover
        try:
            if getattr(self, "_p", None) is not None and self._p.value:
                # the device rides along; released after any Capture block open on this thread
                _release(lambda destroy, p, dev: destroy(p), type(self)._destroy, self._p, self.device)
                self._p = ctypes.c_void_p()
        except Exception:
            pass


class ConvPlan(_Plan):
    """Causal convolution of ``batch`` sequences, ``width`` taps (2 to 8) for
    each of ``channels`` channels::

        out[t, d] = act(bias[d] + sum_k weight[d, k] x[t - (width - 1) + k, d])

    ``activation`` is "silu" or None.  With ``tokens`` the sequences are packed
    and ``length`` is the longest one's.
    """

    _destroy, _get_info = _n.lib.fg_conv_plan_destroy, _n.lib.fg_conv_plan_get_info
    _info = ("forward_tokens", "backward_tokens", "workspace_bytes")

    def __init__(self, batch: int, length: int, channels: int, width: int, device: Device, dtype="bfloat16",
                 activation: str | None = "silu", tokens: int | None = None):
        self._setup(batch, length, tokens, channels, device, dtype)
        self.width = int(width)
        shape = _shape_pack(self.batch, self.length, self.tokens, self.channels, self.width, _DTYPES[self.dtype],
                            self.packed, _check_activation(activation))
        _n.check(_n.lib.fg_conv_plan_create(device.handle, shape, ctypes.byref(self._p)))
        self._state_shape = (self.batch, self.width - 1, self.channels)
        self._state_bytes = self.batch * (self.width - 1) * self.channels * _BYTES[self.dtype]

    def _state(self, x, what: str) -> int:
        return _flat(x, self._state_shape, self.dtype, self._state_bytes, self.device.ordinal, what)

    def forward(self, x, weight, out, bias=None, initial=None, final=None, offsets=None, stream=0) -> None:
        """``weight`` (channels, width) and ``bias`` (channels) float32.
        ``initial``: the (batch, width - 1, channels) rows before each sequence
        (None: zeros); ``final``: room for the last width - 1 rows of (initial,
        x), may be ``initial``."""
        args = _conv_forward_pack(*self._row(x, "x"), *self._row(out, "out"),
                                  self._param(weight, (self.channels, self.width), "weight"),
                                  self._param(bias, (self.channels,), "bias"), self._state(initial, "initial"),
                                  self._state(final, "final"), self._offsets(offsets))
        rc = _n.lib.fg_conv_forward(self._handle(), args, _stream(stream, self.device.ordinal))
        if rc:
            _n.check(rc)

    def backward(self, x, weight, grad_out, grad_x=None, grad_weight=None, grad_bias=None, bias=None, initial=None,
                 grad_initial=None, grad_final=None, offsets=None, stream=0) -> None:
        """Gradients from ``grad_out``, that of ``out``, and ``grad_final``,
        that of ``final`` (None: zeros), given forward's inputs; each is
        written where room for it is given."""
        args = _conv_backward_pack(*self._row(x, "x"), *self._row(grad_out, "grad_out"),
                                   *self._row(grad_x, "grad_x"),
                                   self._param(weight, (self.channels, self.width), "weight"),
                                   self._param(bias, (self.channels,), "bias"), self._state(initial, "initial"),
                                   self._state(grad_final, "grad_final"),
                                   self._param(grad_weight, (self.channels, self.width), "grad_weight"),
                                   self._param(grad_bias, (self.channels,), "grad_bias"),
                                   self._state(grad_initial, "grad_initial"), self._offsets(offsets))
        rc = _n.lib.fg_conv_backward(self._handle(), args, _stream(stream, self.device.ordinal))
        if rc:
            _n.check(rc)


class ScanPlan(_Plan):
    """Selective scan of ``batch`` sequences, ``states`` states (1 to 64) for
    each of ``channels`` channels, which share B and C in ``groups`` groups of
    neighbours::

        dt = softplus(delta + delta_bias)           (softplus=False: without it)
        h_t[d, n] = exp(dt A[d, n]) h_{t-1}[d, n] + dt u B_t[g, n]
        out = (sum_n C_t[g, n] h_t[d, n] + D[d] u) * (z sigmoid(z))

    With ``tokens`` the sequences are packed and ``length`` is the longest
    one's.
    """

    _destroy, _get_info = _n.lib.fg_scan_plan_destroy, _n.lib.fg_scan_plan_get_info
    _info = ("forward_parts", "forward_tokens", "backward_parts", "backward_tokens", "workspace_bytes")

    def __init__(self, batch: int, length: int, channels: int, states: int, device: Device, groups: int = 1,
                 dtype="bfloat16", softplus: bool = True, tokens: int | None = None):
        self._setup(batch, length, tokens, channels, device, dtype)
        self.states, self.groups = int(states), int(groups)
        shape = _scan_shape_pack(self.batch, self.length, self.tokens, self.channels, self.states, self.groups,
                                 _DTYPES[self.dtype], self.packed, bool(softplus))
        _n.check(_n.lib.fg_scan_plan_create(device.handle, shape, ctypes.byref(self._p)))
        n = ctypes.c_size_t()
        _n.check(_n.lib.fg_scan_checkpoint_bytes(self._p, ctypes.byref(n)))
        #: Bytes of the ``checkpoints`` that a backward pass takes.
        self.checkpoint_bytes = n.value

    def _bc(self, x, what: str) -> tuple:
        return _rows(x, self._lead, self.groups * self.states, (self.groups, self.states), self.dtype,
                     self.device.ordinal, what)

    def _state(self, x, what: str) -> int:
        return self._param(x, (self.batch, self.channels, self.states), what)

    def _inputs(self, u, delta, A, B, C, D, z, delta_bias, initial, offsets) -> tuple:
        d = (self.channels,)
        return (*self._row(u, "u"), *self._row(delta, "delta"), *self._bc(B, "B"), *self._bc(C, "C"),
                *self._row(z, "z"), self._param(A, (self.channels, self.states), "A"), self._param(D, d, "D"),
                self._param(delta_bias, d, "delta_bias"), self._state(initial, "initial"), self._offsets(offsets))

    def forward(self, u, delta, A, B, C, out, D=None, z=None, delta_bias=None, initial=None, final=None, offsets=None,
                checkpoints=None, stream=0) -> None:
        """``A`` (channels, states), ``D`` and ``delta_bias`` (channels)
        float32; without ``z`` no gate.  ``initial``: the (batch, channels,
        states) states before each sequence (None: zeros); ``final``: room for
        those after its last token, may be ``initial``.  ``checkpoints``:
        ``checkpoint_bytes`` of room, where backward() follows."""
        args = _scan_forward_pack(*self._inputs(u, delta, A, B, C, D, z, delta_bias, initial, offsets),
                                  *self._row(out, "out"), self._state(final, "final"),
                                  _bytes(checkpoints, self.checkpoint_bytes, self.device.ordinal, "checkpoints"))
        rc = _n.lib.fg_scan_forward(self._handle(), args, _stream(stream, self.device.ordinal))
        if rc:
            _n.check(rc)

    def backward(self, u, delta, A, B, C, grad_out, checkpoints, grad_u=None, grad_delta=None, grad_A=None,
                 grad_B=None, grad_C=None, D=None, z=None, delta_bias=None, grad_D=None, grad_z=None,
                 grad_delta_bias=None, grad_initial=None, grad_final=None, offsets=None, stream=0) -> None:
        """Gradients from ``grad_out``, that of ``out``, and ``grad_final``,
        that of ``final`` (None: zeros), given forward's inputs and the
        ``checkpoints`` it left; each is written where room for it is given."""
        d = (self.channels,)
        args = _scan_backward_pack(*self._inputs(u, delta, A, B, C, D, z, delta_bias, None, offsets),
                                   *self._row(grad_out, "grad_out"),
                                   _bytes(checkpoints, self.checkpoint_bytes, self.device.ordinal, "checkpoints"),
                                   self._state(grad_final, "grad_final"), *self._row(grad_u, "grad_u"),
                                   *self._row(grad_delta, "grad_delta"), *self._bc(grad_B, "grad_B"),
                                   *self._bc(grad_C, "grad_C"), *self._row(grad_z, "grad_z"),
                                   self._param(grad_A, (self.channels, self.states), "grad_A"),
                                   self._param(grad_D, d, "grad_D"),
                                   self._param(grad_delta_bias, d, "grad_delta_bias"),
                                   self._state(grad_initial, "grad_initial"))
        rc = _n.lib.fg_scan_backward(self._handle(), args, _stream(stream, self.device.ordinal))
        if rc:
            _n.check(rc)


def _shape(x) -> tuple:
    return x.shape if hasattr(x, "data_ptr") else ()


def _size(given, shape: tuple, axis: int, what: str) -> int:
    """A size: what the caller gave, else the tensor's."""
    if given is not None:
        return int(given)
    if len(shape) > axis:
        return shape[axis]
    raise ValueError(f"{what} is needed where the array is not a tensor that has it")


def _step_row(x, shape: tuple, inner: tuple, dtype: str, ordinal: int, what: str) -> tuple:
    """_rows() of one token of each row: ``shape`` is (batch, width)."""
    if x is None:
        return 0, 0, 0
    try:  # as in _flat()
        if x.shape == shape and x.dtype is _torch_types[dtype] and x.get_device() == ordinal:
            row, element = x.stride()
            if element == 1:
                return x.data_ptr(), row, 0
    except (AttributeError, KeyError):
        pass
    p, _, row = _rows(x, shape[:1], shape[1], inner, dtype, ordinal, what)
    return p, row, 0


def conv_step(device: Device, x, weight, state, out, bias=None, slots=None, state_out=None, activation="silu",
              batch=None, channels=None, width=None, state_rows=None, dtype=None, stream=0) -> None:
    """ConvPlan's convolution of one token of each of ``batch`` rows.

    ``state``: the (state_rows, width - 1, channels) windows before the token;
    row i takes and moves on window ``slots[i]`` (int32; None: i).  A row whose
    slot is negative or beyond the windows gets zeros and leaves them alone; no
    two rows may share a slot.  ``state_out``: where the moved windows go
    (None: ``state`` itself).  Sizes and ``dtype`` come from tensors; they are
    given where the arrays are DeviceBuffers or addresses."""
    lead = _shape(x)
    batch, channels = _size(batch, lead, 0, "batch"), _size(channels, lead, 1, "channels")
    width = _size(width, _shape(weight), 1, "width")
    state_rows = _size(state_rows, _shape(state), 0, "state_rows")
    dtype = _check_dtype(dtype or (_dtype_of(x) if hasattr(x, "data_ptr") else "bfloat16"))
    at = device.ordinal
    row = (batch, channels)
    shape = (state_rows, width - 1, channels)
    nbytes = state_rows * (width - 1) * channels * _BYTES[dtype]
    s = _flat(state, shape, dtype, nbytes, at, "state")
    args = _conv_step_pack(batch, channels, width, _DTYPES[dtype], _check_activation(activation), state_rows,
                           *_step_row(x, row, (), dtype, at, "x"),
                           *_step_row(out, row, (), dtype, at, "out"),
                           _flat(weight, (channels, width), "float32", 4 * channels * width, at, "weight"),
                           _flat(bias, (channels,), "float32", 4 * channels, at, "bias"), s,
                           s if state_out is None else _flat(state_out, shape, dtype, nbytes, at, "state_out"),
                           _flat(slots, (batch,), "int32", 4 * batch, at, "slots"))
    rc = _n.lib.fg_conv_step(device.handle, args, _stream(stream, at))
    if rc:
        _n.check(rc)


def scan_step(device: Device, u, delta, A, B, C, state, out, D=None, z=None, delta_bias=None, slots=None,
              state_out=None, softplus: bool = True, groups: int | None = None, batch=None, channels=None,
              states=None, state_rows=None, dtype=None, stream=0) -> None:
    """ScanPlan's scan of one token of each of ``batch`` rows.

    ``state``: (state_rows, channels, states) float32; ``slots`` and
    ``state_out`` as for conv_step().  Sizes and ``dtype`` come from tensors
    (``groups`` from B's); they are given where the arrays are DeviceBuffers or
    addresses."""
    lead = _shape(u)
    batch, channels = _size(batch, lead, 0, "batch"), _size(channels, lead, 1, "channels")
    states = _size(states, _shape(A), 1, "states")
    state_rows = _size(state_rows, _shape(state), 0, "state_rows")
    dtype = _check_dtype(dtype or (_dtype_of(u) if hasattr(u, "data_ptr") else "bfloat16"))
    if groups is None:
        groups = 1 if not hasattr(B, "data_ptr") or states < 1 else B.shape[1] if B.dim() == 3 \
            else B.shape[-1] // states
    at = device.ordinal
    row, bc, inner = (batch, channels), (batch, groups * states), (groups, states)
    shape = (state_rows, channels, states)
    nbytes = 4 * state_rows * channels * states
    s = _flat(state, shape, "float32", nbytes, at, "state")
    args = _scan_step_pack(batch, channels, states, groups, _DTYPES[dtype], bool(softplus), state_rows,
                           *_step_row(u, row, (), dtype, at, "u"),
                           *_step_row(delta, row, (), dtype, at, "delta"),
                           *_step_row(B, bc, inner, dtype, at, "B"),
                           *_step_row(C, bc, inner, dtype, at, "C"),
                           *_step_row(z, row, (), dtype, at, "z"),
                           *_step_row(out, row, (), dtype, at, "out"),
                           _flat(A, (channels, states), "float32", 4 * channels * states, at, "A"),
                           _flat(D, (channels,), "float32", 4 * channels, at, "D"),
                           _flat(delta_bias, (channels,), "float32", 4 * channels, at, "delta_bias"), s,
                           s if state_out is None else _flat(state_out, shape, "float32", nbytes, at, "state_out"),
                           _flat(slots, (batch,), "int32", 4 * batch, at, "slots"))
    rc = _n.lib.fg_scan_step(device.handle, args, _stream(stream, at))
    if rc:
        _n.check(rc)
