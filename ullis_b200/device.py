"""Operators on device memory: the methods of `CudaRuntime` that take and return torch tensors.

Tensors lie on the runtime's device; kernels go to torch's current stream of that device, outputs and workspaces come from
torch's allocator on it, and nothing waits for the device, so the calls may be captured into a graph.  A tensor that belongs to
another stream is ordered and kept alive by the caller, as for any torch operation.  Arguments that the operator does not take
raise `UllisCudaError`.  The arithmetic, the 8-bit tape and the limits are described at the entry points of
include/ullis_cuda.h.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple

from .errors import ERR_ARG, ERR_SHAPE, OK, UllisCudaError


class Tape(NamedTuple):
    """Activations in 8 bits: codes int8 (the shape of x), exponents uint8 [rows, ceil(channels / 32)]."""

    codes: object
    exponents: object


class HeadGrad(NamedTuple):
    """row_loss float32 [rows]; hidden, weight: gradients in hidden's type; scale (None for a dense head), bias (None without
    one): gradients in float32 [vocab]."""

    row_loss: object
    hidden: object
    weight: object
    scale: object
    bias: object


_TORCH, _DTYPES, _16, _RAW_STREAM = None, None, None, None


def _torch():
    global _TORCH, _DTYPES, _16, _RAW_STREAM
    if _TORCH is None:
        import torch

        _DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
        _16 = (torch.float16, torch.bfloat16)
        _RAW_STREAM = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
            (lambda device: torch.cuda.current_stream(device).cuda_stream)
        _TORCH = torch
    return _TORCH


_V, _Z, _I, _F, _U = C.c_void_p, C.c_size_t, C.c_int32, C.c_float, C.c_uint32
#: Argument types of the entry points: with them ctypes takes plain numbers, a third of the time of a call of twenty arguments.
_ARGTYPES = {
    "tape_pack": (_V, _V, _I, _V, _Z, _Z, _Z, _V, _V),
    "tape_unpack": (_V, _V, _I, _V, _V, _Z, _Z, _V, _Z),
    "tape_layer_norm": (_V, _V, _I, _V, _Z, _V, _V, _Z, _Z, _V, _V, _V),
    "tape_layer_norm_backward_workspace": (_V, _Z, _Z, _V),
    "tape_layer_norm_backward": (_V, _V, _I, _V, _V, _V, _Z, _V, _V, _Z, _Z, _Z, _V, _V, _V, _V, _Z),
    "tape_weight_grad_workspace": (_V, _Z, _Z, _Z, _V),
    "tape_weight_grad": (_V, _V, _I, _V, _V, _V, _Z, _Z, _Z, _Z, _V, _V, _Z),
    "head_ce_grad_workspace": (_V, _Z, _Z, _Z, _V),
    "head_ce_grad": (_V, _V, _I, _V, _Z, _V, _V, _V, _V, _V, _U, _Z, _Z, _Z, _Z, _F, _V, _V, _V, _V, _V, _V, _Z),
}


def declare(lib) -> None:
    for name, types in _ARGTYPES.items():
        getattr(lib, "ullis_cuda_" + name).argtypes = types


def _p(t):
    return None if t is None else t.data_ptr()


def _shape_error(name, got, expected):
    raise UllisCudaError(ERR_SHAPE, f"{name} length mismatch: got {tuple(got)}, expected {tuple(expected)}")


class DeviceOps:
    """Mixed into CudaRuntime."""

    # ------------------------------------------------------------------------------------------ arguments
    def _on_device(self, t) -> bool:
        return t.is_cuda and t.get_device() == self.device

    def _tensor(self, t, name, dtypes):
        torch = _torch()
        if not isinstance(t, torch.Tensor):
            raise UllisCudaError(ERR_ARG, f"{name} is not a tensor")
        if not self._on_device(t):
            raise UllisCudaError(ERR_ARG, f"{name} is not on the runtime's device (cuda:{self.device})")
        if t.dtype not in dtypes:
            raise UllisCudaError(ERR_ARG, f"{name} has the type {t.dtype}, not one of {', '.join(str(d) for d in dtypes)}")
        return t

    def _matrix(self, t, name, dtypes):
        """(tensor, rows, channels, row stride) of [..., channels] with contiguous channels and evenly spaced rows."""
        t = self._tensor(t, name, dtypes)
        if t.dim() < 2:
            raise UllisCudaError(ERR_SHAPE, f"{name} must have at least two dimensions")
        channels = t.shape[-1]
        if t.dim() != 2 or (channels > 1 and t.stride(1) != 1):
            if not t.is_contiguous():
                raise UllisCudaError(ERR_SHAPE, f"{name} must have contiguous channels and, with more than two dimensions, be contiguous")
            rows = t.numel() // channels if channels else 0
            return t, rows, channels, channels
        rows = t.shape[0]
        stride = t.stride(0) if rows > 1 else channels
        if stride < channels:
            raise UllisCudaError(ERR_SHAPE, f"{name} must not have overlapping rows")
        return t, rows, channels, stride

    def _vector(self, t, name, dtypes, n):
        t = self._tensor(t, name, dtypes)
        if t.numel() != n:
            _shape_error(name, t.shape, (n,))
        if not t.is_contiguous():
            raise UllisCudaError(ERR_SHAPE, f"{name} must be contiguous")
        return t

    def _tape(self, tape):
        torch = _torch()
        try:
            codes, exponents = tape
        except (TypeError, ValueError):
            raise UllisCudaError(ERR_ARG, "tape is not a pair of codes and exponents") from None
        codes = self._tensor(codes, "codes", (torch.int8,))
        exponents = self._tensor(exponents, "exponents", (torch.uint8,))
        if codes.dim() < 2 or not codes.is_contiguous() or not exponents.is_contiguous():
            raise UllisCudaError(ERR_SHAPE, "codes and exponents must be contiguous, codes with at least two dimensions")
        channels = codes.shape[-1]
        rows = codes.numel() // channels if channels else 0
        if exponents.numel() != rows * -(-channels // 32):
            _shape_error("exponents", exponents.shape, (rows, -(-channels // 32)))
        return codes, exponents, rows, channels

    def _workspace(self, like, name, *sizes):
        """(bytes of workspace from torch's allocator, how many); the size is asked for once per shape."""
        try:
            need = self._workspace_bytes[name, sizes]
        except (AttributeError, KeyError):
            value = C.c_size_t(0)
            rc = getattr(self._lib, f"ullis_cuda_{name}_workspace")(self._h, *sizes, C.byref(value))
            if rc != OK:
                raise UllisCudaError(rc, self._lib.ullis_cuda_last_error(None).decode()) from None
            need = value.value
            known = self.__dict__.setdefault("_workspace_bytes", {})
            if len(known) >= 4096:
                known.clear()
            known[name, sizes] = need
        return like.new_empty((need,), dtype=_TORCH.uint8), need

    # ------------------------------------------------------------------------------------------ the 8-bit tape
    def tape_pack(self, x) -> Tape:
        """x [..., channels] (float32, float16, bfloat16) in 8 bits: one exponent per 32 channels of a row."""
        torch = _torch()
        x, rows, channels, stride = self._matrix(x, "x", _DTYPES)
        codes = x.new_empty(x.shape, dtype=torch.int8)
        exponents = x.new_empty((rows, -(-channels // 32)), dtype=torch.uint8)
        self._check(self._lib.ullis_cuda_tape_pack(self._h, _RAW_STREAM(self.device), _DTYPES[x.dtype], _p(x), stride,
                                                   rows, channels, _p(codes), _p(exponents)))
        return Tape(codes, exponents)

    def tape_unpack(self, tape, dtype):
        """What the codes stand for, in `dtype`, in their shape."""
        torch = _torch()
        codes, exponents, rows, channels = self._tape(tape)
        if dtype not in _DTYPES:
            raise UllisCudaError(ERR_ARG, f"a tape does not unpack to {dtype}")
        x = codes.new_empty(codes.shape, dtype=dtype)
        self._check(self._lib.ullis_cuda_tape_unpack(self._h, _RAW_STREAM(self.device), _DTYPES[dtype], _p(codes), _p(exponents),
                                                     rows, channels, _p(x), channels))
        return x

    def tape_layer_norm(self, x, weight, bias):
        """(LayerNorm(x), tape of x): weight and bias float16 [channels]; y has the shape and type of x."""
        torch = _torch()
        x, rows, channels, stride = self._matrix(x, "x", _DTYPES)
        weight = self._vector(weight, "weight", (torch.float16,), channels)
        bias = self._vector(bias, "bias", (torch.float16,), channels)
        y = x.new_empty(x.shape)
        codes = x.new_empty(x.shape, dtype=torch.int8)
        exponents = x.new_empty((rows, -(-channels // 32)), dtype=torch.uint8)
        self._check(self._lib.ullis_cuda_tape_layer_norm(
            self._h, _RAW_STREAM(self.device), _DTYPES[x.dtype], _p(x), stride, _p(weight), _p(bias), rows,
            channels, _p(y), _p(codes), _p(exponents)))
        return y, Tape(codes, exponents)

    def tape_layer_norm_backward(self, tape, gy, weight, residual=None):
        """(gx, g_weight, g_bias) of LayerNorm at what the tape stands for; gx (the type and shape of gy) has `residual`,
        the gradient that comes past the norm, added to it; the gradients of weight and bias are float32."""
        torch = _torch()
        codes, exponents, rows, channels = self._tape(tape)
        gy, g_rows, g_channels, stride = self._matrix(gy, "gy", _DTYPES)
        if (g_rows, g_channels) != (rows, channels):
            _shape_error("gy", gy.shape, codes.shape)
        weight = self._vector(weight, "weight", (torch.float16,), channels)
        r_stride = channels
        if residual is not None:
            residual, r_rows, r_channels, r_stride = self._matrix(residual, "residual", (gy.dtype,))
            if (r_rows, r_channels) != (rows, channels):
                _shape_error("residual", residual.shape, gy.shape)
        gx = gy.new_empty(gy.shape)
        g = gy.new_empty((2, channels), dtype=torch.float32)
        at = g.data_ptr()
        work, size = self._workspace(gy, "tape_layer_norm_backward", rows, channels)
        self._check(self._lib.ullis_cuda_tape_layer_norm_backward(
            self._h, _RAW_STREAM(self.device), _DTYPES[gy.dtype], _p(codes), _p(exponents), _p(gy), stride, _p(weight),
            _p(residual), r_stride, rows, channels, _p(gx), at,
            at + 4 * channels, _p(work), size))
        return (gx, *g.unbind(0))

    def tape_weight_grad(self, tape, gy):
        """Gradient of a linear's weights, float32 [out, in]: gy [..., out] (float16, bfloat16) transposed times what the tape
        of the linear's input stands for."""
        torch = _torch()
        codes, exponents, rows, channels = self._tape(tape)
        gy, g_rows, out, stride = self._matrix(gy, "gy", _16)
        if g_rows != rows:
            _shape_error("gy", gy.shape, (rows, out))
        g = gy.new_empty((out, channels), dtype=torch.float32)
        work, size = self._workspace(gy, "tape_weight_grad", rows, channels, out)
        self._check(self._lib.ullis_cuda_tape_weight_grad(
            self._h, _RAW_STREAM(self.device), _DTYPES[gy.dtype], _p(codes), _p(exponents), _p(gy), stride, rows,
            channels, out, _p(g), _p(work), size))
        return g

    # ------------------------------------------------------------------------------------------ head
    def head_ce_grad(self, hidden, weight, labels, *, scale=None, bias=None, ignore_id: int = 0xFFFFFFFF, time=None,
                     loss_scale: float = 1.0) -> HeadGrad:
        """Next-token cross-entropy of a head with its gradient; logits are never kept.

        hidden [..., channels] float16 or bfloat16; labels int32, one per row (a negative id and `ignore_id` are taken as the
        unsigned 32-bit number they are); `time` rows to a sequence (default: all, or with three dimensions the second).  A
        packed head is `weight` int32 words of sign bits in checkpoint order with `scale` float16 [vocab]; a dense one is
        `weight` [vocab, channels] in hidden's type and no scale.  bias float16 [vocab] or None.  Gradients are of
        loss_scale * sum of row_loss; that of a packed weight is of the +/-1 values."""
        torch = _torch()
        hidden, rows, channels, stride = self._matrix(hidden, "hidden", _16)
        labels = self._vector(labels, "labels", (torch.int32,), rows)
        if time is None:
            time = hidden.shape[-2] if hidden.dim() == 3 else max(rows, 1)
        if scale is not None:
            scale = self._tensor(scale, "scale", (torch.float16,))
            vocab = scale.numel()
            scale = self._vector(scale, "scale", (torch.float16,), vocab)
            weight = self._vector(weight, "weight", (torch.int32,), (vocab * channels + 31) // 32)
        else:
            weight = self._tensor(weight, "weight", (hidden.dtype,))
            if weight.dim() != 2 or weight.shape[1] != channels or not weight.is_contiguous():
                _shape_error("weight", weight.shape, ("vocab", channels))
            vocab = weight.shape[0]
        if bias is not None:
            bias = self._vector(bias, "bias", (torch.float16,), vocab)
        ignore = int(ignore_id)
        if not -(1 << 31) <= ignore < 1 << 32:
            raise UllisCudaError(ERR_ARG, "ignore_id is not a 32-bit number")
        if not 0 < int(time) < 1 << 31 or rows % int(time):
            raise UllisCudaError(ERR_SHAPE, "rows must be a multiple of time")
        row_loss = hidden.new_empty((rows,), dtype=torch.float32)
        g_hidden = hidden.new_empty(hidden.shape)
        g_weight = hidden.new_empty((vocab, channels))
        g_scale = None if scale is None else hidden.new_empty((vocab,), dtype=torch.float32)
        g_bias = None if bias is None else hidden.new_empty((vocab,), dtype=torch.float32)
        work, size = self._workspace(hidden, "head_ce_grad", rows, channels, vocab)
        packed = scale is not None
        self._check(self._lib.ullis_cuda_head_ce_grad(
            self._h, _RAW_STREAM(self.device), _DTYPES[hidden.dtype], _p(hidden), stride, _p(weight if packed else None),
            _p(None if packed else weight), _p(scale), _p(bias), _p(labels), ignore & 0xFFFFFFFF, rows,
            int(time), channels, vocab, float(loss_scale), _p(row_loss), _p(g_hidden), _p(g_weight), _p(g_scale),
            _p(g_bias), _p(work), size))
        return HeadGrad(row_loss, g_hidden, g_weight, g_scale, g_bias)
