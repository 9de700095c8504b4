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


_DTYPES = None


def _torch():
    import torch

    global _DTYPES
    if _DTYPES is None:
        _DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
    return torch


def _z(n):
    return C.c_size_t(n)


def _p(t):
    return C.c_void_p(None if t is None else t.data_ptr())


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

    def _stream_of(self):
        return C.c_void_p(_torch().cuda.current_stream(self.device).cuda_stream)

    def _new(self, shape, dtype):
        torch = _torch()
        return torch.empty(shape, dtype=dtype, device=torch.device("cuda", self.device))

    def _workspace(self, fn, *sizes):
        need = C.c_size_t(0)
        rc = fn(self._h, *sizes, C.byref(need))
        if rc != OK:
            raise UllisCudaError(rc, self._lib.ullis_cuda_last_error(None).decode())
        return self._new((max(need.value, 1),), _torch().uint8), _z(need.value)

    # ------------------------------------------------------------------------------------------ the 8-bit tape
    def tape_pack(self, x) -> Tape:
        """x [..., channels] (float32, float16, bfloat16) in 8 bits: one exponent per 32 channels of a row."""
        torch = _torch()
        x, rows, channels, stride = self._matrix(x, "x", tuple(_DTYPES))
        codes = self._new(x.shape, torch.int8)
        exponents = self._new((rows, -(-channels // 32)), torch.uint8)
        self._check(self._lib.ullis_cuda_tape_pack(self._h, self._stream_of(), C.c_int32(_DTYPES[x.dtype]), _p(x), _z(stride),
                                                   _z(rows), _z(channels), _p(codes), _p(exponents)))
        return Tape(codes, exponents)

    def tape_unpack(self, tape, dtype):
        """What the codes stand for, in `dtype`, in their shape."""
        torch = _torch()
        codes, exponents, rows, channels = self._tape(tape)
        if dtype not in _DTYPES:
            raise UllisCudaError(ERR_ARG, f"a tape does not unpack to {dtype}")
        x = self._new(codes.shape, dtype)
        self._check(self._lib.ullis_cuda_tape_unpack(self._h, self._stream_of(), C.c_int32(_DTYPES[dtype]), _p(codes), _p(exponents),
                                                     _z(rows), _z(channels), _p(x), _z(channels)))
        return x

    def tape_layer_norm(self, x, weight, bias):
        """(LayerNorm(x), tape of x): weight and bias float16 [channels]; y has the shape and type of x."""
        torch = _torch()
        x, rows, channels, stride = self._matrix(x, "x", tuple(_DTYPES))
        weight = self._vector(weight, "weight", (torch.float16,), channels)
        bias = self._vector(bias, "bias", (torch.float16,), channels)
        y = self._new(x.shape, x.dtype)
        codes = self._new(x.shape, torch.int8)
        exponents = self._new((rows, -(-channels // 32)), torch.uint8)
        self._check(self._lib.ullis_cuda_tape_layer_norm(
            self._h, self._stream_of(), C.c_int32(_DTYPES[x.dtype]), _p(x), _z(stride), _p(weight), _p(bias), _z(rows),
            _z(channels), _p(y), _p(codes), _p(exponents)))
        return y, Tape(codes, exponents)

    def tape_layer_norm_backward(self, tape, gy, weight, residual=None):
        """(gx, g_weight, g_bias) of LayerNorm at what the tape stands for; gx (the type and shape of gy) has `residual`,
        the gradient that comes past the norm, added to it; the gradients of weight and bias are float32."""
        torch = _torch()
        codes, exponents, rows, channels = self._tape(tape)
        gy, g_rows, g_channels, stride = self._matrix(gy, "gy", tuple(_DTYPES))
        if (g_rows, g_channels) != (rows, channels):
            _shape_error("gy", gy.shape, codes.shape)
        weight = self._vector(weight, "weight", (torch.float16,), channels)
        r_stride = channels
        if residual is not None:
            residual, r_rows, r_channels, r_stride = self._matrix(residual, "residual", (gy.dtype,))
            if (r_rows, r_channels) != (rows, channels):
                _shape_error("residual", residual.shape, gy.shape)
        gx = self._new(gy.shape, gy.dtype)
        g = self._new((2, channels), torch.float32)
        work, size = self._workspace(self._lib.ullis_cuda_tape_layer_norm_backward_workspace, _z(rows), _z(channels))
        self._check(self._lib.ullis_cuda_tape_layer_norm_backward(
            self._h, self._stream_of(), C.c_int32(_DTYPES[gy.dtype]), _p(codes), _p(exponents), _p(gy), _z(stride), _p(weight),
            _p(residual), _z(r_stride), _z(rows), _z(channels), _p(gx), C.c_void_p(g.data_ptr()),
            C.c_void_p(g.data_ptr() + 4 * channels), _p(work), size))
        return gx, g[0], g[1]

    def tape_weight_grad(self, tape, gy):
        """Gradient of a linear's weights, float32 [out, in]: gy [..., out] (float16, bfloat16) transposed times what the tape
        of the linear's input stands for."""
        torch = _torch()
        codes, exponents, rows, channels = self._tape(tape)
        gy, g_rows, out, stride = self._matrix(gy, "gy", (torch.float16, torch.bfloat16))
        if g_rows != rows:
            _shape_error("gy", gy.shape, (rows, out))
        g = self._new((out, channels), torch.float32)
        work, size = self._workspace(self._lib.ullis_cuda_tape_weight_grad_workspace, _z(rows), _z(channels), _z(out))
        self._check(self._lib.ullis_cuda_tape_weight_grad(
            self._h, self._stream_of(), C.c_int32(_DTYPES[gy.dtype]), _p(codes), _p(exponents), _p(gy), _z(stride), _z(rows),
            _z(channels), _z(out), _p(g), _p(work), size))
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
        hidden, rows, channels, stride = self._matrix(hidden, "hidden", (torch.float16, torch.bfloat16))
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
        row_loss = self._new((rows,), torch.float32)
        g_hidden = self._new(hidden.shape, hidden.dtype)
        g_weight = self._new((vocab, channels), hidden.dtype)
        g_scale = None if scale is None else self._new((vocab,), torch.float32)
        g_bias = None if bias is None else self._new((vocab,), torch.float32)
        work, size = self._workspace(self._lib.ullis_cuda_head_ce_grad_workspace, _z(rows), _z(channels), _z(vocab))
        packed = scale is not None
        self._check(self._lib.ullis_cuda_head_ce_grad(
            self._h, self._stream_of(), C.c_int32(_DTYPES[hidden.dtype]), _p(hidden), _z(stride), _p(weight if packed else None),
            _p(None if packed else weight), _p(scale), _p(bias), _p(labels), C.c_uint32(ignore & 0xFFFFFFFF), _z(rows),
            _z(int(time)), _z(channels), _z(vocab), C.c_float(loss_scale), _p(row_loss), _p(g_hidden), _p(g_weight), _p(g_scale),
            _p(g_bias), _p(work), size))
        return HeadGrad(row_loss, g_hidden, g_weight, g_scale, g_bias)
