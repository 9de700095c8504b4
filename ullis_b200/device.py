"""Operators on device memory: the methods of `CudaRuntime` that take and return torch tensors.

Tensors lie on the runtime's device; kernels go to torch's current stream of that device, outputs and workspaces come from
torch's allocator on it, and nothing waits for the device, so the calls may be captured into a graph.  A tensor that belongs to
another stream is ordered and kept alive by the caller, as for any torch operation.  Autograd does not see the calls: inputs may
require gradients, outputs track nothing.  Arguments that the operator does not take raise `UllisCudaError`, and so does the next
call of the runtime after a kernel that gave up waiting (none does in working order).  The arithmetic, the 8-bit tape and the
limits are described at the entry points of include/ullis_cuda.h.
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


class TopLogits(NamedTuple):
    """ids int32 and logits (the type they were taken from) [..., k]."""

    ids: object
    logits: object


_TORCH = _RAW_STREAM = None
_DTYPES = _16 = _F16 = _I8 = _U8 = _I32 = None   # the types that arguments may have


def _torch():
    global _TORCH, _RAW_STREAM, _DTYPES, _16, _F16, _I8, _U8, _I32
    if _TORCH is None:
        import torch

        _DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
        _16, _F16, _I8, _U8, _I32 = (torch.float16, torch.bfloat16), (torch.float16,), (torch.int8,), (torch.uint8,), (torch.int32,)
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
    "embed": (_V, _V, _I, _V, _Z, _V, _U, _F, _Z, _Z, _Z, _I, _V),
    "embed_grad_workspace": (_V, _I, _Z, _Z, _Z, _V),
    "embed_grad": (_V, _V, _I, _V, _U, _V, _Z, _Z, _Z, _Z, _F, _V, _V, _Z),
    "top_logits": (_V, _V, _I, _V, _Z, _Z, _Z, _Z, _V, _V),
    "head_distill_grad_workspace": (_V, _Z, _Z, _Z, _Z, _I, _I, _V),
    "head_distill_grad": (_V, _V, _I, _V, _Z, _V, _V, _V, _V, _V, _I, _V, _Z, _F, _F, _V, _U, _Z, _Z, _Z, _Z, _F, _V, _V, _V, _V, _V, _V, _Z),
    "head_ce_grad_workspace": (_V, _Z, _Z, _Z, _I, _V),
    "head_ce_grad": (_V, _V, _I, _V, _Z, _V, _V, _V, _V, _V, _U, _Z, _Z, _Z, _Z, _F, _V, _V, _V, _V, _V, _V, _Z),
}


def declare(lib) -> None:
    for name, types in _ARGTYPES.items():
        getattr(lib, "ullis_cuda_" + name).argtypes = types


def _p(t):
    return None if t is None else t.data_ptr()


def _like(t, dtype):
    """An output of t's shape, without gaps.  (Sizes as single numbers: torch takes a tuple of them twice as long.)"""
    return _TORCH.empty_like(t, dtype=dtype) if t.is_contiguous() else _TORCH.empty(*t.shape, dtype=dtype, device=t.device)


def _id32(ignore_id):
    ignore = int(ignore_id)
    if not -(1 << 31) <= ignore < 1 << 32:
        raise UllisCudaError(ERR_ARG, "ignore_id is not a 32-bit number")
    return ignore & 0xFFFFFFFF


def _shape_error(name, got, expected):
    raise UllisCudaError(ERR_SHAPE, f"{name} length mismatch: got {tuple(got)}, expected {tuple(expected)}")


class DeviceOps:
    """Mixed into CudaRuntime."""

    # ------------------------------------------------------------------------------------------ arguments
    # A call's checks are on the way of every launch: each begins with what an ordinary argument is, and only another one is
    # looked at more closely.
    def _on_device(self, t) -> bool:
        return t.get_device() == self.device          # -1 on the host

    def _refuse(self, t, name, dtypes):
        if not isinstance(t, _torch().Tensor):
            raise UllisCudaError(ERR_ARG, f"{name} is not a tensor")
        if not self._on_device(t):
            raise UllisCudaError(ERR_ARG, f"{name} is not on the runtime's device (cuda:{self.device})")
        if t.dtype not in dtypes:
            raise UllisCudaError(ERR_ARG, f"{name} has the type {t.dtype}, not one of {', '.join(str(d) for d in dtypes)}")

    def _matrix(self, t, name, dtypes):
        """(rows, channels, row stride) of [..., channels] with contiguous channels and evenly spaced rows."""
        try:
            if t.dtype in dtypes and self._on_device(t) and t.dim() == 2 and t.is_contiguous():
                rows, channels = t.shape
                return rows, channels, channels
        except AttributeError:
            pass
        self._refuse(t, name, dtypes)
        if t.dim() < 2:
            raise UllisCudaError(ERR_SHAPE, f"{name} must have at least two dimensions")
        channels = t.shape[-1]
        if t.dim() != 2 or (channels > 1 and t.stride(1) != 1):
            if not t.is_contiguous():
                raise UllisCudaError(ERR_SHAPE, f"{name} must have contiguous channels and, with more than two dimensions, be contiguous")
            return (t.numel() // channels if channels else 0), channels, channels
        rows = t.shape[0]
        stride = t.stride(0) if rows > 1 else channels
        if stride < channels:
            raise UllisCudaError(ERR_SHAPE, f"{name} must not have overlapping rows")
        return rows, channels, stride

    def _ids(self, t, name):
        """int32 without gaps, of any shape."""
        try:
            if t.dtype in _I32 and self._on_device(t) and t.is_contiguous():
                return
        except AttributeError:
            pass
        self._refuse(t, name, _I32)
        if not t.is_contiguous():
            raise UllisCudaError(ERR_SHAPE, f"{name} must be contiguous")

    def _vector(self, t, name, dtypes, n):
        try:
            if t.dtype in dtypes and self._on_device(t) and t.numel() == n and t.is_contiguous():
                return
        except AttributeError:
            pass
        self._refuse(t, name, dtypes)
        if t.numel() != n:
            _shape_error(name, t.shape, (n,))
        raise UllisCudaError(ERR_SHAPE, f"{name} must be contiguous")

    def _tape(self, tape):
        _torch()
        try:
            codes, exponents = tape
        except (TypeError, ValueError):
            raise UllisCudaError(ERR_ARG, "tape is not a pair of codes and exponents") from None
        self._refuse(codes, "codes", _I8)
        self._refuse(exponents, "exponents", _U8)
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
        return _TORCH.empty(need, dtype=_TORCH.uint8, device=like.device) if need else None, need

    # ------------------------------------------------------------------------------------------ the 8-bit tape
    def tape_pack(self, x) -> Tape:
        """x [..., channels] (float32, float16, bfloat16) in 8 bits: one exponent per 32 channels of a row."""
        torch = _torch()
        rows, channels, stride = self._matrix(x, "x", _DTYPES)
        codes = _like(x, torch.int8)
        exponents = torch.empty(rows, -(-channels // 32), dtype=torch.uint8, device=x.device)
        self._check(self._lib.ullis_cuda_tape_pack(self._h, _RAW_STREAM(self.device), _DTYPES[x.dtype], x.data_ptr(), stride, rows,
                                                   channels, codes.data_ptr(), exponents.data_ptr()))
        return Tape(codes, exponents)

    def tape_unpack(self, tape, dtype):
        """What the codes stand for, in `dtype`, in their shape."""
        codes, exponents, rows, channels = self._tape(tape)
        if dtype not in _DTYPES:
            raise UllisCudaError(ERR_ARG, f"a tape does not unpack to {dtype}")
        x = _like(codes, dtype)
        self._check(self._lib.ullis_cuda_tape_unpack(self._h, _RAW_STREAM(self.device), _DTYPES[dtype], codes.data_ptr(),
                                                     exponents.data_ptr(), rows, channels, x.data_ptr(), channels))
        return x

    def tape_layer_norm(self, x, weight, bias):
        """(LayerNorm(x), tape of x): weight and bias float16 [channels]; y has the shape and type of x."""
        torch = _torch()
        rows, channels, stride = self._matrix(x, "x", _DTYPES)
        self._vector(weight, "weight", _F16, channels)
        self._vector(bias, "bias", _F16, channels)
        y = _like(x, x.dtype)
        codes = _like(x, torch.int8)
        exponents = torch.empty(rows, -(-channels // 32), dtype=torch.uint8, device=x.device)
        self._check(self._lib.ullis_cuda_tape_layer_norm(
            self._h, _RAW_STREAM(self.device), _DTYPES[x.dtype], x.data_ptr(), stride, weight.data_ptr(), bias.data_ptr(), rows,
            channels, y.data_ptr(), codes.data_ptr(), exponents.data_ptr()))
        return y, Tape(codes, exponents)

    def tape_layer_norm_backward(self, tape, gy, weight, residual=None):
        """(gx, g_weight, g_bias) of LayerNorm at what the tape stands for; gx (the type and shape of gy) has `residual`,
        the gradient that comes past the norm, added to it; the gradients of weight and bias are float32."""
        codes, exponents, rows, channels = self._tape(tape)
        g_rows, g_channels, stride = self._matrix(gy, "gy", _DTYPES)
        if g_rows != rows or g_channels != channels:
            _shape_error("gy", gy.shape, codes.shape)
        self._vector(weight, "weight", _F16, channels)
        past, past_stride = None, channels
        if residual is not None:
            r_rows, r_channels, past_stride = self._matrix(residual, "residual", (gy.dtype,))
            if r_rows != rows or r_channels != channels:
                _shape_error("residual", residual.shape, gy.shape)
            past = residual.data_ptr()
        gx = _like(gy, gy.dtype)
        g_weight, g_bias = _like(weight, _TORCH.float32), _like(weight, _TORCH.float32)
        work, size = self._workspace(gy, "tape_layer_norm_backward", rows, channels)
        self._check(self._lib.ullis_cuda_tape_layer_norm_backward(
            self._h, _RAW_STREAM(self.device), _DTYPES[gy.dtype], codes.data_ptr(), exponents.data_ptr(), gy.data_ptr(), stride,
            weight.data_ptr(), past, past_stride, rows, channels, gx.data_ptr(), g_weight.data_ptr(),
            g_bias.data_ptr(), _p(work), size))
        return gx, g_weight, g_bias

    def tape_weight_grad(self, tape, gy):
        """Gradient of a linear's weights, float32 [out, in]: gy [..., out] (float16, bfloat16) transposed times what the tape
        of the linear's input stands for."""
        codes, exponents, rows, channels = self._tape(tape)
        g_rows, out, stride = self._matrix(gy, "gy", _16)
        if g_rows != rows:
            _shape_error("gy", gy.shape, (rows, out))
        g = _TORCH.empty(out, channels, dtype=_TORCH.float32, device=gy.device)
        work, size = self._workspace(gy, "tape_weight_grad", rows, channels, out)
        self._check(self._lib.ullis_cuda_tape_weight_grad(
            self._h, _RAW_STREAM(self.device), _DTYPES[gy.dtype], codes.data_ptr(), exponents.data_ptr(), gy.data_ptr(), stride, rows,
            channels, out, g.data_ptr(), _p(work), size))
        return g

    # ------------------------------------------------------------------------------------------ embedding
    def embed(self, table, tokens, *, scale: float = 1.0, dtype=None, ignore_id: int = 0xFFFFFFFF):
        """scale * table[tokens], [*tokens.shape, channels] in `dtype` (default: the table's type).

        table [vocab, channels] float32, float16 or bfloat16; tokens int32 of any shape (a negative id and `ignore_id` are taken as
        the unsigned 32-bit number they are).  The row of `ignore_id` is zero, that of any other id outside the table NaN."""
        torch = _torch()
        vocab, channels, stride = self._matrix(table, "table", _DTYPES)
        if table.dim() != 2:
            raise UllisCudaError(ERR_SHAPE, "table must have two dimensions")
        self._ids(tokens, "tokens")
        dtype = table.dtype if dtype is None else dtype
        if dtype not in _DTYPES:
            raise UllisCudaError(ERR_ARG, f"an embedding has no type {dtype}")
        ignore = _id32(ignore_id)
        y = torch.empty(*tokens.shape, channels, dtype=dtype, device=table.device)
        self._check(self._lib.ullis_cuda_embed(
            self._h, _RAW_STREAM(self.device), _DTYPES[table.dtype], table.data_ptr(), stride, tokens.data_ptr(), ignore, float(scale),
            tokens.numel(), channels, vocab, _DTYPES[dtype], y.data_ptr()))
        return y

    def embed_grad(self, tokens, gy, vocab: int, *, scale: float = 1.0, ignore_id: int = 0xFFFFFFFF):
        """Gradient of `embed`'s table, float32 [vocab, channels]: scale * the sum of gy [*tokens.shape, channels] (float32, float16,
        bfloat16) over the rows of each token.  `ignore_id` and ids outside the table add nothing."""
        torch = _torch()
        self._ids(tokens, "tokens")
        if tokens.dim() == 0 and isinstance(gy, torch.Tensor) and gy.dim() == 1:
            gy = gy[None]                  # of a token without dimensions, whose row `embed` gives without them too
        rows, channels, stride = self._matrix(gy, "gy", _DTYPES)
        if tokens.numel() != rows:
            _shape_error("tokens", tokens.shape, gy.shape[:-1])
        vocab, ignore = int(vocab), _id32(ignore_id)
        if not 0 < vocab < 1 << 31:
            raise UllisCudaError(ERR_SHAPE, "vocab must be positive and below 2^31")
        g = torch.empty(vocab, channels, dtype=torch.float32, device=gy.device)
        work, size = self._workspace(gy, "embed_grad", _DTYPES[gy.dtype], rows, channels, vocab)
        self._check(self._lib.ullis_cuda_embed_grad(
            self._h, _RAW_STREAM(self.device), _DTYPES[gy.dtype], tokens.data_ptr(), ignore, gy.data_ptr(), stride, rows,
            channels, vocab, float(scale), g.data_ptr(), _p(work), size))
        return g

    # ------------------------------------------------------------------------------------------ a teacher's logits
    def top_logits(self, logits, k: int) -> TopLogits:
        """The k largest of logits [..., vocab] (float32, float16, bfloat16) in falling order, equal ones by rising id; NaN is
        above all others.  k at most 256."""
        torch = _torch()
        rows, vocab, stride = self._matrix(logits, "logits", _DTYPES)
        k = int(k)
        if not 0 < k <= min(vocab, 256):
            raise UllisCudaError(ERR_SHAPE, f"top logits: k must be at least 1 and at most {min(vocab, 256)}")
        lead, device = logits.shape[:-1], logits.device
        ids = torch.empty(*lead, k, dtype=torch.int32, device=device)
        top = torch.empty(*lead, k, dtype=logits.dtype, device=device)
        self._check(self._lib.ullis_cuda_top_logits(self._h, _RAW_STREAM(self.device), _DTYPES[logits.dtype], logits.data_ptr(), stride,
                                                    rows, vocab, k, ids.data_ptr(), top.data_ptr()))
        return TopLogits(ids, top)

    # ------------------------------------------------------------------------------------------ head
    def head_ce_grad(self, hidden, weight, labels, *, scale=None, bias=None, ignore_id: int = 0xFFFFFFFF, time=None,
                     loss_scale: float = 1.0) -> HeadGrad:
        """Next-token cross-entropy of a head with its gradient; logits are never kept.

        hidden [..., channels] float16 or bfloat16; labels int32, one per row (a negative id and `ignore_id` are taken as the
        unsigned 32-bit number they are); `time` rows to a sequence (default: all, or with three dimensions the second; at
        most 2^24 in all).  A
        packed head is `weight` int32 words of sign bits in checkpoint order with `scale` float16 [vocab]; a dense one is
        `weight` [vocab, channels] in hidden's type and no scale.  bias float16 [vocab] or None.  Gradients are of
        loss_scale * sum of row_loss; that of a packed weight is of the +/-1 values."""
        _torch()
        rows, channels, stride = self._matrix(hidden, "hidden", _16)
        self._vector(labels, "labels", _I32, rows)
        vocab = self._head(hidden, channels, weight, scale, bias)
        ignore, time = _id32(ignore_id), self._time(hidden, rows, time)
        outputs, copies = self._head_outputs(hidden, rows, channels, vocab, weight, scale, bias)
        at = weight.data_ptr()
        work, size = self._workspace(hidden, "head_ce_grad", rows, channels, vocab, copies)
        self._check(self._lib.ullis_cuda_head_ce_grad(
            self._h, _RAW_STREAM(self.device), _DTYPES[hidden.dtype], hidden.data_ptr(), stride, at if scale is not None else None,
            at if scale is None else None, _p(scale), _p(bias), labels.data_ptr(), ignore, rows, time, channels, vocab,
            float(loss_scale), *(_p(t) for t in outputs), _p(work), size))
        return outputs

    def head_distill_grad(self, hidden, weight, top_ids, top_logits, *, scale=None, bias=None, labels=None, alpha: float = 1.0,
                          temperature: float = 1.0, ignore_id: int = 0xFFFFFFFF, time=None, loss_scale: float = 1.0) -> HeadGrad:
        """A head's distillation from a teacher's largest logits, with its gradient; the student's logits are never kept.

        hidden, weight, scale, bias, ignore_id, time, loss_scale and what is returned are `head_ce_grad`'s.  top_ids int32 and
        top_logits (float32, float16, bfloat16) [..., k], k at most 256: what the teacher says of the token after each row, as
        `top_logits` gives it; a negative id is no entry, and one that comes twice has the sum of both probabilities.  The
        teacher's distribution is softmax(top_logits / temperature) over a row's entries, and

            row_loss = (1 - alpha) * cross-entropy(label) + alpha * temperature^2 * KL(teacher, softmax(logits / temperature)).

        With `labels` a row counts as in `head_ce_grad`, for both parts; one without entries has the first part alone.  Without
        labels there is the second part alone, and a row counts if it has entries.  alpha in 0..1, temperature in 1/128..128."""
        _torch()
        rows, channels, stride = self._matrix(hidden, "hidden", _16)
        if labels is not None:
            self._vector(labels, "labels", _I32, rows)
        self._ids(top_ids, "top_ids")
        top = top_ids.shape[-1] if top_ids.dim() else 0
        if not 0 < top <= 256:
            raise UllisCudaError(ERR_SHAPE, "head distillation takes 1 to 256 entries of a row")
        if top_ids.numel() != rows * top:
            _shape_error("top_ids", top_ids.shape, (rows, top))
        self._vector(top_logits, "top_logits", _DTYPES, rows * top)
        if top_logits.shape != top_ids.shape:
            _shape_error("top_logits", top_logits.shape, top_ids.shape)
        alpha, temperature = float(alpha), float(temperature)
        if not 0.0 <= alpha <= 1.0 or not 1 / 128 <= temperature <= 128:
            raise UllisCudaError(ERR_ARG, "alpha must be in 0 .. 1, temperature in 1/128 .. 128")
        vocab = self._head(hidden, channels, weight, scale, bias)
        ignore, time = _id32(ignore_id), self._time(hidden, rows, time)
        outputs, copies = self._head_outputs(hidden, rows, channels, vocab, weight, scale, bias)
        at = weight.data_ptr()
        work, size = self._workspace(hidden, "head_distill_grad", rows, channels, vocab, top, int(labels is not None), copies)
        self._check(self._lib.ullis_cuda_head_distill_grad(
            self._h, _RAW_STREAM(self.device), _DTYPES[hidden.dtype], hidden.data_ptr(), stride, at if scale is not None else None,
            at if scale is None else None, _p(scale), _p(bias), top_ids.data_ptr(), _DTYPES[top_logits.dtype], top_logits.data_ptr(), top,
            alpha, temperature, _p(labels), ignore, rows, time, channels, vocab, float(loss_scale), *(_p(t) for t in outputs),
            _p(work), size))
        return outputs

    def _time(self, hidden, rows, time) -> int:
        if time is None:
            time = max(1, hidden.shape[-2] if hidden.dim() == 3 else rows)
        time = int(time)
        if not 0 < time < 1 << 31 or rows % time:
            raise UllisCudaError(ERR_SHAPE, "rows must be a multiple of time")
        return time

    def _head(self, hidden, channels, weight, scale, bias) -> int:
        """The vocabulary of a packed or dense head."""
        if scale is not None:
            self._refuse(scale, "scale", _F16)
            vocab = scale.numel()
            self._vector(scale, "scale", _F16, vocab)
            self._vector(weight, "weight", _I32, (vocab * channels + 31) // 32)
        else:
            self._refuse(weight, "weight", (hidden.dtype,))
            if weight.dim() != 2 or weight.shape[1] != channels or not weight.is_contiguous():
                _shape_error("weight", weight.shape, ("vocab", channels))
            vocab = weight.shape[0]
        if bias is not None:
            self._vector(bias, "bias", _F16, vocab)
        return vocab

    def _head_outputs(self, hidden, rows, channels, vocab, weight, scale, bias):
        """(where the gradients go, whether the workspace holds the weights)."""
        empty, f32, device = _TORCH.empty, _TORCH.float32, hidden.device
        outputs = HeadGrad(empty(rows, dtype=f32, device=device), _like(hidden, hidden.dtype),
                           empty(vocab, channels, dtype=hidden.dtype, device=device), None if scale is None else _like(scale, f32),
                           None if bias is None else _like(bias, f32))
        return outputs, int(scale is not None or channels % 8 != 0 or weight.data_ptr() % 16 != 0)
