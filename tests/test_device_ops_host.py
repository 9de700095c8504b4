"""The operators on device memory as far as they go without a device: the tape's exponent rule, compiled for the host, and
what the Python layer refuses before it calls the library."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest
import torch

from ullis_b200 import cuda, device
from ullis_b200.device import DeviceOps

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="session")
def exponent_bytes(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("tape_host") / "libtape_host.so")
    cuda_home = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    subprocess.run(["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-I", os.path.join(cuda_home, "include"),
                    os.path.join(ROOT, "tests", "host_harness", "tape_host.cpp"), "-o", out], check=True)
    lib = C.CDLL(out)

    def run(bits):
        bits = np.ascontiguousarray(bits, np.uint32)
        got = np.zeros(bits.size, np.uint8)
        lib.tape_exponent_bytes(C.c_void_p(bits.ctypes.data), C.c_void_p(got.ctypes.data), C.c_size_t(bits.size))
        return got.astype(np.int64)

    return run


def test_the_exponent_is_the_smallest_that_holds_the_largest_value(exponent_bytes):
    edges = np.uint32([(e << 23) + m for e in range(255) for m in (0, 1, 0x400000, 0x7DFFFF, 0x7E0000, 0x7E0001, 0x7FFFFF)])
    drawn = np.random.default_rng(3).integers(0, 0x7F800000, 200_000).astype(np.uint32)
    bits = np.concatenate([edges[edges < 0x7F800000], drawn])
    top = bits.view(np.float32).astype(np.float64)
    e = exponent_bytes(bits) - 127
    assert (e >= -126).all() and (e <= 121).all()
    assert ((127.0 * np.exp2(e) >= top) | (e == 121)).all()
    assert ((127.0 * np.exp2(e - 1.0) < top) | (e == -126)).all()
    assert (exponent_bytes([0x7F800000, 0x7FC00000, 0x7FFFFFFF]) == 255).all()


class Fake(DeviceOps):
    """The Python checks alone: CPU tensors stand for the device's, and a library call is a failure."""

    device = 0

    def _on_device(self, t):
        return t.device.type == "cpu"

    class _Lib:
        def __getattr__(self, name):
            raise AssertionError(f"{name} was reached")

    _lib, _h = _Lib(), None


H, F, I8, U8 = torch.float16, torch.float32, torch.int8, torch.uint8


def codes(rows=4, channels=64):
    return torch.zeros(rows, channels, dtype=I8), torch.zeros(rows, -(-channels // 32), dtype=U8)


def hidden(rows=4, channels=64):
    return torch.zeros(rows, channels, dtype=H)


def dense(vocab=9, channels=64):
    return torch.zeros(vocab, channels, dtype=H)


def labels(rows):
    return torch.zeros(rows, dtype=torch.int32)


REFUSED = {
    "pack: an array": (lambda rt: rt.tape_pack(np.zeros((4, 64), np.float32)), cuda.ERR_ARG),
    "pack: another device": (lambda rt: rt.tape_pack(torch.zeros(4, 64, device="meta")), cuda.ERR_ARG),
    "pack: a type": (lambda rt: rt.tape_pack(torch.zeros(4, 64, dtype=torch.float64)), cuda.ERR_ARG),
    "pack: one dimension": (lambda rt: rt.tape_pack(torch.zeros(64)), cuda.ERR_SHAPE),
    "pack: transposed": (lambda rt: rt.tape_pack(torch.zeros(64, 4).t()), cuda.ERR_SHAPE),
    "pack: rows on top of each other": (lambda rt: rt.tape_pack(torch.zeros(1, 64).expand(4, 64)), cuda.ERR_SHAPE),
    "pack: a sliced cube": (lambda rt: rt.tape_pack(torch.zeros(2, 4, 80)[:, :, :64]), cuda.ERR_SHAPE),
    "unpack: no pair": (lambda rt: rt.tape_unpack(torch.zeros(4, 64, dtype=I8), F), cuda.ERR_ARG),
    "unpack: unsigned codes": (lambda rt: rt.tape_unpack((torch.zeros(4, 64, dtype=U8), codes()[1]), F), cuda.ERR_ARG),
    "unpack: too few exponents": (lambda rt: rt.tape_unpack((codes()[0], codes(4, 32)[1]), F), cuda.ERR_SHAPE),
    "unpack: codes with gaps": (lambda rt: rt.tape_unpack((codes(4, 128)[0][:, :64], codes()[1]), F), cuda.ERR_SHAPE),
    "unpack: to integers": (lambda rt: rt.tape_unpack(codes(), torch.int32), cuda.ERR_ARG),
    "norm: f32 weights": (lambda rt: rt.tape_layer_norm(torch.zeros(4, 64), torch.zeros(64), torch.zeros(64, dtype=H)), cuda.ERR_ARG),
    "norm: short bias": (lambda rt: rt.tape_layer_norm(torch.zeros(4, 64), torch.zeros(64, dtype=H), torch.zeros(63, dtype=H)),
                         cuda.ERR_SHAPE),
    "norm backward: rows": (lambda rt: rt.tape_layer_norm_backward(codes(), torch.zeros(5, 64), torch.zeros(64, dtype=H)),
                            cuda.ERR_SHAPE),
    "norm backward: residual's type": (lambda rt: rt.tape_layer_norm_backward(
        codes(), torch.zeros(4, 64), torch.zeros(64, dtype=H), residual=torch.zeros(4, 64, dtype=H)), cuda.ERR_ARG),
    "weight gradient: f32": (lambda rt: rt.tape_weight_grad(codes(), torch.zeros(4, 8)), cuda.ERR_ARG),
    "weight gradient: rows": (lambda rt: rt.tape_weight_grad(codes(), torch.zeros(3, 8, dtype=H)), cuda.ERR_SHAPE),
    "head: f32": (lambda rt: rt.head_ce_grad(torch.zeros(4, 64), torch.zeros(9, 64), labels(4)), cuda.ERR_ARG),
    "head: labels": (lambda rt: rt.head_ce_grad(hidden(), dense(), labels(5)), cuda.ERR_SHAPE),
    "head: 64-bit labels": (lambda rt: rt.head_ce_grad(hidden(), dense(), labels(4).long()), cuda.ERR_ARG),
    "head: time": (lambda rt: rt.head_ce_grad(hidden(), dense(), labels(4), time=3), cuda.ERR_SHAPE),
    "head: no time": (lambda rt: rt.head_ce_grad(hidden(), dense(), labels(4), time=0), cuda.ERR_SHAPE),
    "head: channels": (lambda rt: rt.head_ce_grad(hidden(), dense(9, 32), labels(4)), cuda.ERR_SHAPE),
    "head: transposed weights": (lambda rt: rt.head_ce_grad(hidden(), dense(64, 9).t(), labels(4)), cuda.ERR_SHAPE),
    "head: weight's type": (lambda rt: rt.head_ce_grad(hidden(), dense().bfloat16(), labels(4)), cuda.ERR_ARG),
    "head: packed without scales": (lambda rt: rt.head_ce_grad(hidden(), torch.zeros(18, dtype=torch.int32), labels(4)), cuda.ERR_ARG),
    "head: too few words": (lambda rt: rt.head_ce_grad(hidden(), torch.zeros(17, dtype=torch.int32), labels(4),
                                                       scale=torch.zeros(9, dtype=H)), cuda.ERR_SHAPE),
    "head: bias": (lambda rt: rt.head_ce_grad(hidden(), dense(), labels(4), bias=torch.zeros(8, dtype=H)), cuda.ERR_SHAPE),
    "head: bias's type": (lambda rt: rt.head_ce_grad(hidden(), dense(), labels(4), bias=torch.zeros(9)), cuda.ERR_ARG),
    "head: ignore_id": (lambda rt: rt.head_ce_grad(hidden(), dense(), labels(4), ignore_id=1 << 32), cuda.ERR_ARG),
    "norm backward: residual's rows": (lambda rt: rt.tape_layer_norm_backward(
        codes(), torch.zeros(4, 64), torch.zeros(64, dtype=H), residual=torch.zeros(3, 64)), cuda.ERR_SHAPE),
}


class Taking(Fake):
    """Every call of the library succeeds; the last one's arguments are kept."""

    class _Lib:
        def __getattr__(self, name):
            def call(*arguments):
                Taking.arguments = arguments
                return cuda.OK
            return call

    _lib = _Lib()

    def _check(self, rc):
        assert rc == cuda.OK


@pytest.mark.parametrize("shape,time", [((3, 0, 64), 1), ((0, 5, 64), 5), ((0, 64), 1), ((3, 4, 64), 4), ((12, 64), 12)])
def test_the_time_that_a_shape_gives(monkeypatch, shape, time):
    """Zero rows are no error, whichever of the leading sizes is 0."""
    device._torch()
    monkeypatch.setattr(device, "_RAW_STREAM", lambda d: 0)
    rows = shape[0] if len(shape) == 2 else shape[0] * shape[1]
    r = Taking().head_ce_grad(torch.zeros(shape, dtype=H), dense(), torch.zeros(shape[:-1], dtype=torch.int32))
    assert Taking.arguments[11:14] == (rows, time, 64) and rows % time == 0
    assert r.hidden.shape == shape and r.row_loss.shape == (rows,) and r.weight.shape == (9, 64)


@pytest.mark.parametrize("call,code", REFUSED.values(), ids=REFUSED.keys())
def test_refused_before_the_library_is_called(call, code):
    with pytest.raises(cuda.UllisCudaError) as e:
        call(Fake())
    assert e.value.code == code
