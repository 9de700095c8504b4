"""The entry points of the operators on device memory with every array one element into its buffer, inputs, outputs and tapes alike:
the header asks for the alignment of the elements and no more.  Against the same call on arrays as torch allocates them, which takes
the wide loads and stores.  What goes through sums may be contracted differently there: fewer than 16 roundings of 2^-24 of the largest
term per value, and as many per row in a sum over rows."""
import pytest
import torch

from ullis_b200 import cuda

pytestmark = pytest.mark.gpu

DTYPES = {"f32": (0, torch.float32), "f16": (1, torch.float16), "bf16": (2, torch.bfloat16)}
GUARD = 8


class Moved:
    """Flat copies and outputs that start one element into their buffers, which are checked for what was written beside them."""

    def __init__(self):
        self.buffers = []

    def like(self, t, fill=None):
        b = torch.full((t.numel() + 1 + GUARD,), 77, dtype=t.dtype, device="cuda")
        assert b.data_ptr() % 256 == 0
        self.buffers.append((b, t.numel()))
        return b[1:1 + t.numel()].view(t.shape)

    def copy(self, t):
        return None if t is None else self.like(t).copy_(t)

    def check(self):
        for b, n in self.buffers:
            assert b[0] == 77 and (b[1 + n:] == 77).all()


def p(t):
    return None if t is None else t.data_ptr()


def run(rt, name, *arguments, sizes=None):
    stream = torch.cuda.current_stream().cuda_stream
    work = ()
    if sizes is not None:
        import ctypes as C
        need = C.c_size_t(0)
        assert getattr(rt._lib, f"ullis_cuda_{name}_workspace")(rt._h, *sizes, C.byref(need)) == cuda.OK
        space = torch.full((need.value,), 0xFF, dtype=torch.uint8, device="cuda")
        work = (space.data_ptr(), need.value)
    rc = getattr(rt._lib, f"ullis_cuda_{name}")(rt._h, stream, *arguments, *work)
    assert rc == cuda.OK, rt._lib.ullis_cuda_last_error(rt._h)
    torch.cuda.synchronize()


def near(got, want, roundings=16, sizes=None):
    sizes = want.double().abs().max() if sizes is None else sizes
    step = torch.finfo(want.dtype).eps if want.dtype != torch.float32 else 0.0      # what was rounded to 16 bits may fall to the neighbour
    assert ((got.double() - want.double()).abs() <= roundings * 2.0 ** -24 * sizes + step * want.double().abs()).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,c", [(37, 64), (21, 520), (5, 2048)])
def test_tape_and_norm(cuda_rt, rows, c, dtype):
    code, t = DTYPES[dtype]
    g = torch.Generator("cuda").manual_seed(c)
    x = torch.randn(rows, c, generator=g, device="cuda").to(t)
    gy, past = (torch.randn(rows, c, generator=g, device="cuda").to(t) for _ in range(2))
    w, b = ((k + 0.1 * torch.randn(c, generator=g, device="cuda")).half() for k in (1.0, 0.0))
    y, tape = cuda_rt.tape_layer_norm(x, w, b)
    gx, gw, gb = cuda_rt.tape_layer_norm_backward(tape, gy, w, residual=past)
    m = Moved()
    mx, mw, mb, mgy, mpast = (m.copy(a) for a in (x, w, b, gy, past))
    codes, exponents = m.like(tape.codes), m.like(tape.exponents)
    run(cuda_rt, "tape_pack", code, p(mx), c, rows, c, p(codes), p(exponents))
    assert torch.equal(codes, tape.codes) and torch.equal(exponents, tape.exponents)
    back = m.like(x)
    run(cuda_rt, "tape_unpack", code, p(codes), p(exponents), rows, c, p(back), c)
    assert torch.equal(back, cuda_rt.tape_unpack(tape, t))
    codes.zero_(), exponents.zero_()
    my = m.like(y)
    run(cuda_rt, "tape_layer_norm", code, p(mx), c, p(mw), p(mb), rows, c, p(my), p(codes), p(exponents))
    assert torch.equal(codes, tape.codes) and torch.equal(exponents, tape.exponents)
    near(my, y)
    mgx, mgw, mgb = m.like(gx), m.like(gw), m.like(gb)
    run(cuda_rt, "tape_layer_norm_backward", code, p(codes), p(exponents), p(mgy), c, p(mw), p(mpast), c, rows, c, p(mgx), p(mgw), p(mgb),
        sizes=(rows, c))
    near(mgx, gx)
    near(mgw, gw, 16 * rows)
    near(mgb, gb, 16 * rows)
    m.check()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("rows,i,o,far", [(150, 64, 40, 0), (700, 264, 72, 0), (700, 264, 72, 50), (9000, 512, 512, 0)])
def test_weight_gradient(cuda_rt, rows, i, o, far, dtype):
    code, t = DTYPES[dtype]
    g = torch.Generator("cuda").manual_seed(rows)
    x, gy = torch.randn(rows, i, generator=g, device="cuda"), torch.randn(rows, o, generator=g, device="cuda").to(t)
    x[3] *= 2.0 ** far
    tape = cuda_rt.tape_pack(x)
    want = cuda_rt.tape_weight_grad(tape, gy)
    m = Moved()
    codes, exponents, mgy, got = m.copy(tape.codes), m.copy(tape.exponents), m.copy(gy), m.like(want)
    run(cuda_rt, "tape_weight_grad", code, p(codes), p(exponents), p(mgy), o, rows, i, o, p(got), sizes=(rows, i, o))
    assert torch.equal(got, want)
    m.check()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("packed", [True, False], ids=["packed", "dense"])
@pytest.mark.parametrize("rows,d,vocab", [(90, 64, 300), (1300, 512, 777), (300, 200, 20000)])
def test_head(cuda_rt, rows, d, vocab, packed, dtype):
    code, t = DTYPES[dtype]
    g = torch.Generator("cuda").manual_seed(vocab)
    hidden = torch.randn(rows, d, generator=g, device="cuda").to(t)
    labels = torch.randint(0, vocab, (rows,), generator=g, device="cuda").to(torch.int32)
    labels[::7] = -1
    bias = (0.1 * torch.randn(vocab, generator=g, device="cuda")).half()
    if packed:
        weight = torch.randint(-(1 << 31), 1 << 31, ((vocab * d + 31) // 32,), generator=g, device="cuda").to(torch.int32)
        scale = (0.01 + 0.01 * torch.rand(vocab, generator=g, device="cuda")).half()
    else:
        weight, scale = (0.0125 * torch.randn(vocab, d, generator=g, device="cuda")).to(t), None
    want = cuda_rt.head_ce_grad(hidden, weight, labels, scale=scale, bias=bias, ignore_id=-1)
    m = Moved()
    mh, mw, ml, ms, mb = (m.copy(a) for a in (hidden, weight, labels, scale, bias))
    got = [None if a is None else m.like(a) for a in want]
    run(cuda_rt, "head_ce_grad", code, p(mh), d, p(mw) if packed else None, None if packed else p(mw), p(ms), p(mb), p(ml), 0xFFFFFFFF, rows,
        rows, d, vocab, 1.0, *(p(a) for a in got), sizes=(rows, d, vocab, 1))
    for a, b in zip(got, want):
        assert (a is None and b is None) or torch.equal(a, b)
    m.check()
