"""The 8-bit tape and LayerNorm over it (CudaRuntime.tape_*) against plain implementations in 64 bits.

Codes and exponents are exact.  For sums in f32 the tolerances count roundings: a sum of n terms is off by at most
n * 2^-24 * sum |terms|, and what leaves in 16 bits by half a step more."""
import pytest
import torch

from ullis_b200 import cuda

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def plain_tape(x):
    """(codes, exponent bytes, values in 64 bits) by the definition."""
    rows, c = x.shape
    b = torch.nn.functional.pad(x.double(), (0, -c % 32)).reshape(rows, -1, 32)
    finite = torch.isfinite(b).all(2, keepdim=True)
    top = torch.where(finite, b, 0.0).abs().amax(2, keepdim=True)
    e = torch.full_like(top, -126.0)
    for k in range(-125, 122):
        e = torch.where(127.0 * 2.0 ** (k - 1) < top, torch.full_like(e, float(k)), e)
    step = torch.exp2(e)
    codes = torch.where(finite, torch.round(b / step).clamp(-127, 127), 0.0)
    values = torch.where(finite, codes * step, torch.nan)
    byte = torch.where(finite, e + 127, 255.0)
    return codes.reshape(rows, -1)[:, :c].to(torch.int8), byte[:, :, 0].to(torch.uint8), values.reshape(rows, -1)[:, :c]


def activations(rows, c, dtype, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)
    size = torch.exp(torch.randn(c, generator=g, device="cuda"))
    return (torch.randn(rows, c, generator=g, device="cuda") * size).to(dtype)


SHAPES = [(1, 1), (1, 32), (3, 7), (5, 31), (4, 33), (130, 64), (9, 100), (3, 256), (7, 264), (64, 512), (5, 1000), (33, 1024),
          (3, 2048), (2, 2056), (3, 4096), (2, 8191), (2, 8192), (1, 20000)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_pack_and_unpack(cuda_rt, shape, dtype):
    x = activations(*shape, TYPES[dtype])
    codes, byte, values = plain_tape(x)
    tape = cuda_rt.tape_pack(x)
    assert torch.equal(tape.codes, codes) and torch.equal(tape.exponents, byte)
    for to in TYPES.values():
        back = cuda_rt.tape_unpack(tape, to)
        assert back.dtype == to and torch.equal(back, values.to(to))


def test_values_that_a_block_hardly_holds(cuda_rt):
    tiny, huge = 2.0 ** -149, 3.4028234e38
    rows = [[0.0], [tiny], [2.0 ** -126, -tiny], [huge, -huge, 1.0], [127.0, 126.5, -126.5, 0.5], [127.5, 127.0, 63.5],
            [float("inf"), 1.0], [1.0, float("nan")], [-float("inf")], [65504.0, 1e-8]]
    x = torch.zeros(len(rows), 40, device="cuda")
    for i, r in enumerate(rows):
        x[i, 4:4 + len(r)] = torch.tensor(r)
        x[i, 33] = 1.0                       # the neighbouring block is not touched by what this one holds
    codes, byte, values = plain_tape(x)
    tape = cuda_rt.tape_pack(x)
    assert torch.equal(tape.codes, codes) and torch.equal(tape.exponents, byte)
    back = cuda_rt.tape_unpack(tape, torch.float32)
    assert torch.equal(torch.nan_to_num(back, nan=7.0), torch.nan_to_num(values, nan=7.0).float())
    assert torch.equal(torch.isnan(back).any(1), torch.tensor([i in (6, 7, 8) for i in range(len(rows))], device="cuda"))
    assert (back[:, 33] == 1.0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offset,stride", [(0, 96), (1, 101), (8, 72), (3, 64)])
def test_rows_with_gaps_and_odd_starts(cuda_rt, dtype, offset, stride):
    base = torch.randn(40 * stride + offset, device="cuda").to(TYPES[dtype])
    x = base[offset:].as_strided((37, 64), (stride, 1), base.storage_offset() + offset)
    codes, byte, values = plain_tape(x)
    tape = cuda_rt.tape_pack(x)
    assert torch.equal(tape.codes, codes) and torch.equal(tape.exponents, byte)
    w, b = torch.ones(64, device="cuda").half(), torch.zeros(64, device="cuda").half()
    y, tape2 = cuda_rt.tape_layer_norm(x, w, b)
    y3, _ = cuda_rt.tape_layer_norm(x.contiguous(), w, b)
    assert torch.equal(tape2.codes, codes) and torch.equal(y, y3)
    got = cuda_rt.tape_layer_norm_backward(tape, x, w, residual=x)
    want = cuda_rt.tape_layer_norm_backward(tape, x.contiguous(), w, residual=x.contiguous())
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def normed(x):
    mean = x.mean(1, keepdim=True)
    inv = 1.0 / torch.sqrt((x - mean).square().mean(1, keepdim=True) + 1e-5)
    return (x - mean) * inv, inv


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [s for s in SHAPES if s[1] <= 8192] + [(2500, 512), (700, 264)], ids=str)
def test_layer_norm_and_its_backward_pass(cuda_rt, shape, dtype):
    rows, c = shape
    t = TYPES[dtype]
    half = torch.finfo(t).eps / 2 if t != torch.float32 else 0.0
    x = activations(rows, c, t, 1)
    gy, residual = activations(rows, c, t, 2), activations(rows, c, t, 3)
    w = (1.0 + 0.1 * torch.randn(c, device="cuda")).half()
    b = (0.1 * torch.randn(c, device="cuda")).half()
    y, tape = cuda_rt.tape_layer_norm(x, w, b)
    codes, byte, kept = plain_tape(x)
    assert torch.equal(tape.codes, codes) and torch.equal(tape.exponents, byte)
    wd, bd = w.double(), b.double()
    # a lane adds 16 values, then the lanes and the warps: 16 + 5 + 16 steps; the mean's error counts in every value and, through
    # the variance, in 1 / deviation; 8 more roundings from there to y
    n = 48
    xd = x.double()
    xh, inv = normed(xd)
    reach = (xd.abs().amax(1, keepdim=True) + xd.abs().mean(1, keepdim=True)) * inv
    want = xh * wd + bd
    tol = half * want.abs() + U * n * ((reach + xh.abs()) * (1 + xh.abs()) * wd.abs() + bd.abs()) + 1e-7 * half
    assert ((y.double() - want).abs() <= tol).all()

    xh, inv = normed(kept)
    reach = (kept.abs().amax(1, keepdim=True) + kept.abs().mean(1, keepdim=True)) * inv
    off = U * n * (reach + xh.abs()) * (1 + xh.abs())          # of xh
    g, dx = gy.double(), gy.double() * wd
    for res in (None, residual):
        gx, gw, gb = cuda_rt.tape_layer_norm_backward(tape, gy, w, residual=res)
        assert gx.dtype == t and gw.dtype == gb.dtype == torch.float32
        add = 0.0 if res is None else res.double()
        s2 = (dx * xh).mean(1, keepdim=True)
        want = add + inv * (dx - dx.mean(1, keepdim=True) - xh * s2)
        s2_off = (dx.abs() * off).mean(1, keepdim=True) + U * n * (dx * xh).abs().mean(1, keepdim=True)
        tol = half * want.abs() + U * n * (dx.abs() * inv * (1 + reach) + inv * dx.abs().mean(1, keepdim=True) * (1 + reach)) + \
            inv * (off * s2.abs() + xh.abs() * s2_off + U * n * (xh * s2).abs() * (1 + reach)) + U * 4 * (want.abs() + abs(add)) + 1e-7 * half
        assert ((gx.double() - want).abs() <= tol).all()
        terms = 64 + rows / 8      # a thread's rows, then the CTA's and the CTAs'
        assert ((gw.double() - (g * xh).sum(0)).abs() <= (g.abs() * off + U * terms * (g * xh).abs()).sum(0)).all()
        assert ((gb.double() - g.sum(0)).abs() <= U * terms * g.abs().sum(0)).all()


def test_gradient_against_differences(cuda_rt):
    """gx by differences of a loss of the normed values, in 64 bits, at what the tape stands for."""
    rows, c = 3, 40
    x = activations(rows, c, torch.float32, 5)
    w, b = torch.randn(c, device="cuda").half(), torch.randn(c, device="cuda").half()
    gy = torch.randn(rows, c, device="cuda")
    tape = cuda_rt.tape_pack(x)
    kept = cuda_rt.tape_unpack(tape, torch.float32).double()

    def loss(v):
        return ((normed(v)[0] * w.double() + b.double()) * gy.double()).sum()

    gx = cuda_rt.tape_layer_norm_backward(tape, gy, w)[0].double()
    for r, i in [(0, 0), (1, 17), (2, 39), (2, 32)]:
        d = torch.zeros_like(kept)
        d[r, i] = 1e-4
        slope = (loss(kept + d) - loss(kept - d)) / 2e-4
        assert abs(slope - gx[r, i]) <= 1e-5 * gx[r].abs().max() + 1e-6


def test_zero_rows(cuda_rt):
    x = torch.empty(0, 64, device="cuda")
    w = torch.ones(64, device="cuda").half()
    y, tape = cuda_rt.tape_layer_norm(x, w, w)
    assert y.shape == (0, 64) and tape.codes.shape == (0, 64) and tape.exponents.shape == (0, 2)
    assert cuda_rt.tape_pack(x).codes.shape == (0, 64) and cuda_rt.tape_unpack(tape, torch.float16).shape == (0, 64)
    gx, gw, gb = cuda_rt.tape_layer_norm_backward(tape, x, w)
    assert gx.shape == (0, 64) and not gw.any() and not gb.any() and gw.shape == gb.shape == (64,)


def test_leading_dimensions_and_other_streams(cuda_rt):
    x = activations(60, 96, torch.bfloat16).reshape(3, 20, 96)
    w = torch.ones(96, device="cuda").half()
    want, tape = cuda_rt.tape_layer_norm(x.reshape(60, 96), w, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y, tape2 = cuda_rt.tape_layer_norm(x, w, w)
        gx, _, _ = cuda_rt.tape_layer_norm_backward(tape2, y, w, residual=x)
        back = cuda_rt.tape_unpack(tape2, torch.bfloat16)
    torch.cuda.current_stream().wait_stream(side)
    assert y.shape == gx.shape == back.shape == x.shape
    assert torch.equal(y.reshape(60, 96), want) and torch.equal(tape2.codes.reshape(60, 96), tape.codes)


def test_two_graphs_replayed_at_once(cuda_rt):
    """Captured calls have workspaces of their own: replays on two streams side by side give what eager calls give."""
    w = torch.ones(512, device="cuda").half()
    data = [(activations(3000, 512, torch.float32, s), activations(3000, 512, torch.float32, s + 9)) for s in (1, 2)]
    want = []
    for x, gy in data:
        want.append(cuda_rt.tape_layer_norm_backward(cuda_rt.tape_pack(x), gy, w, residual=x))
    torch.cuda.synchronize()
    graphs, got = [], []
    for x, gy in data:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got.append(cuda_rt.tape_layer_norm_backward(cuda_rt.tape_pack(x), gy, w, residual=x))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_gx_in_the_place_of_the_other_gradient(cuda_rt):
    """The C entry point takes residual for gx."""
    import ctypes as C
    for dtype, code in ((torch.float32, 0), (torch.bfloat16, 2)):
        for rows, c in ((3000, 512), (37, 100), (9, 2048)):
            x, gy = activations(rows, c, dtype, 1), activations(rows, c, dtype, 2)
            res, w = activations(rows, c, dtype, 3), torch.ones(c, device="cuda").half()
            tape = cuda_rt.tape_pack(x)
            want = cuda_rt.tape_layer_norm_backward(tape, gy, w, residual=res)
            g = torch.empty(2, c, device="cuda")
            need = C.c_size_t(0)
            assert cuda_rt._lib.ullis_cuda_tape_layer_norm_backward_workspace(cuda_rt._h, rows, c, C.byref(need)) == cuda.OK
            work = torch.empty(need.value, dtype=torch.uint8, device="cuda")
            fn = cuda_rt._lib.ullis_cuda_tape_layer_norm_backward
            stream = torch.cuda.current_stream().cuda_stream
            args = (tape.codes.data_ptr(), tape.exponents.data_ptr(), gy.data_ptr(), c, w.data_ptr(), res.data_ptr())
            end = (rows, c, res.data_ptr(), g[0].data_ptr(), g[1].data_ptr(), work.data_ptr())
            assert fn(cuda_rt._h, stream, code, *args, c + 8, *end, need) == cuda.ERR_ARG      # rows that do not lie on one another
            assert fn(cuda_rt._h, stream, code, *args, c, *end, C.c_size_t(need.value - 1)) == cuda.ERR_SHAPE
            assert fn(cuda_rt._h, stream, code, *args, c, *end, need) == cuda.OK
            assert torch.equal(res, want[0]) and torch.equal(g[0], want[1]) and torch.equal(g[1], want[2])


def test_offsets_past_32_bits(cuda_rt):
    c, stride = 96, 2 ** 32 + 16
    base = torch.empty(stride + c, dtype=torch.bfloat16, device="cuda")
    x = base.as_strided((2, c), (stride, 1))
    x.copy_(activations(2, c, torch.bfloat16))
    codes, byte, _ = plain_tape(x.contiguous())
    tape = cuda_rt.tape_pack(x)
    assert torch.equal(tape.codes, codes) and torch.equal(tape.exponents, byte)


def test_more_than_2_to_the_32_elements(cuda_rt):
    """Rows at both ends as a call of those rows alone has them; the sums over rows have nothing of the others, whose gy is 0."""
    rows, c, t = 2 ** 22 + 128, 1032, torch.bfloat16
    g = torch.Generator("cuda").manual_seed(3)
    x, gy, past = (torch.randn(256, c, generator=g, device="cuda").to(t) for _ in range(3))
    w = (1 + 0.1 * torch.randn(c, generator=g, device="cuda")).half()
    ends = torch.cat([torch.arange(128), torch.arange(rows - 128, rows)]).cuda()
    big_x, big_gy = torch.ones(rows, c, dtype=t, device="cuda"), torch.zeros(rows, c, dtype=t, device="cuda")
    big_x[ends], big_gy[ends] = x, gy
    y, tape = cuda_rt.tape_layer_norm(big_x, w, w)
    big_x[ends] = past
    got = cuda_rt.tape_layer_norm_backward(tape, big_gy, w, residual=big_x)
    small_y, small_tape = cuda_rt.tape_layer_norm(x, w, w)
    want = cuda_rt.tape_layer_norm_backward(small_tape, gy, w, residual=past)
    assert torch.equal(y[ends], small_y) and torch.equal(tape.codes[ends], small_tape.codes)
    assert torch.equal(tape.exponents[ends], small_tape.exponents) and torch.equal(got[0][ends], want[0])
    # 256 terms gy * xh, |xh| < 8, in two orders, each sum off by 2^-24 of its terms' sizes per addition
    for a, b in zip(got[1:], want[1:]):
        assert ((a - b).abs() <= 2 * 256 * 2.0 ** -24 * 8 * gy.float().abs().sum(0)).all()
    assert torch.equal(cuda_rt.tape_unpack(tape, t)[ends], cuda_rt.tape_unpack(small_tape, t))
    packed = cuda_rt.tape_pack(big_x)
    assert torch.equal(packed.codes[ends], cuda_rt.tape_pack(past).codes)


def test_refusals_of_the_library(cuda_rt):
    x = torch.zeros(2, 9000, device="cuda")
    w = torch.zeros(9000, device="cuda").half()
    with pytest.raises(cuda.UllisCudaError) as e:
        cuda_rt.tape_layer_norm(x, w, w)
    assert e.value.code == cuda.ERR_SHAPE and "8192" in e.value.message
    with pytest.raises(cuda.UllisCudaError) as e:
        cuda_rt.tape_layer_norm_backward(cuda_rt.tape_pack(x), x, w)
    assert e.value.code == cuda.ERR_SHAPE
    import ctypes as C
    call = cuda_rt._lib.ullis_cuda_tape_pack
    buf = C.c_void_p(x.data_ptr())
    for args, code in (((7, buf, 64, 2, 64, buf, buf), cuda.ERR_ARG), ((0, None, 64, 2, 64, buf, buf), cuda.ERR_ARG),
                       ((0, buf, 63, 2, 64, buf, buf), cuda.ERR_SHAPE), ((0, buf, 64, 2, 0, buf, buf), cuda.ERR_SHAPE),
                       ((0, C.c_void_p(x.data_ptr() + 2), 64, 2, 64, buf, buf), cuda.ERR_ARG)):
        dtype, px, stride, rows, channels, pc, pe = args
        rc = call(cuda_rt._h, None, C.c_int32(dtype), px, C.c_size_t(stride), C.c_size_t(rows), C.c_size_t(channels), pc, pe)
        assert rc == code
    assert not x.any()
