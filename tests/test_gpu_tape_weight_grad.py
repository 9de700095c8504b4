"""CudaRuntime.tape_weight_grad against the product in 64 bits.  Products of 16-bit numbers and codes are exact in f32; within 1024
rows the tensor cores cut off each addition (2^-23 per term), everything else is added with rounding (2^-24)."""
import ctypes as C

import pytest
import torch

from ullis_b200 import cuda

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def tape_of(rows, c, seed=0, spread=1.0):
    g = torch.Generator("cuda").manual_seed(seed)
    size = torch.exp(spread * torch.randn(rows, -(-c // 32), generator=g, device="cuda"))
    codes = torch.randint(-127, 128, (rows, c), generator=g, device="cuda").to(torch.int8)
    exponents = (torch.floor(torch.log2(size)) + 120).to(torch.uint8)
    return codes, exponents


def values(codes, exponents):
    e = torch.exp2(exponents.double() - 127.0)
    e = torch.where(exponents == 255, torch.nan, e)
    return codes.double() * e.repeat_interleave(32, 1)[:, : codes.shape[1]]


def check(got, gy, tape):
    x, g = values(*tape), gy.double()
    want, sizes = g.t() @ x, g.abs().t() @ x.abs()
    rows = gy.shape[0]
    off = U * (2 * min(rows, 1024) + 32 + rows / 1024) * sizes
    assert got.dtype == torch.float32 and ((got.double() - want).abs() <= off).all()


CASES = [(1, 1, 1), (1, 64, 200), (3, 33, 7), (63, 64, 64), (64, 256, 256), (65, 250, 1000), (333, 512, 96), (1024, 100, 300),
         (1025, 520, 264), (3000, 2048, 64), (5000, 129, 2050), (16384, 64, 8), (20000, 512, 512)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", CASES, ids=str)
def test_the_product(cuda_rt, case, dtype):
    rows, i, o = case
    tape = tape_of(rows, i, rows)
    gy = (1e-2 * torch.randn(rows, o, device="cuda")).to(TYPES[dtype])
    check(cuda_rt.tape_weight_grad(tape, gy), gy, tape)


def test_terms_of_one_sign(cuda_rt):
    """What the tensor cores cut off adds up where all terms have one sign."""
    codes, exponents = tape_of(16384, 128, 3)
    tape = codes.abs(), exponents
    gy = torch.rand(16384, 64, device="cuda").half()
    got = cuda_rt.tape_weight_grad(tape, gy)
    want = gy.double().t() @ values(*tape)
    assert (got.double() - want).norm() <= 1.5e-5 * want.norm()      # 64 accumulations of 16 terms: 64 * 2^-23 at most, and roundings


@pytest.mark.parametrize("dtype", TYPES)
def test_what_is_cut_off_does_not_grow_with_the_rows(cuda_rt, dtype):
    """Sums of one sign over 512 rows, and over 32 times as many: no more than 512 terms are added up without rounding, so what is lost
    of a sum is what is lost of its parts.  Their 32 additions are off by 2^-25 each, up and down."""
    lost = []
    for rows in (512, 16384):
        codes, exponents = tape_of(rows, 512, 3)
        gy = torch.rand(rows, 512, device="cuda").to(TYPES[dtype])
        want = gy.double().t() @ values(codes.abs(), exponents)
        got = cuda_rt.tape_weight_grad((codes.abs(), exponents), gy)
        lost.append(((want - got.double()) / want).mean().item())
    assert 0.0 < lost[1] <= 1.25 * lost[0] + 2.0 ** -24, lost


@pytest.mark.parametrize("dtype", TYPES)
def test_blocks_of_every_exponent(cuda_rt, dtype):
    """A block's exponents 30 binades apart lose nothing in FP16; blocks of very different size do not meet."""
    codes, _ = tape_of(512, 160, 1)
    g = torch.Generator("cuda").manual_seed(2)
    exponents = torch.empty(512, 5, dtype=torch.uint8, device="cuda")
    for b, base in enumerate((1, 40, 127, 180, 215)):
        exponents[:, b] = (base + torch.randint(0, 31, (512,), generator=g, device="cuda")).to(torch.uint8)
    gy = (1e-2 * torch.randn(512, 72, device="cuda")).to(TYPES[dtype])
    tape = codes, exponents
    x = values(*tape)
    got = cuda_rt.tape_weight_grad(tape, gy).double()
    want, sizes = gy.double().t() @ x, gy.double().abs().t() @ x.abs()
    assert ((got - want).abs() <= U * 1100 * sizes + 2.0 ** -149 * 512).all()


def close(got, gy, tape):
    """512 terms at a time with what the tensor cores cut off; then those sums with rounding, at most two for 512 rows (gy in two
    parts, the smaller one below 2^-8 of the other: 1 + 2^-7 times the sizes)."""
    rows = gy.shape[0]
    want, sizes = gy.double().t() @ values(*tape), gy.double().abs().t() @ values(*tape).abs()
    off = (1 + 2.0 ** -7) * U * (2 * min(rows, 512) + 32 + 2 * rows / 512) * sizes + 2.0 ** -149 * rows
    bad = ~((got.double() - want).abs() <= off)
    assert not bad.any(), (int(bad.sum()), got[bad][:4].tolist(), want[bad][:4].tolist(), off[bad][:4].tolist())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", [(300, 96, 72), (300, 70, 7), (2100, 264, 300), (20000, 64, 8)], ids=str)
def test_a_row_far_above_the_others(cuda_rt, case, dtype):
    """What a row of very large values holds has no effect where its gy is 0, and no more than its own where gy is not."""
    rows, i, o = case
    g = torch.Generator("cuda").manual_seed(4)
    codes, exponents = tape_of(rows, i, 2)
    gy = (1e-2 * torch.randn(rows, o, generator=g, device="cuda")).to(TYPES[dtype])
    for binades, at in ((33, 0), (45, rows - 1), (70, rows // 2), (100, 17)):
        high = exponents.clone()
        high[at] += binades
        masked = gy.clone()
        masked[at] = 0.0
        got = cuda_rt.tape_weight_grad((codes, high), masked)
        close(got, masked, (codes, high))
        assert got.abs().min() > 0.0
        masked[at, ::3] = 6e-5                   # the other outputs still have nothing of that row
        close(cuda_rt.tape_weight_grad((codes, high), masked), masked, (codes, high))


@pytest.mark.parametrize("dtype", TYPES)
def test_exponents_all_over(cuda_rt, dtype):
    """Every exponent of a tape in one block, beside a block that 16 bits hold and one that lies at the range's end."""
    g = torch.Generator("cuda").manual_seed(6)
    codes = torch.randint(-127, 128, (1500, 100), generator=g, device="cuda").to(torch.int8)
    exponents = torch.randint(1, 249, (1500, 4), generator=g, device="cuda").to(torch.uint8)
    exponents[:, 1] = 130
    exponents[:, 3] = torch.where(exponents[:, 3] > 120, 248, 216).to(torch.uint8)
    gy = (2.0 ** -10 * torch.randn(1500, 300, generator=g, device="cuda")).to(TYPES[dtype])
    close(cuda_rt.tape_weight_grad((codes, exponents), gy), gy, (codes, exponents))
    # rows of nothing, whose exponent is the lowest, take no block out of 16 bits
    codes[::2], exponents[::2], exponents[1::2] = 0, 1, 130
    got = cuda_rt.tape_weight_grad((codes, exponents), gy)
    close(got, gy, (codes, exponents))
    exponents[::2] = 130
    assert torch.equal(got, cuda_rt.tape_weight_grad((codes, exponents), gy))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offset,stride", [(0, 136), (3, 136), (0, 131)])
def test_far_values_in_a_few_blocks(cuda_rt, offset, stride, dtype):
    """Some stretches of some columns need more than FP16, their neighbours do not; and gy may have to be copied."""
    codes, exponents = tape_of(3000, 600, 3)
    exponents[1100, 2] += 60                     # rows 1024 .. 1535, columns 0 .. 255
    exponents[2999, 18] += 50                    # the last rows, the last columns
    base = torch.full((3000 * stride + offset + 130,), float("nan"), device="cuda").to(TYPES[dtype])
    gy = base.as_strided((3000, 130), (stride, 1), offset)
    gy.copy_(torch.randn(3000, 130, device="cuda"))
    gy[1100] = 0.0
    gy[2999, ::2] = 0.0
    got = cuda_rt.tape_weight_grad((codes, exponents), gy)
    close(got, gy, (codes, exponents))
    assert torch.equal(got, cuda_rt.tape_weight_grad((codes, exponents), gy.contiguous()))


@pytest.mark.parametrize("dtype", TYPES)
def test_codes_of_the_lowest_exponent(cuda_rt, dtype):
    """A block of zeros has it too: what is not 0 there counts where nothing else does."""
    codes, exponents = tape_of(100, 96, 8)
    gy = torch.zeros(100, 40, device="cuda").to(TYPES[dtype])
    exponents[41], gy[41] = 1, 1000.0
    codes[7], exponents[7] = 0, 1
    got = cuda_rt.tape_weight_grad((codes, exponents), gy)
    close(got, gy, (codes, exponents))
    assert torch.equal(got != 0, (codes[41] != 0).expand(40, 96))


def test_infinite_gradients_with_far_values(cuda_rt):
    """An infinity in gy is one in every product it is in, however gy is held: 0 times it is NaN, anything else infinite."""
    for high in (0, 60):
        codes, exponents = tape_of(200, 64, 8)
        codes[9, :4] = torch.tensor([0, 1, -1, 127], dtype=torch.int8)
        exponents[100] += high
        gy = (1e-2 * torch.randn(200, 8, device="cuda")).half()
        gy[9, 2], gy[9, 3] = float("inf"), -float("inf")
        got = cuda_rt.tape_weight_grad((codes, exponents), gy)
        inf = float("inf")
        assert torch.isnan(got[2:4, 0]).all()
        assert got[2, 1:4].tolist() == [inf, -inf, inf] and got[3, 1:4].tolist() == [-inf, inf, -inf]
        keep = torch.tensor([0, 1, 4, 5, 6, 7], device="cuda")
        close(got[keep], gy[:, keep], (codes, exponents))


def test_a_block_that_is_not_finite(cuda_rt):
    codes, exponents = tape_of(100, 96, 5)
    exponents[17, 1] = 255
    for dtype in TYPES.values():
        gy = torch.randn(100, 40, device="cuda").to(dtype)
        got = cuda_rt.tape_weight_grad((codes, exponents), gy)
        assert torch.isnan(got[:, 32:64]).all() and torch.isfinite(got[:, :32]).all() and torch.isfinite(got[:, 64:]).all()


@pytest.mark.parametrize("offset,stride", [(0, 104), (1, 97), (8, 96), (3, 96)])
def test_rows_with_gaps_and_odd_starts(cuda_rt, offset, stride):
    tape = tape_of(300, 64)
    base = torch.full((300 * stride + offset + 96,), float("nan"), device="cuda").half()
    gy = base.as_strided((300, 96), (stride, 1), offset)
    gy.copy_(torch.randn(300, 96, device="cuda"))
    got = cuda_rt.tape_weight_grad(tape, gy)
    assert torch.equal(got, cuda_rt.tape_weight_grad(tape, gy.contiguous()))
    check(got, gy, tape)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("inputs", [64, 63])
@pytest.mark.parametrize("rows,ranges", [(200, False), (20000, True)])
def test_an_output_that_starts_anywhere(cuda_rt, rows, ranges, inputs, dtype):
    """g at every offset into a buffer (the entry point asks for the alignment of its elements), with one range of K, which the product
    writes itself, and with several, whose sum is."""
    out = 40
    tape, gy = tape_of(rows, inputs, 1), torch.randn(rows, out, device="cuda").to(TYPES[dtype])
    want = cuda_rt.tape_weight_grad(tape, gy)
    size = C.c_size_t(0)
    assert cuda_rt._lib.ullis_cuda_tape_weight_grad_workspace(cuda_rt._h, rows, inputs, out, C.byref(size)) == cuda.OK
    work = torch.empty(size.value, dtype=torch.uint8, device="cuda")
    for offset in (0, 1, 2, 3):
        g = torch.full((out * inputs + 8,), 7.0, device="cuda")
        before = cuda_rt.launch_count
        assert cuda_rt._lib.ullis_cuda_tape_weight_grad(
            cuda_rt._h, torch.cuda.current_stream().cuda_stream, {"f16": 1, "bf16": 2}[dtype], tape[0].data_ptr(), tape[1].data_ptr(),
            gy.data_ptr(), out, rows, inputs, out, g.data_ptr() + 4 * offset, work.data_ptr(), size.value) == cuda.OK
        assert cuda_rt.launch_count - before == 2 + ranges          # operand, product, and the sum
        assert torch.equal(g[offset:offset + out * inputs].view(out, inputs), want)
        assert (g[:offset] == 7.0).all() and (g[offset + out * inputs:] == 7.0).all()


def test_zero_rows_and_leading_dimensions(cuda_rt):
    empty = torch.zeros(0, 64, dtype=torch.int8, device="cuda"), torch.zeros(0, 2, dtype=torch.uint8, device="cuda")
    got = cuda_rt.tape_weight_grad(empty, torch.zeros(0, 24, device="cuda").half())
    assert got.shape == (24, 64) and not got.any()
    x = torch.randn(3, 50, 64, device="cuda").half()
    gy = torch.randn(3, 50, 24, device="cuda").half()
    tape = cuda_rt.tape_pack(x)
    assert tape.codes.shape == (3, 50, 64)
    flat = tape.codes.reshape(150, 64), tape.exponents
    assert torch.equal(cuda_rt.tape_weight_grad(tape, gy), cuda_rt.tape_weight_grad(flat, gy.reshape(150, 24)))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", [(70, 40, 30), (5000, 100, 300), (20000, 512, 512)], ids=str)
def test_nothing_depends_on_what_the_workspace_held(cuda_rt, case, dtype):
    rows, i, o = case
    tape, gy = tape_of(rows, i, 1), torch.randn(rows, o, device="cuda").to(TYPES[dtype])
    want = cuda_rt.tape_weight_grad(tape, gy)
    for byte in (0xFF, 0x7B):     # NaN; large numbers
        torch.cuda.empty_cache()
        dirt = torch.full((1 << 29,), byte, dtype=torch.uint8, device="cuda")
        del dirt                  # the next blocks come out of it
        assert torch.equal(cuda_rt.tape_weight_grad(tape, gy), want)


@pytest.mark.parametrize("dtype", TYPES)
def test_a_graph_replayed_with_other_inputs(cuda_rt, dtype):
    """Which stretches need more than FP16 is known on the device only; and whatever lies in the workspace, nothing of it shows."""
    def inputs(seed, far):
        codes, exponents = tape_of(1400, 264, seed)
        exponents[600] += far                    # rows 512 .. 1023
        gy = torch.randn(1400, 96, device="cuda").to(TYPES[dtype])
        gy[600] = 0.0
        return [codes, exponents, gy]

    cases = [inputs(1, 0), inputs(2, 60), inputs(3, 0)]
    want = [cuda_rt.tape_weight_grad((c, e), gy) for c, e, gy in cases]
    held = [t.clone() for t in cases[0]]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = cuda_rt.tape_weight_grad((held[0], held[1]), held[2])
        dirt = torch.full((1 << 26,), 0xFF, dtype=torch.uint8, device="cuda")   # over what the call gave back
    for k in (0, 1, 2, 1, 1, 0):
        for t, v in zip(held, cases[k]):
            t.copy_(v)
        g.replay()
        assert torch.equal(got, want[k])
        close(got, cases[k][2], cases[k][:2])
    del dirt


def test_calls_on_two_streams_at_once(cuda_rt):
    tape = [tape_of(9000, 512, seed) for seed in (1, 2)]
    tape[1][1][77] += 60
    gy = [torch.randn(9000, 384, device="cuda").half() for _ in range(2)]
    gy[1][77] = 0.0
    want = [cuda_rt.tape_weight_grad(t, g) for t, g in zip(tape, gy)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(8):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                got[k].append(cuda_rt.tape_weight_grad(tape[k], gy[k]))
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(x, want[k]) for x in got[k])
    cuda_rt.synchronize()


def test_norm_linear_and_head_together(cuda_rt):
    """Norm, linear and head of a small model from the 8-bit tape: every gradient as autograd gives it in 64 bits at the values that
    the tape keeps."""
    rows, time, d, vocab = 256, 64, 96, 500
    t = torch.bfloat16
    x = torch.randn(rows, d, device="cuda").to(t)
    nw = (1 + 0.1 * torch.randn(d, device="cuda")).half()
    nb = (0.1 * torch.randn(d, device="cuda")).half()
    lin = (torch.randn(d, d, device="cuda") / d ** 0.5).to(t)
    head = (0.05 * torch.randn(vocab, d, device="cuda")).to(t)
    labels = torch.randint(0, vocab, (rows,), device="cuda").to(torch.int32)
    y, tape_x = cuda_rt.tape_layer_norm(x, nw, nb)
    tape_y = cuda_rt.tape_pack(y)
    h = y @ lin.t()
    r = cuda_rt.head_ce_grad(h, head, labels, time=time)
    g_lin = cuda_rt.tape_weight_grad(tape_y, r.hidden)
    gy = (r.hidden.float() @ lin.float()).to(t)
    gx, gw, gb = cuda_rt.tape_layer_norm_backward(tape_x, gy, nw)

    kept = cuda_rt.tape_unpack(tape_x, torch.float32).double().requires_grad_()
    wd, bd = nw.double().requires_grad_(), nb.double().requires_grad_()
    ld = lin.double().requires_grad_()
    yd = torch.nn.functional.layer_norm(kept, (d,), wd, bd, 1e-5)
    hd = yd @ ld.t()
    z = hd @ head.double().t()
    loss = (torch.logsumexp(z, 1) - z.gather(1, torch.roll(labels, -1).long()[:, None])[:, 0])
    loss[torch.arange(rows, device="cuda") % time < time - 1].sum().backward()
    # 8-bit inputs, and four 16-bit roundings on the way: half a step of 2^-7 is the largest of them
    for name, got, want in (("x", gx, kept.grad), ("norm weight", gw, wd.grad), ("norm bias", gb, bd.grad), ("linear", g_lin, ld.grad)):
        assert (got.double() - want).norm() <= 4 * 2.0 ** -7 * want.norm(), name


def test_offsets_past_32_bits(cuda_rt):
    """More than 2^32 elements of both operands; what is not zero lies at both ends."""
    rows, i, o = 2 ** 22 + 128, 1030, 1040
    small, gy = tape_of(256, i), torch.randn(256, o, device="cuda").half()
    ends = torch.cat([torch.arange(128), torch.arange(rows - 128, rows)]).cuda()
    codes = torch.zeros(rows, i, dtype=torch.int8, device="cuda")
    exponents = torch.full((rows, small[1].shape[1]), 127, dtype=torch.uint8, device="cuda")
    big = torch.zeros(rows, o, dtype=torch.float16, device="cuda")
    codes[ends], exponents[ends], big[ends] = small[0], small[1], gy
    check(cuda_rt.tape_weight_grad((codes, exponents), big), gy, small)
