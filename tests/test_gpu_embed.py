"""CudaRuntime.embed and embed_grad against their formulas in 64 bits.

Tolerances: a product with the scale is off by 2^-24, what leaves in 16 bits by half a step of its type; a sum of n terms in f32 by
fewer than n + 8 roundings of 2^-24 of the sum of the terms' sizes."""
import math

import pytest
import torch

from ullis_b200 import cuda

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
IGNORED = -1


def draw_tokens(rows, vocab, kind, g):
    if kind == "same":
        return torch.full((rows,), vocab // 2, dtype=torch.int32, device="cuda")
    u = torch.rand(rows, generator=g, device="cuda")
    t = u * vocab if kind == "even" else torch.exp(u * math.log(vocab)) - 1.0
    return t.clamp(0, vocab - 1).to(torch.int32)


def formula_grad(tokens, gy, vocab, scale):
    live = (tokens >= 0) & (tokens < vocab)
    at = torch.where(live, tokens, 0).long().reshape(-1)
    x = torch.where(live.reshape(-1, 1), gy.reshape(at.numel(), -1).double(), 0.0)
    g = torch.zeros(vocab, x.shape[1], dtype=torch.float64, device="cuda").index_add_(0, at, x)
    sizes = torch.zeros_like(g).index_add_(0, at, x.abs())
    n = torch.zeros(vocab, dtype=torch.float64, device="cuda").index_add_(0, at, live.reshape(-1).double())
    return g * scale, abs(scale) * (n[:, None] + 8) * U * sizes


def check_grad(got, tokens, gy, vocab, scale=1.0):
    want, off = formula_grad(tokens, gy, vocab, scale)
    assert got.dtype == torch.float32 and got.shape == want.shape
    bad = ~((got.double() - want).abs() <= off)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist(), got[bad][:4].tolist(), want[bad][:4].tolist())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("table_dtype", TYPES)
@pytest.mark.parametrize("rows,d,vocab", [(1, 1, 1), (1, 512, 8192), (7, 3, 5), (33, 100, 300), (513, 256, 8192), (4099, 130, 1001), (300, 8, 70000)])
def test_lookup(cuda_rt, rows, d, vocab, table_dtype, dtype):
    g = torch.Generator("cuda").manual_seed(rows + d)
    table = torch.randn(vocab, d, generator=g, device="cuda").to(TYPES[table_dtype])
    tokens = draw_tokens(rows, vocab, "even", g)
    tokens[rows // 2:: 5] = IGNORED
    tokens[rows // 3 + 1:: 7] = vocab
    scale = math.sqrt(d)
    y = cuda_rt.embed(table, tokens, scale=scale, dtype=TYPES[dtype], ignore_id=IGNORED)
    assert y.shape == (rows, d) and y.dtype == TYPES[dtype]
    live = (tokens >= 0) & (tokens < vocab)
    want = table[torch.where(live, tokens, 0).long()].double() * scale
    info = torch.finfo(TYPES[dtype])
    off = want.abs() * (info.eps / 2 + 2 * U) + info.smallest_normal * info.eps / 2
    assert ((y.double() - want).abs() <= off)[live].all()
    assert (y[tokens == IGNORED] == 0).all() and y[tokens == vocab].isnan().all()


def test_lookup_shapes_types_and_views(cuda_rt):
    g = torch.Generator("cuda").manual_seed(5)
    wide = torch.randn(100, 80, generator=g, device="cuda").half()
    tokens = torch.randint(0, 100, (3, 4, 5), generator=g, device="cuda").to(torch.int32)
    for at in (0, 1, 8):
        table = wide[:, at:at + 64]
        y = cuda_rt.embed(table, tokens)
        assert y.shape == (3, 4, 5, 64) and torch.equal(y, table[tokens.long()])
    assert cuda_rt.embed(wide, tokens[0, 0, 0]).shape == (80,)
    assert cuda_rt.embed(wide, tokens[:0]).shape == (0, 4, 5, 80)
    # the default ignore_id is the largest id
    assert (cuda_rt.embed(wide, torch.full((2,), -1, dtype=torch.int32, device="cuda")) == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["words", "same", "even"])
@pytest.mark.parametrize("rows,d,vocab", [
    (1, 1, 1), (1, 64, 3), (2, 5, 2), (31, 7, 100), (512, 256, 8192), (1023, 130, 50), (1024, 512, 3), (1025, 512, 3), (1500, 3, 5000),
    (2048, 64, 257), (2049, 100, 1000), (5000, 500, 700), (16384, 512, 8192), (32768, 40, 1021), (32769, 40, 1021), (70001, 24, 50021),
    (700, 2100, 40), (3000, 1100, 33),
])
def test_gradient(cuda_rt, rows, d, vocab, kind, dtype):
    g = torch.Generator("cuda").manual_seed(rows + d + vocab)
    tokens = draw_tokens(rows, vocab, kind, g)
    gy = torch.randn(rows, d, generator=g, device="cuda").to(TYPES[dtype])
    got = cuda_rt.embed_grad(tokens, gy, vocab, scale=1.5)
    check_grad(got, tokens, gy, vocab, 1.5)
    assert torch.equal(got, cuda_rt.embed_grad(tokens, gy, vocab, scale=1.5))


@pytest.mark.parametrize("rows,vocab", [(1500, (1 << 21) + 5), (1500, (1 << 21) - 3), (1500, (1 << 21) - 2), (1500, (1 << 21) - 1),
                                        (40000, 600_001), (40000, (1 << 19) - 2), (40000, (1 << 19) - 1), (60, 3_000_000)])
def test_gradient_of_large_tables(cuda_rt, rows, vocab):
    """Tokens whose sort keys need 64 bits, and those that just do not."""
    g = torch.Generator("cuda").manual_seed(rows)
    tokens = draw_tokens(rows, vocab, "even", g)
    tokens[:9] = vocab - 1
    tokens[9:20] = IGNORED
    gy = torch.randn(rows, 3, generator=g, device="cuda")
    check_grad(cuda_rt.embed_grad(tokens, gy, vocab), tokens, gy, vocab)


@pytest.mark.parametrize("rows", [300, 3000, 40000])
def test_rows_that_do_not_count(cuda_rt, rows):
    """Ignored tokens and tokens outside the table add nothing, whatever gy holds there."""
    g = torch.Generator("cuda").manual_seed(rows)
    tokens = draw_tokens(rows, 200, "words", g)
    gy = torch.randn(rows, 72, generator=g, device="cuda").half()
    out = torch.rand(rows, generator=g, device="cuda") < 0.4
    tokens = torch.where(out, torch.tensor([IGNORED, 200, 201, 1 << 30], device="cuda", dtype=torch.int32)[torch.arange(rows, device="cuda") % 4],
                         tokens)
    gy[out] = float("nan")
    clean = torch.where(out[:, None], torch.zeros_like(gy), gy)
    check_grad(cuda_rt.embed_grad(tokens, gy, 200), tokens, clean, 200)
    # an id of the table that is ignored
    got = cuda_rt.embed_grad(tokens, gy, 200, ignore_id=7)
    want = torch.where(tokens == 7, IGNORED, tokens)
    assert (got[7] == 0).all()
    check_grad(got, want, clean, 200)
    nothing = torch.full_like(tokens, IGNORED)
    assert (cuda_rt.embed_grad(nothing, torch.full_like(gy, float("inf")), 200) == 0).all()


def test_infinities_stay_with_their_token(cuda_rt):
    for rows in (500, 5000):
        tokens = (torch.arange(rows, device="cuda") % 11).to(torch.int32)
        gy = torch.ones(rows, 16, device="cuda")
        gy[4, 3], gy[15, 3], gy[6, 5] = float("inf"), -float("inf"), float("nan")
        got = cuda_rt.embed_grad(tokens, gy, 12)
        assert got[4, 3].isnan() and got[6, 5].isnan() and int((~got.isfinite()).sum()) == 2 and (got[11] == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [200, 6000])
def test_views_and_odd_starts(cuda_rt, rows, dtype):
    g = torch.Generator("cuda").manual_seed(rows)
    wide = torch.randn(rows, 160, generator=g, device="cuda").to(TYPES[dtype])
    tokens = draw_tokens(rows + 1, 90, "words", g)
    for at, d in ((0, 128), (8, 96), (1, 64), (3, 57)):
        gy = wide[:, at:at + d]
        check_grad(cuda_rt.embed_grad(tokens[1:], gy, 90), tokens[1:], gy.contiguous(), 90)
    cube = wide.view(2, rows // 2, 160)
    check_grad(cuda_rt.embed_grad(tokens[1:].view(2, -1), cube, 90), tokens[1:], wide, 90)


def test_zero_rows(cuda_rt):
    g = cuda_rt.embed_grad(torch.zeros(0, dtype=torch.int32, device="cuda"), torch.zeros(0, 24, device="cuda"), 9)
    assert g.shape == (9, 24) and (g == 0).all()


def test_the_library_writes_what_it_says_and_no_more(cuda_rt):
    """Outputs one element into their buffers, workspaces full of NaN."""
    import ctypes as C
    for rows, d, vocab in ((700, 36, 50), (2500, 36, 50), (9000, 512, 50)):
        g = torch.Generator("cuda").manual_seed(rows)
        tokens, gy = draw_tokens(rows, vocab, "words", g), torch.randn(rows, d, generator=g, device="cuda").half()
        table = torch.randn(vocab, d, generator=g, device="cuda").half()
        stream = torch.cuda.current_stream().cuda_stream
        for start in (1, 4):
            out = torch.full((vocab * d + 8,), 77.0, device="cuda")
            y = torch.full((rows * d + 8,), 77.0, device="cuda").half()
            need = C.c_size_t(0)
            assert cuda_rt._lib.ullis_cuda_embed_grad_workspace(cuda_rt._h, 1, rows, d, vocab, C.byref(need)) == cuda.OK
            work = torch.full((need.value,), 0xFF, dtype=torch.uint8, device="cuda")
            assert cuda_rt._lib.ullis_cuda_embed_grad(cuda_rt._h, stream, 1, tokens.data_ptr(), 0xFFFFFFFF, gy.data_ptr(), d, rows, d, vocab, 2.0,
                                                      out.data_ptr() + 4 * start, work.data_ptr(), need.value) == cuda.OK
            assert cuda_rt._lib.ullis_cuda_embed(cuda_rt._h, stream, 1, table.data_ptr(), d, tokens.data_ptr(), 0xFFFFFFFF, 1.0, rows, d, vocab, 1,
                                                 y.data_ptr() + 2 * start) == cuda.OK
            n = vocab * d
            assert (out[:start] == 77).all() and (out[start + n:] == 77).all()
            check_grad(out[start:start + n].view(vocab, d), tokens, gy, vocab, 2.0)
            assert (y[:start] == 77).all() and (y[start + rows * d:] == 77).all()
            assert torch.equal(y[start:start + rows * d].view(rows, d), table[tokens.long()])


def test_a_replayed_graph_and_two_streams(cuda_rt):
    """A captured call sorts the tokens that are there when it is replayed; two calls at once keep apart."""
    rows, d, vocab = 9000, 128, 400
    g = torch.Generator("cuda").manual_seed(1)
    tokens, gy = draw_tokens(rows, vocab, "words", g), torch.randn(rows, d, generator=g, device="cuda")
    table = torch.randn(vocab, d, generator=g, device="cuda")
    cuda_rt.embed_grad(tokens, gy, vocab)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = cuda_rt.embed(table, tokens)
        got = cuda_rt.embed_grad(tokens, gy, vocab)
    for kind in ("even", "same", "words"):
        tokens.copy_(draw_tokens(rows, vocab, kind, g))
        gy.normal_(generator=g)
        graph.replay()
        check_grad(got, tokens, gy, vocab)
        assert torch.equal(y, table[tokens.long()])
    others = [(draw_tokens(rows, vocab, "words", g), torch.randn(rows, d, generator=g, device="cuda"), torch.cuda.Stream()) for _ in range(2)]
    torch.cuda.synchronize()
    found = []
    for t, x, stream in others * 2:
        with torch.cuda.stream(stream):
            found.append(cuda_rt.embed_grad(t, x, vocab))
    torch.cuda.synchronize()
    for (t, x, _), f in zip(others * 2, found):
        check_grad(f, t, x, vocab)


def test_the_gradient_is_that_of_the_lookup(cuda_rt):
    """<gy, embed(table + h) - embed(table)> = <embed_grad(gy), h> (the lookup is linear)."""
    g = torch.Generator("cuda").manual_seed(8)
    table, h = (torch.randn(300, 48, generator=g, device="cuda") for _ in range(2))
    tokens, gy = draw_tokens(2000, 300, "words", g), torch.randn(2000, 48, generator=g, device="cuda")
    both = [cuda_rt.embed(t, tokens, scale=3.0).double() for t in (table + h, table)]
    left, right = (gy.double() * (both[0] - both[1])).sum(), (cuda_rt.embed_grad(tokens, gy, 300, scale=3.0).double() * h.double()).sum()
    # embed's outputs and table + h are rounded to f32, the sums of the gradient too
    sizes = (gy.double().abs() * (both[0].abs() + both[1].abs())).sum() + 2008 * (gy.double().abs() * 3.0 * h.double().abs()[tokens.long()]).sum()
    assert abs(left - right) <= 4 * U * sizes


@pytest.mark.parametrize("rows,vocab,kind", [(140_000, 3000, "words"), (300_001, 50, "even"), (300_001, 200_000, "words"), (131_073, 7, "same")])
def test_gradient_of_many_chunks(cuda_rt, rows, vocab, kind):
    """Rows in more chunks than a CTA holds the samples of at once, tokens with tens of thousands of rows."""
    g = torch.Generator("cuda").manual_seed(rows)
    tokens = draw_tokens(rows, vocab, kind, g)
    tokens[::1001] = IGNORED
    gy = torch.randn(rows, 12, generator=g, device="cuda").bfloat16()
    check_grad(cuda_rt.embed_grad(tokens, gy, vocab), tokens, gy, vocab)


@pytest.mark.parametrize("rows", [196_608, 196_609, 212_993, 262_144, 262_145, 600_001, (1 << 20) + 3])
@pytest.mark.parametrize("vocab,kind", [(3000, "words"), (1 << 20, "even"), (5, "same")])
def test_gradient_of_chunks_that_are_merged(cuda_rt, rows, vocab, kind):
    """Four to seven merges, the last runs with and without a partner; from one chunk fewer, which is not merged, on."""
    g = torch.Generator("cuda").manual_seed(rows)
    tokens = draw_tokens(rows, vocab, kind, g)
    tokens[::977] = IGNORED
    gy = torch.randn(rows, 4, generator=g, device="cuda").half()
    got = cuda_rt.embed_grad(tokens, gy, vocab)
    check_grad(got, tokens, gy, vocab)
    assert torch.equal(got, cuda_rt.embed_grad(tokens, gy, vocab))


def test_past_32_bits_of_elements(cuda_rt):
    """Tables, gradients and rows beyond 2^32 elements."""
    vocab, d = 8_400_000, 512                                  # 4.3e9
    table = torch.zeros(vocab, d, dtype=torch.float16, device="cuda")
    at = torch.tensor([0, 1, 4_194_304, 8_388_607, 8_388_608, vocab - 1], device="cuda")
    table[at] = (torch.arange(6, device="cuda")[:, None] + 1 + torch.arange(d, device="cuda") / 1024).half()
    tokens = at.repeat(300).to(torch.int32)                    # 1800 rows: sorted; 6: few
    for t in (tokens, tokens[:6]):
        assert torch.equal(cuda_rt.embed(table, t), table[t.long()])
        gy = torch.ones(t.numel(), d, device="cuda").half()
        g = cuda_rt.embed_grad(t, gy, vocab)
        assert (g[at] == t.numel() // 6).all() and float(g.sum(dtype=torch.float64)) == t.numel() * d
        del g
    del table
    rows = vocab                                               # gy beyond 2^32
    gy = torch.zeros(rows, d, dtype=torch.float16, device="cuda")
    gy[at] = 1.0
    tokens = (torch.arange(rows, device="cuda") % 1000).to(torch.int32)
    g = cuda_rt.embed_grad(tokens, gy, 1000)
    want = torch.zeros(1000, device="cuda").index_add_(0, at % 1000, torch.ones(6, device="cuda"))
    assert torch.equal(g, want[:, None].expand(1000, d))
    y = cuda_rt.embed(torch.arange(1000, device="cuda")[:, None].expand(1000, d).half().contiguous(), tokens)
    assert (y[at, 7] == (at % 1000).half()).all() and float(y[-1].float().sum()) == ((rows - 1) % 1000) * d   # (in f32: FP16 has no 511 488)


def test_the_library_refuses(cuda_rt):
    """Statuses of the entry points themselves; nothing is written."""
    import ctypes as C
    lib, h, stream = cuda_rt._lib, cuda_rt._h, torch.cuda.current_stream().cuda_stream
    t = torch.zeros(8, 16, device="cuda")
    tok = torch.zeros(2000, dtype=torch.int32, device="cuda")
    gy, out = torch.zeros(2000, 16, device="cuda"), torch.full((2000, 16), 77.0, device="cuda")

    def embed(dtype=0, table=t.data_ptr(), stride=16, tokens=tok.data_ptr(), scale=1.0, rows=8, c=16, vocab=8, out_dtype=0, y=out.data_ptr()):
        return lib.ullis_cuda_embed(h, stream, dtype, table, stride, tokens, 0xFFFFFFFF, scale, rows, c, vocab, out_dtype, y)

    assert embed() == cuda.OK
    out.fill_(77.0)
    for bad in (dict(dtype=3), dict(out_dtype=-1), dict(scale=float("nan")), dict(table=None), dict(tokens=None), dict(y=None),
                dict(tokens=tok.data_ptr() + 2), dict(table=t.data_ptr() + 1)):
        assert embed(**bad) == cuda.ERR_ARG, bad
    for bad in (dict(stride=15), dict(c=0), dict(vocab=0), dict(rows=1 << 31), dict(c=1 << 24, stride=1 << 24), dict(vocab=1 << 31)):
        assert embed(**bad) == cuda.ERR_SHAPE, bad
    assert lib.ullis_cuda_embed(None, stream, 0, t.data_ptr(), 16, tok.data_ptr(), 0, 1.0, 8, 16, 8, 0, out.data_ptr()) == cuda.ERR_ARG
    need = C.c_size_t(0)
    assert lib.ullis_cuda_embed_grad_workspace(h, 0, 2000, 16, 8, C.byref(need)) == cuda.OK
    work = torch.zeros(need.value + 256, dtype=torch.uint8, device="cuda")

    def grad(dtype=0, tokens=tok.data_ptr(), x=gy.data_ptr(), stride=16, rows=2000, c=16, vocab=8, scale=1.0, g=out.data_ptr(), w=work.data_ptr(),
             size=need.value):
        return lib.ullis_cuda_embed_grad(h, stream, dtype, tokens, 0xFFFFFFFF, x, stride, rows, c, vocab, scale, g, w, size)

    for bad in (dict(dtype=9), dict(scale=float("inf")), dict(tokens=None), dict(x=None), dict(g=None), dict(w=None), dict(w=work.data_ptr() + 4),
                dict(g=out.data_ptr() + 2)):
        assert grad(**bad) == cuda.ERR_ARG, bad
    for bad in (dict(stride=8), dict(size=need.value - 1), dict(vocab=0), dict(c=0), dict(rows=1 << 31)):
        assert grad(**bad) == cuda.ERR_SHAPE, bad
    torch.cuda.synchronize()
    assert (out == 77).all()
    assert grad() == cuda.OK
    ids, top = torch.zeros(8, 300, dtype=torch.int32, device="cuda"), torch.zeros(8, 300, device="cuda")
    for k, vocab, stride, code in ((0, 16, 16, cuda.ERR_SHAPE), (17, 16, 16, cuda.ERR_SHAPE), (257, 1000, 1000, cuda.ERR_SHAPE), (4, 16, 15, cuda.ERR_SHAPE),
                                   (4, 16, 16, cuda.OK)):
        assert lib.ullis_cuda_top_logits(h, stream, 0, t.data_ptr(), stride, 8, vocab, k, ids.data_ptr(), top.data_ptr()) == code
    assert lib.ullis_cuda_top_logits(h, stream, 0, t.data_ptr(), 16, 8, 16, 4, None, top.data_ptr()) == cuda.ERR_ARG


@pytest.mark.parametrize("shape", [(), (1,), (1, 1)])
def test_a_single_token(cuda_rt, shape):
    """A token of no dimensions has a row of one, and its gradient is taken as it comes."""
    table = torch.randn(9, 40, device="cuda")
    tokens = torch.full(shape, 4, dtype=torch.int32, device="cuda")
    y = cuda_rt.embed(table, tokens)
    assert y.shape == (*shape, 40) and torch.equal(y.reshape(40), table[4])
    g = cuda_rt.embed_grad(tokens, y, 9, scale=2.0)
    assert torch.equal(g[4], 2.0 * table[4]) and not g[:4].any() and not g[5:].any()
    with pytest.raises(cuda.UllisCudaError):
        cuda_rt.embed_grad(tokens, y.reshape(2, 20), 9)
