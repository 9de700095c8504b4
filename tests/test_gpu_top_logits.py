"""CudaRuntime.top_logits against a stable sort in 64 bits: the same columns and the same values, whatever the order, ties, infinities
and NaN of the rows."""
import pytest
import torch

from ullis_b200 import cuda

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def check(got, logits, k):
    values, ids = torch.sort((logits + 0.0).double(), dim=-1, descending=True, stable=True)      # NaN first
    assert got.ids.dtype == torch.int32 and got.logits.dtype == logits.dtype
    assert torch.equal(got.ids.long(), ids[..., :k])
    assert torch.equal(torch.nan_to_num(got.logits.double(), nan=3e38), torch.nan_to_num(values[..., :k], nan=3e38))


def made(kind, rows, vocab, dtype, g):
    z = torch.randn(rows, vocab, generator=g, device="cuda")
    if kind == "ties":
        z = torch.round(z)
    elif kind == "constant":
        z = torch.zeros_like(z)
        z[::2] = -0.0
    elif kind == "rising":
        z = torch.sort(z, 1).values
    elif kind == "falling":
        z = torch.sort(z, 1, descending=True).values
    elif kind == "masked":
        z = torch.where(torch.rand(rows, vocab, generator=g, device="cuda") < 0.98, -torch.inf, z)
        z[rows // 2] = -torch.inf
    elif kind == "lowest":
        z = torch.where(torch.rand(rows, vocab, generator=g, device="cuda") < 0.99, torch.finfo(TYPES[dtype]).min, z)
    elif kind == "odd":
        u = torch.rand(rows, vocab, generator=g, device="cuda")
        z = torch.where(u < 0.01, torch.nan, torch.where(u < 0.02, torch.inf, torch.where(u < 0.03, -torch.inf, z)))
        z = torch.where((u > 0.5) & (u < 0.6), -torch.nan, z)
        z[0] = torch.nan
    return z.to(TYPES[dtype])


KINDS = ["normal", "ties", "constant", "rising", "falling", "masked", "lowest", "odd"]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,vocab,k", [(1, 1, 1), (3, 2, 2), (5, 33, 7), (9, 300, 256), (32, 8192, 16), (7, 1023, 64), (40, 10007, 20), (3, 50021, 65),
                                          (2, 70000, 128), (1, 131072, 256), (2600, 4099, 64), (2500, 2048, 33)])
def test_against_a_sort(cuda_rt, rows, vocab, k, kind, dtype):
    g = torch.Generator("cuda").manual_seed(rows + vocab + k)
    logits = made(kind, rows, vocab, dtype, g)
    got = cuda_rt.top_logits(logits, k)
    check(got, logits, k)


@pytest.mark.parametrize("k", [1, 2, 31, 32, 33, 63, 64, 65, 96, 127, 128, 129, 200, 255, 256])
def test_every_width(cuda_rt, k):
    g = torch.Generator("cuda").manual_seed(k)
    for rows, vocab in ((11, 8192), (3000, 512)):
        logits = made("ties", rows, vocab, "f32", g) + torch.randn(rows, vocab, generator=g, device="cuda").clamp(min=0)
        check(cuda_rt.top_logits(logits, k), logits, k)


@pytest.mark.parametrize("dtype", TYPES)
def test_views_shapes_and_odd_starts(cuda_rt, dtype):
    g = torch.Generator("cuda").manual_seed(2)
    wide = torch.randn(64, 3001, generator=g, device="cuda").to(TYPES[dtype])
    wide[:, 0], wide[:, -1] = 100.0, 100.0                     # what lies beside a view is larger than anything in it
    for first, last in ((1, 3000), (3, 2999), (8, 3000), (0, 3001), (1, 2), (1, 9), (2, 12), (17, 1041)):
        view = wide[:, first:last]
        if first and last < 3001:
            k = min(40, last - first)
            check(cuda_rt.top_logits(view, k), view, k)
    cube = wide[:, :2000].contiguous().view(4, 16, 2000)
    got = cuda_rt.top_logits(cube, 5)
    assert got.ids.shape == got.logits.shape == (4, 16, 5)
    check(got, cube, 5)
    none = cuda_rt.top_logits(cube[:0], 5)
    assert none.ids.shape == (0, 16, 5)


def test_rows_past_32_bits(cuda_rt):
    rows, vocab = 17000, 131072                                # 2.2e9 elements
    logits = torch.zeros(rows, vocab, dtype=torch.bfloat16, device="cuda")
    at = (torch.arange(rows, device="cuda") * 7919) % (vocab - 3)
    for j in range(3):
        logits[torch.arange(rows, device="cuda"), at + j] = 3.0 - j
    got = cuda_rt.top_logits(logits, 3)
    assert torch.equal(got.ids.long(), at[:, None] + torch.arange(3, device="cuda"))
    assert (got.logits == torch.tensor([3.0, 2.0, 1.0], device="cuda")).all()


def test_a_replayed_graph_and_no_more_written(cuda_rt):
    g = torch.Generator("cuda").manual_seed(4)
    logits = torch.randn(50, 9001, generator=g, device="cuda")
    cuda_rt.top_logits(logits, 10)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = cuda_rt.top_logits(logits, 10)
    for _ in range(3):
        logits.normal_(generator=g)
        graph.replay()
        check(got, logits, 10)
    for rows, k in ((50, 10), (1, 1), (33, 70)):
        ids, top = torch.full((rows * k + 8,), 77, dtype=torch.int32, device="cuda"), torch.full((rows * k + 8,), 77.0, device="cuda")
        assert cuda_rt._lib.ullis_cuda_top_logits(cuda_rt._h, torch.cuda.current_stream().cuda_stream, 0, logits.data_ptr(), 9001, rows, 9001, k,
                                                  ids.data_ptr() + 4, top.data_ptr() + 4) == cuda.OK
        check(type(got)(ids[1:1 + rows * k].view(rows, k), top[1:1 + rows * k].view(rows, k)), logits[:rows], k)
        assert ids[0] == 77 and (ids[1 + rows * k:] == 77).all() and top[0] == 77 and (top[1 + rows * k:] == 77).all()
