"""CudaRuntime.head_ce_grad against the formulas in 64 bits.

Tolerances bound every rounding from above, element by element: tensor cores cut off each addition (2^-23 of the sum of the
terms' sizes per term), f32 steps are off by 2^-24, exp by 2^-21, the operand g * scale and what leaves in 16 bits by half a step
of their type."""
import math

import pytest
import torch

from ullis_b200 import cuda

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def signs(words, vocab, d):
    b = torch.stack([(words.view(torch.uint8) >> k) & 1 for k in range(8)], 1).reshape(-1)[: vocab * d]
    return 2.0 * b.reshape(vocab, d).double() - 1.0


def inputs(rows, time, d, vocab, dtype, packed, ignored=0.0, seed=0, lean=1.0, bias=True, size=0.0125):
    g = torch.Generator("cuda").manual_seed(seed)
    rand = lambda *s: torch.rand(*s, generator=g, device="cuda")    # noqa: E731
    randn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    labels = (rand(rows) * vocab).to(torch.int32).clamp(max=vocab - 1)
    after = torch.roll(labels, -1).long()
    hidden = randn(rows, d)
    scale = None
    if packed:
        n = (vocab * d + 31) // 32
        weight = torch.randint(-(1 << 31), 1 << 31, (n,), generator=g, device="cuda").to(torch.int32)
        scale = (size * (0.5 + rand(vocab))).half()
        hidden += lean * signs(weight, vocab, d)[after].float()
    else:
        weight = (size * randn(vocab, d)).to(TYPES[dtype])
        hidden += lean * torch.sign(weight[after].float())
    labels = torch.where(rand(rows) < ignored, torch.full_like(labels, -1), labels)
    return {"hidden": hidden.to(TYPES[dtype]), "weight": weight, "labels": labels, "scale": scale,
            "bias": (0.1 * randn(vocab)).half() if bias else None, "time": time}


def formulas(s, ignore_id=-1, loss_scale=1.0):
    """{output: (value, tolerance)} in 64 bits."""
    h, t = s["hidden"].double(), s["hidden"].dtype
    rows, d = h.shape
    packed = s["scale"] is not None
    vocab = s["scale"].numel() if packed else s["weight"].shape[0]
    w = signs(s["weight"], vocab, d) if packed else s["weight"].double()
    scale = s["scale"].double() if packed else torch.ones(vocab, dtype=torch.float64, device="cuda")
    bias = s["bias"].double() if s["bias"] is not None else torch.zeros_like(scale)
    at = torch.arange(rows, device="cuda")
    after = torch.roll(s["labels"], -1)
    counts = (at % s["time"] + 1 < s["time"]) & (after != ignore_id)
    after = torch.where(counts, after, 0).long()
    h = torch.where(counts[:, None], h, 0.0)
    a = h @ w.t()
    a_off = 2 * U * d * (h.abs() @ w.abs().t())
    z = a * scale + bias
    z_off = a_off * scale.abs() + 4 * U * ((a * scale).abs() + bias.abs())
    lse = torch.logsumexp(z, 1)
    terms = 80 + vocab / 256                       # additions behind one sum of exp
    p = torch.exp(z - lse[:, None])
    lse_off = (p * z_off).sum(1) + (terms * U + 2.0 ** -21) + 4 * U * lse.abs()
    loss = lse - z.gather(1, after[:, None])[:, 0]
    loss_off = lse_off + z_off.gather(1, after[:, None])[:, 0] + 4 * U * loss.abs()
    g = p.clone()
    g[at, after] -= 1.0
    g_off = p * (z_off + lse_off[:, None] + 2.0 ** -21 + 4 * U * (z - lse[:, None]).abs()) + U
    live = counts[:, None].double()
    g, g_off = g * live, g_off * live
    half = torch.finfo(t).eps / 2
    gs, gs_off = g * scale, g_off * scale.abs() + half * (g * scale).abs()
    if t == torch.float16:                         # below 2^-14 FP16 has steps of 2^-24; the largest scale lies at 2^14
        top = 2.0 ** (14 - math.floor(math.log2(max(scale.abs().max().item(), 2.0 ** -24))))
        gs_off = gs_off + 2.0 ** -25 / top * live
    lowest = torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2
    k = abs(loss_scale)

    def out16(value, off, n_terms, sizes):
        value = loss_scale * value
        return value, k * (off + 2 * U * n_terms * sizes) + half * value.abs() + lowest + 4 * U * value.abs()

    n = 16 + rows                                  # additions behind one sum over the rows
    found = {"row_loss": (torch.where(counts, loss, 0.0), torch.where(counts, loss_off, 0.0)),
             "hidden": out16(gs @ w, gs_off @ w.abs(), vocab, gs.abs() @ w.abs()),
             "weight": out16(gs.t() @ h, gs_off.t() @ h.abs(), rows, gs.abs().t() @ h.abs())}
    if s["bias"] is not None:
        found["bias"] = (loss_scale * g.sum(0), k * (g_off.sum(0) + U * n * g.abs().sum(0)))
    if packed:
        found["scale"] = (loss_scale * (g * a).sum(0),
                          k * ((g_off * a.abs() + g.abs() * a_off).sum(0) + U * n * (g * a).abs().sum(0)))
    return found


def call(rt, s, **more):
    return rt.head_ce_grad(s["hidden"], s["weight"], s["labels"], scale=s["scale"], bias=s["bias"], ignore_id=more.pop("ignore_id", -1),
                           time=s["time"], **more)


def check(got, want):
    for name, (value, off) in want.items():
        x = getattr(got, name).double().reshape(value.shape)
        # beyond the type's largest number an infinity of the right sign is the rounded value
        over = torch.isinf(x) & (torch.sign(x) == torch.sign(value)) & (value.abs() + off >= torch.finfo(getattr(got, name).dtype).max)
        bad = ~(((x - value).abs() <= off) | over)
        assert not bad.any(), (name, int(bad.sum()), x[bad][:4].tolist(), value[bad][:4].tolist(), off[bad][:4].tolist())
    for name in ("scale", "bias"):
        assert (getattr(got, name) is not None) == (name in want)


CASES = [
    # rows, time, channels, vocab, ignored
    (2, 2, 8, 1, 0.0),                # one token of one
    (1, 1, 64, 100, 0.0),             # nothing to predict
    (3, 3, 1, 2, 0.0),
    (5, 5, 7, 33, 0.0),
    (32, 32, 256, 8192, 0.0),
    (96, 32, 64, 257, 0.3),
    (130, 13, 100, 1000, 0.0),
    (256, 256, 64, 256, 0.0),
    (257, 257, 72, 511, 0.5),
    (300, 100, 200, 4099, 0.0),
    (1021, 1021, 512, 777, 0.2),
    (2048, 512, 520, 1030, 0.0),
    (640, 64, 768, 10007, 0.7),
    (128, 128, 1000, 30011, 0.0),
    (4096, 2048, 129, 6001, 0.0),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("packed", [True, False], ids=["packed", "dense"])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_the_formulas(cuda_rt, case, packed, dtype):
    rows, time, d, vocab, ignored = case
    s = inputs(rows, time, d, vocab, dtype, packed, ignored, seed=rows + vocab)
    k = 2.0 ** math.ceil(math.log2(max(1, time - 1))) / max(1, time - 1)
    got = call(cuda_rt, s, loss_scale=k)
    assert got.hidden.dtype == got.weight.dtype == TYPES[dtype]
    check(got, formulas(s, loss_scale=k))


@pytest.mark.parametrize("packed,dtype", [(True, "f16"), (False, "bf16")])
def test_a_vocabulary_in_several_pieces(cuda_rt, packed, dtype):
    """More than 2^27 logits: the hidden gradient grows over two pieces, the last column tile is a narrow one."""
    s = inputs(8192 + 300, 8192 + 300, 64, 16400 + 9, dtype, packed, 0.1)
    check(call(cuda_rt, s), formulas(s))


@pytest.mark.parametrize("packed,dtype", [(True, "bf16"), (False, "f16")])
def test_a_vocabulary_in_several_pieces_of_the_largest_size(cuda_rt, packed, dtype):
    """More than 2^28 logits, which the workspace holds of one piece."""
    s = inputs(16384 + 40, 16384 + 40, 64, 16500, dtype, packed, 0.02)
    check(call(cuda_rt, s), formulas(s))


@pytest.mark.parametrize("rows,d,vocab,packed,dtype", [(4096, 64, 70000, True, "f16"), (4000, 66, 70000, False, "bf16"),
                                                       (40000, 40, 8000, True, "bf16"), (40000, 33, 8000, False, "f16")])
def test_sums_over_pieces_and_ranges(cuda_rt, rows, d, vocab, packed, dtype):
    """Two pieces of the vocabulary, and one of the gradient products in several ranges of its sums: the hidden states' (few rows, a large
    vocabulary), whose sum over the pieces lies in f32 between them, or the weights' (many rows).  The launches show that it is so:
    list, operands, log sum exp, rows' losses; for each piece the gradient, columns' sums, two products and the sum of the ranges."""
    s = inputs(rows, rows // 8, d, vocab, dtype, packed, 0.1, seed=vocab + d)
    before = cuda_rt.launch_count
    got = call(cuda_rt, s)
    assert cuda_rt.launch_count - before == 4 + 2 * 5
    check(got, formulas(s))


def lost(got, want):
    """Mean relative error of sums, positive where they are too small; what rounds them to 16 bits has a mean of 0."""
    return ((want - got.double()) / want).mean().item()


@pytest.mark.parametrize("over", ["rows", "vocabulary"])
def test_long_sums_of_one_sign(cuda_rt, over):
    """What the tensor cores cut off of a sum does not grow with its length.  All logits are 0 and every probability 1 / vocab, in FP16 the
    number p; so the weights' gradient is p times the sum of the rows of h (no weights, h in [1, 2)), the hidden states' p times that of the
    weights (no h, weights in [1, 2), the target's 0), all terms of one sign.  Of 1024 sums, each rounded by half a step of FP16 at most,
    the mean is off by 2^-11 / sqrt(3 * 1024) < 1e-5 (one sigma); what is lost has to stay below 2^-12, the smallest half step there is."""
    d, found = 1024, {}
    for length in (16000, 65000, 200000) if over == "rows" else (16000, 65000):
        g = torch.Generator("cuda").manual_seed(length)
        rows, vocab = (length + 1, 4000) if over == "rows" else (4096, length)
        # (2^14: what the call multiplies g by in FP16; an f32 probability rounds to the same number)
        p, near = (torch.tensor([x * 2.0 ** 14 / vocab for x in (1.0, 1 - 1e-5, 1 + 1e-5)], dtype=torch.float64).half().split([1, 2]))
        assert (near == p).all()
        ones = (1 + torch.randint(0, 1024, (length, d), generator=g, device="cuda") / 1024).half()
        if over == "rows":
            hidden = torch.cat([ones, torch.full_like(ones[:1], float("nan"))])
            weight = torch.zeros(vocab, d, dtype=torch.float16, device="cuda")
        else:
            hidden = torch.zeros(rows, d, dtype=torch.float16, device="cuda")
            weight = ones
            weight[0] = 0.0
        r = cuda_rt.head_ce_grad(hidden, weight, torch.zeros(rows, dtype=torch.int32, device="cuda"), time=rows)
        got = r.weight[1:] if over == "rows" else r.hidden[:-1]
        assert torch.equal(got, got[:1].expand_as(got))
        found[length] = lost(got[0], ones.sum(0, dtype=torch.float64) * (p.item() * 2.0 ** -14))
    assert max(found.values()) <= 1.25 * found[16000] + 5e-5, found
    assert max(found.values()) <= 2.0 ** -12, found


def test_drawn_sizes(cuda_rt):
    import random
    rng = random.Random(7)
    for seed in range(40):
        time = rng.choice([1, 2, 3, 31, 64, 65, 127, 200, 333])
        rows = time * rng.randint(1, max(1, 900 // time))
        d = rng.choice([1, 3, 8, 15, 16, 40, 64, 65, 96, 128, 250, 264])
        vocab = rng.choice([1, 2, 5, 63, 64, 65, 255, 256, 257, 500, 777, 1024, 1500])
        s = inputs(rows, time, d, vocab, rng.choice(["f16", "bf16"]), rng.random() < 0.5, rng.choice([0.0, 0.1, 0.5, 0.9]), seed=seed,
                   bias=rng.random() < 0.7)
        check(call(cuda_rt, s), formulas(s))


def test_scales_of_every_size(cuda_rt):
    s = inputs(200, 200, 64, 600, "f16", True)
    s["scale"][::7] = 0.0
    s["scale"][1::7] *= -1.0
    s["scale"][3] = 2.0 ** -24
    check(call(cuda_rt, s), formulas(s))
    for size in (2.0 ** -20, 6.0e4):           # all small; so large that the softmax is one column
        s = inputs(100, 100, 8, 64, "f16", True, size=size, lean=0.0)
        s["scale"].clamp_(max=65504.0)         # (an infinite scale has no gradient)
        check(call(cuda_rt, s), formulas(s))


def test_a_softmax_that_is_almost_one_hot(cuda_rt):
    for dtype in TYPES:
        s = inputs(300, 300, 256, 2000, dtype, True, lean=4.0, size=0.05)
        want = formulas(s)
        assert want["row_loss"][0].median() < 1e-3
        check(call(cuda_rt, s), want)


def test_rows_that_are_sure_have_small_gradients(cuda_rt):
    """Gradients of rows whose loss is 1e-8 to 1e-4, to a relative bound.  Hidden states are multiples of 1/8 and weights +-1, so
    the products are exact in any order, and a logit in units of ln 2, below 64, is off by the roundings of its scale and its
    bias and of itself, 3 * 2^-24 * 64.  A target's 1 - p, and p of another column, take two logits and a sum of 400
    terms: off by less than 2 * 1.2e-5 * ln 2 + 80 * 2^-24 + 2^-21 < 2^-14 relatively."""
    g = torch.Generator("cuda").manual_seed(5)
    rows, d, vocab = 600, 1000, 400
    s = inputs(rows, rows, d, vocab, "bf16", True, lean=2.0)
    s["hidden"] = ((torch.randn(rows, d, generator=g, device="cuda") * 8).round() / 8).clamp(-6, 6)
    s["hidden"] += 2.0 * signs(s["weight"], vocab, d)[torch.roll(s["labels"], -1).long()].float()
    s["hidden"] = s["hidden"].bfloat16()
    assert torch.equal(s["hidden"].float() * 8, (s["hidden"].float() * 8).round())
    s["scale"].clamp_(max=0.0155)
    got = call(cuda_rt, s)
    a = s["hidden"].double() @ signs(s["weight"], vocab, d).t()
    z = a * s["scale"].double() + s["bias"].double()
    assert z.abs().max() / math.log(2.0) < 64
    after, at = torch.roll(s["labels"], -1).long(), torch.arange(rows, device="cuda")
    rest = torch.exp(z).scatter(1, after[:, None], 0.0)
    hit = torch.exp(z.gather(1, after[:, None])[:, 0])
    p = rest / (rest.sum(1) + hit)[:, None]
    p[at, after] = -rest.sum(1) / (rest.sum(1) + hit)
    p[-1] = 0.0
    loss = torch.log1p(rest.sum(1) / hit)[:-1]
    assert 1e-12 < loss.min() and loss.median() < 1e-4
    assert ((got.row_loss[:-1].double() - loss).abs() <= 2.0 ** -14 * loss).all()
    for x, value in ((got.bias, p), (got.scale, p * a)):
        off = (2.0 ** -14 + U * (16 + rows)) * value.abs().sum(0)
        assert ((x.double() - value.sum(0)).abs() <= off).all()


@pytest.mark.parametrize("packed", [True, False], ids=["packed", "dense"])
def test_masked_rows_hold_anything(cuda_rt, packed):
    s = inputs(260, 130, 64, 500, "bf16", packed, 0.4)
    want = call(cuda_rt, s)
    after = torch.roll(s["labels"], -1)
    masked = (after == -1) | (torch.arange(260, device="cuda") % 130 == 129)
    dirty = dict(s, hidden=s["hidden"].clone())
    dirty["hidden"][masked] = torch.tensor([float("nan"), float("inf"), -float("inf"), 3e38], device="cuda").bfloat16().repeat(16)
    got = call(cuda_rt, dirty)
    for a, b in zip(got, want):
        assert (a is None and b is None) or torch.equal(a, b)
    assert not got.row_loss[masked].any() and not got.hidden[masked].any()


def test_no_row_counts(cuda_rt):
    s = inputs(100, 100, 64, 300, "f16", True, ignored=2.0)
    got = call(cuda_rt, s)
    for x in got:
        assert torch.equal(x, torch.zeros_like(x))


def test_bias_that_bans_tokens(cuda_rt):
    s = inputs(200, 200, 64, 700, "f16", True)
    banned = torch.arange(700, device="cuda") % 3 == 1
    s["labels"] = (s["labels"] // 3 * 3).clamp(max=699)          # no target is banned
    for low in (-65504.0, -float("inf")):
        s["bias"] = torch.where(banned, torch.tensor(low, device="cuda").half(), s["bias"])
        got = call(cuda_rt, s)
        keep = torch.nonzero(~banned)[:, 0]
        # the head without them
        w = signs(s["weight"], 700, 64)
        dense = {"hidden": s["hidden"], "weight": (w[keep]).half(), "scale": None, "bias": None, "labels": s["labels"], "time": 200}
        assert not got.bias[banned].any() and not got.scale[banned].any() and not got.weight[banned].any()
        z = s["hidden"].double() @ w[keep].t() * s["scale"][keep].double() + s["bias"][keep].double()
        at = torch.searchsorted(keep, torch.roll(s["labels"], -1).long())
        loss = torch.logsumexp(z, 1) - z.gather(1, at[:, None])[:, 0]
        loss[-1] = 0.0
        assert (got.row_loss.double() - loss).abs().max() <= 1e-4
        assert dense["weight"].shape[0] == keep.numel()
    s["bias"][s["labels"][1].item()] = -float("inf")             # the target of row 0 has no probability
    got = call(cuda_rt, s)
    assert got.row_loss[0] == float("inf") and torch.isfinite(got.hidden).all()


def test_a_label_outside_the_vocabulary(cuda_rt):
    s = inputs(64, 64, 64, 300, "f16", True)
    s["labels"][10], s["labels"][11] = 300, -5
    got = call(cuda_rt, s)
    assert torch.isnan(got.row_loss[9]) and torch.isnan(got.row_loss[10]) and torch.isfinite(got.row_loss[11:]).all()
    s["labels"][10] = s["labels"][11] = -1
    want = call(cuda_rt, s)
    for name in ("hidden", "weight", "scale", "bias"):
        assert torch.equal(getattr(got, name), getattr(want, name))


def test_a_row_that_is_not_finite_shows(cuda_rt):
    s = inputs(64, 64, 64, 300, "f16", True)
    s["hidden"][5, 3] = float("inf")
    got = call(cuda_rt, s)
    assert torch.isnan(got.row_loss[5]) and torch.isnan(got.hidden[5]).all()
    assert torch.isfinite(got.row_loss[6:]).all() and torch.isfinite(got.hidden[6:]).all()


def test_ignore_id_is_a_number_like_any(cuda_rt):
    s = inputs(128, 64, 64, 300, "f16", False)
    s["labels"][::5] = 7
    check(call(cuda_rt, s, ignore_id=7), formulas(s, ignore_id=7))
    a, b = call(cuda_rt, s, ignore_id=-1), call(cuda_rt, s, ignore_id=0xFFFFFFFF)
    assert torch.equal(a.row_loss, b.row_loss)


@pytest.mark.parametrize("offset,stride", [(0, 104), (1, 97), (8, 96), (3, 96)])
def test_rows_with_gaps_and_odd_starts(cuda_rt, offset, stride):
    s = inputs(200, 100, 96, 333, "bf16", False)
    want = call(cuda_rt, s)
    base = torch.full((200 * stride + offset + 96,), float("nan"), device="cuda").bfloat16()
    view = base.as_strided((200, 96), (stride, 1), offset)
    view.copy_(s["hidden"])
    odd = torch.empty(333 * 96 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(333, 96)
    odd.copy_(s["weight"])
    got = call(cuda_rt, dict(s, hidden=view, weight=odd))
    for a, b in zip(got, want):
        assert (a is None and b is None) or torch.equal(a, b)


def test_leading_dimensions_give_the_time(cuda_rt):
    s = inputs(120, 30, 64, 100, "f16", False)
    want = call(cuda_rt, s)
    got = cuda_rt.head_ce_grad(s["hidden"].reshape(4, 30, 64), s["weight"], s["labels"].reshape(4, 30), bias=s["bias"], ignore_id=-1)
    assert got.hidden.shape == (4, 30, 64) and torch.equal(got.hidden.reshape(120, 64), want.hidden)
    assert torch.equal(got.row_loss, want.row_loss)


def test_zero_rows(cuda_rt):
    s = inputs(2, 2, 64, 100, "f16", True)
    got = cuda_rt.head_ce_grad(s["hidden"][:0], s["weight"], s["labels"][:0], scale=s["scale"], bias=s["bias"])
    assert got.row_loss.shape == (0,) and got.hidden.shape == (0, 64)
    assert not got.weight.any() and not got.scale.any() and not got.bias.any()


def test_the_gradient_against_differences(cuda_rt):
    """Central differences of the summed losses, in 64 bits by the formulas, along random directions."""
    s = inputs(48, 16, 40, 130, "f16", True)
    got = call(cuda_rt, s)
    w = signs(s["weight"], 130, 40)
    after = torch.roll(s["labels"], -1).long()
    counts = torch.arange(48, device="cuda") % 16 < 15

    def loss(h, w, scale, bias):
        z = h @ w.t() * scale + bias
        return (torch.logsumexp(z, 1) - z.gather(1, after[:, None])[:, 0])[counts].sum()

    at = [s["hidden"].double(), w, s["scale"].double(), s["bias"].double()]
    for i, g in enumerate((got.hidden, got.weight, got.scale, got.bias)):
        gen = torch.Generator("cuda").manual_seed(i)
        d = torch.randn(at[i].shape, generator=gen, device="cuda", dtype=torch.float64)
        step = 1e-4 / max(1.0, d.abs().max().item()) * (0.01 if i == 2 else 1.0)
        plus, minus = ([x + k * step * d if j == i else x for j, x in enumerate(at)] for k in (1, -1))
        slope = ((loss(*plus) - loss(*minus)) / (2 * step)).item()
        size = (g.double() * d).abs().sum().item()
        assert abs(slope - (g.double() * d).sum().item()) <= 2.0 ** -10 * size + 1e-6


def test_graphs_streams_and_the_same_result_every_time(cuda_rt):
    data = [inputs(700, 350, 128, 3000, "bf16", True, 0.2, seed=k) for k in (1, 2)]
    want = [call(cuda_rt, s) for s in data]
    graphs, got = [], []
    for s in data:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got.append(call(cuda_rt, s))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for stream, g in zip(streams, graphs):
            with torch.cuda.stream(stream):
                g.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    cuda_rt.synchronize()


@pytest.mark.parametrize("rows,vocab", [(96, 700), (2600, 3000)])
def test_a_graph_replayed_with_other_inputs(cuda_rt, rows, vocab):
    """How many rows count, and which, is known on the device only; and whatever lies in the workspace, nothing of it shows."""
    first, second = (inputs(rows, rows // 2, 72, vocab, "bf16", True, ignored, seed=k) for k, ignored in ((1, 0.8), (2, 0.1)))
    want = [call(cuda_rt, s) for s in (first, second)]
    held = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in first.items()}
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = call(cuda_rt, held)
        dirt = torch.full((1 << 28,), 0xFF, dtype=torch.uint8, device="cuda")   # NaN in f32 and 16 bits, over what the call gave back
    for k in (0, 1, 0, 1, 1):
        for name, v in (first, second)[k].items():
            if isinstance(v, torch.Tensor):
                held[name].copy_(v)
        g.replay()
        for a, b in zip(got, want[k]):
            assert torch.equal(a, b)
    del dirt


@pytest.mark.parametrize("rows,vocab", [(5, 40), (96, 700), (2600, 3000), (9000, 16400)])
def test_nothing_depends_on_what_the_workspace_held(cuda_rt, rows, vocab):
    s = inputs(rows, rows, 72, vocab, "f16", True, 0.3, seed=9)
    want = call(cuda_rt, s)
    for byte in (0xFF, 0x7B):     # NaN; large numbers
        torch.cuda.empty_cache()
        dirt = torch.full((1 << 30,), byte, dtype=torch.uint8, device="cuda")
        del dirt                  # the next blocks come out of it
        for a, b in zip(call(cuda_rt, s), want):
            assert torch.equal(a, b)


def test_refusals_of_the_library(cuda_rt):
    s = inputs(64, 64, 64, 300, "f16", True)
    with pytest.raises(cuda.UllisCudaError) as e:
        call(cuda_rt, s, loss_scale=float("nan"))
    assert e.value.code == cuda.ERR_ARG
    import ctypes as C
    p, n = (lambda t: C.c_void_p(t.data_ptr() if t is not None else None)), C.c_size_t
    out = torch.zeros(300 * 64, device="cuda")
    work = torch.empty(1 << 26, dtype=torch.uint8, device="cuda")
    fn = cuda_rt._lib.ullis_cuda_head_ce_grad

    def rc(**change):
        a = {"dtype": 1, "hidden": s["hidden"], "stride": 64, "bits": s["weight"], "weight": None, "scale": s["scale"], "rows": 64,
             "time": 64, "size": work.numel(), "g_scale": out} | change
        return fn(cuda_rt._h, None, C.c_int32(a["dtype"]), p(a["hidden"]), n(a["stride"]), p(a["bits"]), p(a["weight"]), p(a["scale"]),
                  p(s["bias"]), p(s["labels"]), C.c_uint32(0xFFFFFFFF), n(a["rows"]), n(a["time"]), n(64), n(300), C.c_float(1.0), p(out),
                  p(out), p(out), p(a["g_scale"]), p(out), p(work), n(a["size"]))

    assert rc(dtype=0) == cuda.ERR_ARG and rc(stride=63) == cuda.ERR_SHAPE and rc(time=63) == cuda.ERR_SHAPE
    assert rc(weight=s["hidden"]) == cuda.ERR_ARG and rc(scale=None) == cuda.ERR_ARG and rc(bits=None) == cuda.ERR_ARG
    assert rc(size=1000) == cuda.ERR_SHAPE and rc(hidden=None) == cuda.ERR_ARG
    assert rc(bits=None, weight=s["hidden"], scale=None) == cuda.ERR_ARG      # g_scale without scales
    torch.cuda.synchronize()
    assert not out.any()


def test_more_rows_than_the_list_is_made_for(cuda_rt):
    import ctypes as C
    size = C.c_size_t(7)
    fn = cuda_rt._lib.ullis_cuda_head_ce_grad_workspace
    assert fn(cuda_rt._h, 1 << 24, 8, 100, 1, C.byref(size)) == cuda.OK and size.value > 0
    assert fn(cuda_rt._h, (1 << 24) + 1, 8, 100, 1, C.byref(size)) == cuda.ERR_SHAPE and size.value == 0


def test_offsets_past_32_bits(cuda_rt):
    """More than 2^32 elements of hidden and of its gradient; rows that count at both ends, NaN in all others."""
    rows, d, vocab, time = 2 ** 22 + 128, 1032, 70, 64
    s = inputs(256, time, d, vocab, "bf16", True)
    ends = torch.cat([torch.arange(128), torch.arange(rows - 128, rows)]).cuda()
    big = dict(s, hidden=torch.full((rows, d), float("nan"), dtype=torch.bfloat16, device="cuda"),
               labels=torch.full((rows,), -1, dtype=torch.int32, device="cuda"))
    big["hidden"][ends], big["labels"][ends] = s["hidden"], s["labels"]
    got = call(cuda_rt, big)
    assert not got.hidden[128:-128].any() and not got.row_loss[128:-128].any()
    check(got._replace(hidden=got.hidden[ends], row_loss=got.row_loss[ends]), formulas(s))
