"""CudaRuntime.head_distill_grad against the formulas in 64 bits.

Tolerances bound every rounding from above, element by element, as in test_gpu_head_grad.py: tensor cores cut off each addition
(2^-23 of the sum of the terms' sizes per term), f32 steps are off by 2^-24, exp by 2^-21, the operand g * scale and what leaves in 16
bits by half a step of their type.  The teacher's probabilities are off by the roundings of (t - top) / T, of exp and of their sum."""
import math

import pytest
import torch

from test_gpu_head_grad import TYPES, U, check, inputs, signs

from ullis_b200 import cuda

pytestmark = pytest.mark.gpu

TOP_TYPES = {"f32": torch.float32, **TYPES}


def student(rows, time, d, vocab, dtype, packed, k, *, labels=True, alpha=0.5, temperature=2.0, ignored=0.0, absent=0.0, holes=0.0, hot=False,
            top_dtype="f32", seed=0, **more):
    s = inputs(rows, time, d, vocab, dtype, packed, ignored, seed, **more)
    g = torch.Generator("cuda").manual_seed(seed + 1)
    rand = lambda *n: torch.rand(*n, generator=g, device="cuda")    # noqa: E731
    # distinct ids in any order (hot: all of them among the first columns)
    n = min(vocab, k + 3) if hot else vocab
    if rows * n <= 1 << 26:
        ids = torch.argsort(rand(rows, n), 1)[:, :k]
    else:
        ids = ((torch.arange(k, device="cuda") + rand(rows, k)) * (n / k)).long().clamp(max=n - 1)
    if ids.shape[1] < k:
        ids = torch.cat([ids, torch.full((rows, k - ids.shape[1]), -1, device="cuda")], 1)
    after = torch.roll(s["labels"], -1)
    put = (rand(rows) < 0.8) & (after >= 0)
    ids[:, 0] = torch.where(put & ~(ids == after[:, None]).any(1), after, ids[:, 0])
    ids = torch.where((rand(rows, k) < holes) | (rand(rows, 1) < absent), -1 - (rand(rows, k) * 1000).long(), ids)
    s["top_ids"] = ids.to(torch.int32)
    s["top_logits"] = (3.0 * torch.randn(rows, k, generator=g, device="cuda")).to(TOP_TYPES[top_dtype])
    s.update(alpha=alpha, temperature=temperature)
    if not labels:
        s["labels"] = None
    return s


def formulas(s, ignore_id=-1, loss_scale=1.0, operand=None):
    """{output: (value, tolerance)} in 64 bits.  operand: how far g * scale is rounded, half a step of hidden's type."""
    h, t = s["hidden"].double(), s["hidden"].dtype
    rows, d = h.shape
    packed = s["scale"] is not None
    vocab = s["scale"].numel() if packed else s["weight"].shape[0]
    w16 = signs(s["weight"], vocab, d) if packed else s["weight"].double()
    scale = s["scale"].double() if packed else torch.ones(vocab, dtype=torch.float64, device="cuda")
    bias = s["bias"].double() if s["bias"] is not None else torch.zeros_like(scale)
    at = torch.arange(rows, device="cuda")
    alpha, tau = float(torch.tensor(s["alpha"], dtype=torch.float32)), float(torch.tensor(s["temperature"], dtype=torch.float32))
    ids, said = s["top_ids"].long(), s["top_logits"].double()
    entry = ids >= 0
    said = torch.where(entry, said, -torch.inf)
    has = (said > -torch.inf).any(1)
    if s["labels"] is None:
        counts, hard = has, torch.zeros(rows, dtype=torch.float64, device="cuda")
        after = torch.zeros(rows, dtype=torch.long, device="cuda")
    else:
        after = torch.roll(s["labels"], -1)
        counts = (at % s["time"] + 1 < s["time"]) & (after != ignore_id)
        after = torch.where(counts, after, 0).long()
        hard = torch.where(counts, 1.0 - alpha, 0.0)
    soft = torch.where(counts & has, alpha * tau, 0.0)
    h = torch.where(counts[:, None], h, 0.0)
    # the teacher
    top_said = torch.where(has, said.amax(1), 0.0)[:, None]
    x = torch.where(has[:, None], (said - top_said) / tau, -torch.inf)
    total = torch.where(has, torch.exp(x).sum(1), 1.0)[:, None]
    p = torch.exp(x) / total
    log_p = torch.where(p > 0, x - torch.log(total), 0.0)
    small = torch.where(p > 0, x.abs(), 0.0)
    p_off = p * (2.0 ** -20 + 8 * U * small + 8 * U * ids.shape[1])
    entropy = (p * log_p).sum(1)
    entropy_off = (p_off * log_p.abs() + p * (8 * U * small + 2.0 ** -20) + 8 * U * ids.shape[1] * (p * log_p).abs()).sum(1)
    live_ids = torch.where(entry, ids, 0)
    w = torch.zeros(rows, vocab, dtype=torch.float64, device="cuda").scatter_add_(1, live_ids, soft[:, None] * p)
    w_off = torch.zeros_like(w).scatter_add_(1, live_ids, soft[:, None] * (p_off + 4 * U * p))
    w[at, after] += hard
    w_off[at, after] += 2 * U * hard
    # the student
    a = h @ w16.t()
    a_off = 2 * U * d * (h.abs() @ w16.abs().t())
    z = a * scale + bias
    z_off = a_off * scale.abs() + 4 * U * ((a * scale).abs() + bias.abs())
    terms = 80 + vocab / 256                       # additions behind one sum of exp
    dense = torch.zeros_like(z)
    g_off = w_off + U * w
    loss = soft * tau * entropy
    loss_off = soft * tau * entropy_off + 4 * U * loss.abs()
    top = z.amax(1)
    for share, times, of_loss in ((hard, 1.0, hard), (soft, 1.0 / tau, soft * tau)):
        lse = torch.logsumexp(z * times, 1)
        q = torch.exp(z * times - lse[:, None])
        lse_off = (q * z_off).sum(1) * times + (terms * U + 2.0 ** -21) + 4 * U * lse.abs()
        dense += share[:, None] * q
        g_off += share[:, None] * q * (z_off * times + lse_off[:, None] + 2.0 ** -20 + 8 * U * ((z * times).abs() + lse.abs()[:, None] + 8))
        loss = loss + of_loss * (lse - top * times)
        loss_off = loss_off + of_loss * (lse_off + 8 * U * ((top * times).abs() + lse.abs()))
    off = w * (top[:, None] - z)
    loss = loss + off.sum(1)
    loss_off = loss_off + (w * (z_off + z_off.amax(1)[:, None] + 8 * U * (z.abs() + top.abs()[:, None])) + w_off * (top[:, None] - z)
                           + 32 * U * off).sum(1) + 8 * U * ids.shape[1] * soft * top.abs() + 8 * U * loss.abs()
    g = dense - w
    sizes = dense + w
    g_off = g_off + 2 * U * sizes
    half = torch.finfo(t).eps / 2
    gs, gs_off = g * scale, g_off * scale.abs() + (half if operand is None else operand) * (g * scale).abs()
    if t == torch.float16:                         # below 2^-14 FP16 has steps of 2^-24; the largest scale and share lie at 2^14
        room = max(0, math.ceil(math.log2(max(1e-30, float(hard.max()) + alpha * tau))))
        biggest = 2.0 ** (14 - room - math.floor(math.log2(max(scale.abs().max().item(), 2.0 ** -24))))
        gs_off = gs_off + 2.0 ** -25 / biggest * counts[:, None].double()
    lowest = torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2
    k = abs(loss_scale)

    def out16(value, off, n_terms, sizes):
        value = loss_scale * value
        return value, k * (off + 2 * U * n_terms * sizes) + half * value.abs() + lowest + 4 * U * value.abs()

    n = 48 + rows                                  # additions behind one sum over the rows
    found = {"row_loss": (torch.where(counts, loss, 0.0), torch.where(counts, loss_off, 0.0)),
             "hidden": out16(gs @ w16, gs_off @ w16.abs(), vocab, gs.abs() @ w16.abs()),
             "weight": out16(gs.t() @ h, gs_off.t() @ h.abs(), rows, gs.abs().t() @ h.abs())}
    if s["bias"] is not None:
        found["bias"] = (loss_scale * g.sum(0), k * (g_off.sum(0) + U * n * sizes.sum(0)))
    if packed:
        found["scale"] = (loss_scale * (g * a).sum(0),
                          k * ((g_off * a.abs() + g.abs() * a_off).sum(0) + U * n * (sizes * a.abs()).sum(0)))
    return found


def call(rt, s, **more):
    return rt.head_distill_grad(s["hidden"], s["weight"], s["top_ids"], s["top_logits"], scale=s["scale"], bias=s["bias"], labels=s["labels"],
                                alpha=s["alpha"], temperature=s["temperature"], ignore_id=more.pop("ignore_id", -1), time=s["time"], **more)


CASES = [
    # rows, time, channels, vocab, k
    (1, 1, 64, 100, 3, dict(labels=False, alpha=1.0)),
    (2, 2, 8, 1, 1, dict()),
    (3, 3, 1, 2, 2, dict(labels=False)),
    (5, 5, 7, 33, 4, dict(temperature=1.0)),
    (32, 32, 256, 8192, 16, dict()),
    (96, 32, 64, 257, 20, dict(ignored=0.3, absent=0.2, holes=0.3)),
    (130, 13, 100, 1000, 64, dict(labels=False, temperature=0.7, holes=0.5)),
    (256, 256, 64, 256, 256, dict(hot=True)),
    (257, 257, 72, 511, 33, dict(ignored=0.5, alpha=0.3, temperature=4.0)),
    (300, 100, 200, 4099, 7, dict(labels=False, alpha=0.4, absent=0.5)),
    (1021, 1021, 512, 777, 100, dict(hot=True, temperature=1.0)),
    (2048, 512, 520, 1030, 64, dict(hot=True, labels=False, temperature=1.0)),
    (1100, 50, 64, 300, 200, dict(hot=True, temperature=3.0)),
    (640, 64, 768, 10007, 5, dict(ignored=0.7, alpha=0.9)),
    (128, 128, 1000, 30011, 31, dict(labels=False, temperature=16.0)),
    (4096, 2048, 129, 6001, 12, dict(alpha=1.0)),
    (1500, 1500, 64, 900, 1, dict(absent=0.6, temperature=1.0, alpha=0.75)),
    (70, 70, 64, 500, 9, dict(alpha=0.0)),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("packed", [True, False], ids=["packed", "dense"])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_the_formulas(cuda_rt, case, packed, dtype):
    rows, time, d, vocab, k, more = case
    s = student(rows, time, d, vocab, dtype, packed, k, seed=rows + vocab, top_dtype=list(TOP_TYPES)[rows % 3], **more)
    steps = max(1, time - 1)
    loss_scale = 2.0 ** math.ceil(math.log2(steps)) / steps
    got = call(cuda_rt, s, loss_scale=loss_scale)
    check(got, formulas(s, loss_scale=loss_scale))
    again = call(cuda_rt, s, loss_scale=loss_scale)
    for a, b in zip(got, again):
        assert (a is None and b is None) or torch.equal(a, b)


def test_pieces_of_the_vocabulary(cuda_rt):
    """More than 2^28 logits: entries of later pieces, and groups of columns that the first piece ends at."""
    s = student(4096, 4096, 64, 70001, "f16", True, 40, seed=3, temperature=2.0)
    check(call(cuda_rt, s), formulas(s))


def test_a_teacher_that_is_sure_is_the_label(cuda_rt):
    """One entry per row, the next token: cross-entropy, whatever the teacher's share; the gradients are head_ce_grad's but for the
    order of a few additions."""
    s = inputs(600, 200, 128, 999, "f16", True, 0.2, seed=5)
    after = torch.roll(s["labels"], -1)
    want = cuda_rt.head_ce_grad(s["hidden"], s["weight"], s["labels"], scale=s["scale"], bias=s["bias"], ignore_id=-1, time=200)
    for alpha in (0.0, 0.5, 1.0):
        s.update(alpha=alpha, temperature=1.0, top_ids=after[:, None].contiguous(), top_logits=torch.zeros(600, 1, device="cuda"))
        check(call(cuda_rt, s), formulas(s))
        got = call(cuda_rt, s)
        assert torch.allclose(got.row_loss, want.row_loss, rtol=0, atol=2e-5) and torch.allclose(got.bias, want.bias, rtol=0, atol=2e-4)


def test_masked_entries(cuda_rt):
    """Negative ids hide whatever their logits are; -infinity and the type's lowest value are probabilities of 0; rows without an entry
    have the first part alone."""
    for labels in (True, False):
        for dtype in ("f32", "f16", "bf16"):
            s = student(300, 100, 64, 700, "bf16", False, 12, labels=labels, holes=0.4, absent=0.2, top_dtype=dtype, seed=9)
            t = s["top_logits"].dtype
            gone = s["top_ids"] < 0
            fill = torch.tensor([math.nan, math.inf, -math.inf, 7.0], device="cuda", dtype=t)[torch.arange(300 * 12, device="cuda").view(300, 12) % 4]
            s["top_logits"] = torch.where(gone, fill, s["top_logits"])
            s["top_logits"][::3, 5] = -math.inf
            s["top_logits"][1::3, 2] = torch.finfo(t).min
            s["top_logits"][4] = -math.inf                   # ids without a probability among them
            s["top_ids"][7] = torch.arange(12, device="cuda").to(torch.int32)
            s["top_logits"][7] = torch.finfo(t).min          # all the same
            got = call(cuda_rt, s)
            check(got, formulas(s))
            if not labels:
                assert got.row_loss[4] == 0 and (got.hidden[4] == 0).all()


def test_an_id_that_comes_twice(cuda_rt):
    s = student(200, 100, 64, 130, "f16", True, 10, seed=4)
    s["top_ids"][:, 3] = s["top_ids"][:, 1]
    s["top_ids"][::2, 7] = s["top_ids"][::2, 1]
    s["top_ids"][50:60] = 77
    check(call(cuda_rt, s), formulas(s))


def test_rows_that_teach_nothing_sound(cuda_rt):
    """Ids outside the vocabulary and logits that are no numbers: a loss of NaN and no gradient; other rows as without them."""
    s = student(300, 100, 64, 700, "f16", True, 6, labels=False, seed=2)
    bad = torch.tensor([3, 40, 41, 299], device="cuda")
    s["top_ids"][3, 2] = 700
    s["top_ids"][40, 0] = 1 << 30
    s["top_logits"][41, 5] = math.nan
    s["top_logits"][299, 1] = math.inf
    got = call(cuda_rt, s)
    assert got.row_loss[bad].isnan().all() and (got.hidden[bad] == 0).all()
    s["top_ids"][bad] = -1
    want = call(cuda_rt, s)
    assert torch.equal(torch.nan_to_num(got.row_loss), want.row_loss)
    for a, b in zip(got[1:], want[1:]):
        assert torch.equal(a, b)
    # a label outside the vocabulary, and labels that are ignored whatever the teacher says there
    s = student(300, 100, 64, 700, "f16", True, 6, seed=2, ignored=0.2)
    s["labels"][11] = 700
    s["top_ids"][torch.roll(s["labels"], -1) == -1] = 5000
    got = call(cuda_rt, s)
    assert got.row_loss[10].isnan() and int(got.row_loss.isnan().sum()) == 1 and (got.hidden[10] == 0).all()


@pytest.mark.parametrize("alpha,temperature", [(0.5, 1.0), (0.5, 128.0), (0.5, 1 / 128), (1.0, 128.0), (1.0, 1 / 128)])
def test_the_range_of_temperatures(cuda_rt, alpha, temperature):
    s = student(200, 100, 64, 300, "f16", True, 8, alpha=alpha, temperature=temperature, seed=6)
    check(call(cuda_rt, s), formulas(s))


def test_rows_that_count_for_nothing(cuda_rt):
    for labels in (True, False):
        s = student(400, 100, 64, 300, "f16", True, 8, labels=labels, seed=6)
        if labels:
            s["labels"].fill_(-1)
        s["top_ids"].fill_(-1)
        s["hidden"].fill_(math.nan)
        got = call(cuda_rt, s)
        assert all((t == 0).all() for t in got)
    none = cuda_rt.head_distill_grad(s["hidden"][:0], s["weight"], s["top_ids"][:0], s["top_logits"][:0], scale=s["scale"], bias=s["bias"])
    assert none.row_loss.shape == (0,) and (none.weight == 0).all() and (none.scale == 0).all() and (none.bias == 0).all()


def test_shapes_and_views(cuda_rt):
    s = student(60, 20, 64, 300, "bf16", False, 8, seed=7, bias=False)
    want = call(cuda_rt, s)
    assert want.scale is None and want.bias is None
    cube = cuda_rt.head_distill_grad(s["hidden"].view(3, 20, 64), s["weight"], s["top_ids"].view(3, 20, 8), s["top_logits"].view(3, 20, 8),
                                     labels=s["labels"].view(3, 20), alpha=0.5, temperature=2.0, ignore_id=-1)
    assert cube.hidden.shape == (3, 20, 64) and torch.equal(cube.hidden.view(60, 64), want.hidden) and torch.equal(cube.weight, want.weight)
    wide = torch.full((60, 81), 9.0, device="cuda").bfloat16()
    wide[:, 3:67] = s["hidden"]
    s["hidden"] = wide[:, 3:67]
    got = call(cuda_rt, s)
    assert torch.equal(got.hidden, want.hidden) and torch.equal(got.row_loss, want.row_loss)


def test_a_replayed_graph_two_streams_and_workspaces_of_nan(cuda_rt):
    import ctypes as C
    s = student(1500, 100, 128, 900, "f16", True, 17, seed=8)
    call(cuda_rt, s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call(cuda_rt, s)
    for seed in (20, 21):
        other = student(1500, 100, 128, 900, "f16", True, 17, seed=seed, holes=0.2 * (seed - 20), ignored=0.4)
        for name in ("hidden", "weight", "labels", "scale", "bias", "top_ids", "top_logits"):
            s[name].copy_(other[name])
        graph.replay()
        check(got, formulas(s))
    others = [(student(700, 100, 128, 900, "f16", True, 17, seed=30 + i), torch.cuda.Stream()) for i in range(2)]
    torch.cuda.synchronize()
    found = []
    for o, stream in others * 2:
        with torch.cuda.stream(stream):
            found.append(call(cuda_rt, o))
    torch.cuda.synchronize()
    for (o, _), f in zip(others * 2, found):
        check(f, formulas(o))
    for labels in (True, False):
        s = student(500, 100, 96, 900, "f16", True, 17, seed=8, labels=labels)
        need = C.c_size_t(0)
        assert cuda_rt._lib.ullis_cuda_head_distill_grad_workspace(cuda_rt._h, 500, 96, 900, 17, int(labels), 1, C.byref(need)) == cuda.OK
        work = torch.full((need.value,), 0xFF, dtype=torch.uint8, device="cuda")
        want = call(cuda_rt, s)
        buffers = [torch.full((t.numel() + 9,), 77, dtype=t.dtype, device="cuda") for t in want]
        p = lambda t: None if t is None else t.data_ptr()   # noqa: E731
        assert cuda_rt._lib.ullis_cuda_head_distill_grad(
            cuda_rt._h, torch.cuda.current_stream().cuda_stream, 1, p(s["hidden"]), 96, p(s["weight"]), None, p(s["scale"]), p(s["bias"]),
            p(s["top_ids"]), 0, p(s["top_logits"]), 17, 0.5, 2.0, p(s["labels"]), 0xFFFFFFFF, 500, 100, 96, 900, 1.0,
            *(b.data_ptr() + b.element_size() for b in buffers), work.data_ptr(), need.value) == cuda.OK
        for b, t in zip(buffers, want):
            assert b[0] == 77 and (b[1 + t.numel():] == 77).all() and torch.equal(b[1:1 + t.numel()].view(t.shape), t)


def test_gradients_are_differences_of_the_loss(cuda_rt):
    """The loss along a direction of bias: differences of the row losses' sum in 64 bits over a step that FP16 biases hold."""
    s = student(64, 64, 64, 200, "bf16", False, 10, seed=12, alpha=0.6, temperature=2.0)
    s["bias"] = torch.zeros(200, device="cuda").half()
    got = call(cuda_rt, s)
    g = torch.Generator("cuda").manual_seed(1)
    way = torch.randint(-4, 5, (200,), generator=g, device="cuda").double()
    step = 2.0 ** -7
    sums = []
    for sign in (1, -1):
        s["bias"] = (sign * step * way).half()           # exact
        sums.append(call(cuda_rt, s).row_loss.double().sum())
    slope = (sums[0] - sums[1]) / (2 * step)
    # the third derivative of a log sum exp along `way` is at most the cube of its spread (8); the losses are off by 1e-5 each
    bound = 64 * 1.6 * 8.0 ** 3 * step ** 2 / 6 + 64 * 2e-5 / step
    want = (got.bias.double() * way).sum()
    assert abs(slope - want) <= bound and abs(want) > 2 * bound


def test_a_step_from_teacher_to_table(cuda_rt):
    """The operators of a distilled step one after the other: lookup, norm over the tape, the teacher's top logits, distillation, the
    norm's backward pass and the table's gradient, against 64-bit autograd of the same model in the forms the operators are given in."""
    rows, d, vocab, k = 512, 64, 300, 24
    g = torch.Generator("cuda").manual_seed(3)
    table = torch.randn(vocab, d, generator=g, device="cuda")
    tokens = (torch.rand(rows, generator=g, device="cuda") ** 3 * vocab).to(torch.int32)
    w, b = (1.0 + 0.1 * torch.randn(d, generator=g, device="cuda")).half(), (0.1 * torch.randn(d, generator=g, device="cuda")).half()
    head = (0.1 * torch.randn(vocab, d, generator=g, device="cuda")).bfloat16()
    teacher = cuda_rt.top_logits(2.0 * torch.randn(rows, vocab, generator=g, device="cuda"), k)
    scale = math.sqrt(d)
    x = cuda_rt.embed(table, tokens, scale=scale)
    y, tape = cuda_rt.tape_layer_norm(x, w, b)
    y16 = y.bfloat16()
    out = cuda_rt.head_distill_grad(y16, head, teacher.ids, teacher.logits, temperature=2.0)
    gx, _, _ = cuda_rt.tape_layer_norm_backward(tape, out.hidden.float(), w)
    got = cuda_rt.embed_grad(tokens, gx, vocab, scale=scale)
    # the same in 64 bits, each operator at the inputs that it was given
    y64, head64 = y16.double(), head.double()
    logits = (y64 @ head64.t()).requires_grad_()
    log_q = torch.log_softmax(logits / 2.0, 1).gather(1, teacher.ids.long())
    log_p = torch.log_softmax(teacher.logits.double() / 2.0, 1)
    loss = 4.0 * (log_p.exp() * (log_p - log_q)).sum(1)
    (gz,) = torch.autograd.grad(loss.sum(), logits)
    # logits of up to 4 and losses of up to 16 in f32, 64 + 300 + 24 terms behind them: below 400 roundings of 2^-24 of 32
    assert ((out.row_loss.double() - loss).abs() <= 400 * U * 32).all()
    # g is rounded to bf16 before its product with the head (half a step, 2^-8), the sum when it leaves; the f32 steps are below 2^-12
    gy = gz @ head64
    assert ((out.hidden.double() - gy).abs() <= (2.0 ** -8 + 2.0 ** -12) * (gz.abs() @ head64.abs() + gy.abs())).all()
    x64 = cuda_rt.tape_unpack(tape, torch.float32).double().requires_grad_()
    normed = torch.nn.functional.layer_norm(x64, (d,), w.double(), b.double(), 1e-5)
    (gx64,) = torch.autograd.grad(normed, x64, out.hidden.double())
    at = tokens.long()
    t64 = torch.zeros(vocab, d, dtype=torch.float64, device="cuda").index_add_(0, at, gx64) * scale
    # gx = inv * (dx - mean(dx) - xh * mean(dx * xh)): fewer than 4 * 64 + 32 roundings of 2^-24 of its terms' sizes; the rows' sum 512 more
    dx = (out.hidden.double() * w.double()).abs()
    centred = x64.detach() - x64.detach().mean(1, keepdim=True)
    inv = (centred.square().mean(1, keepdim=True) + 1e-5).rsqrt()
    xh = (centred * inv).abs()
    sizes = inv * (dx + dx.mean(1, keepdim=True) + xh * (dx * xh).mean(1, keepdim=True))
    off = torch.zeros_like(t64).index_add_(0, at, sizes) * scale * (4 * 64 + 32 + 520) * U
    assert ((got.double() - t64).abs() <= off).all()


@pytest.mark.parametrize("vocab", [(1 << 19) - 256, (1 << 19) + 70])
def test_large_vocabularies(cuda_rt, vocab):
    """Sort keys of the entries in 32 bits up to 524 032 columns, in 64 beyond them."""
    s = student(70, 70, 8, vocab, "bf16", False, 30, seed=2)
    s["top_ids"][:, 4] = vocab - 1 - torch.arange(70, device="cuda").to(torch.int32) % 3
    s["top_ids"][::2, 9] = s["top_ids"][::2, 4]
    check(call(cuda_rt, s), formulas(s))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("temperature", [2.0, 4.0, 1.9999999, 3.0])
def test_temperatures_that_are_squared(cuda_rt, temperature, dtype):
    """At 2 and 4 the first softmax comes of the second's squares; sure rows, whose other columns' exps are far below 1, with them."""
    for lean in (1.0, 8.0):
        s = student(700, 100, 96, 1500, dtype, True, 24, temperature=temperature, lean=lean, seed=11, absent=0.2)
        check(call(cuda_rt, s), formulas(s))


def test_the_library_refuses(cuda_rt):
    """Statuses of the entry point itself; nothing is written."""
    import ctypes as C
    s = student(40, 20, 64, 300, "f16", False, 8, seed=7)
    need = C.c_size_t(0)
    lib, h = cuda_rt._lib, cuda_rt._h
    for top, code in ((0, cuda.ERR_SHAPE), (257, cuda.ERR_SHAPE), (8, cuda.OK)):
        assert lib.ullis_cuda_head_distill_grad_workspace(h, 40, 64, 300, top, 1, 0, C.byref(need)) == code
    work = torch.zeros(need.value, dtype=torch.uint8, device="cuda")
    outs = [torch.full((n,), 77, dtype=t, device="cuda") for n, t in ((40, torch.float32), (40 * 64, torch.float16), (300 * 64, torch.float16), (300, torch.float32))]

    def go(dtype=1, ids=s["top_ids"].data_ptr(), top_dtype=0, logits=s["top_logits"].data_ptr(), top=8, alpha=0.5, temperature=2.0,
           labels=s["labels"].data_ptr(), time=20, weight=s["weight"].data_ptr(), loss_scale=1.0, size=need.value, g_scale=None):
        return lib.ullis_cuda_head_distill_grad(h, torch.cuda.current_stream().cuda_stream, dtype, s["hidden"].data_ptr(), 64, None, weight, None,
                                                s["bias"].data_ptr(), ids, top_dtype, logits, top, alpha, temperature, labels, 0xFFFFFFFF, 40, time, 64,
                                                300, loss_scale, outs[0].data_ptr(), outs[1].data_ptr(), outs[2].data_ptr(), g_scale, outs[3].data_ptr(),
                                                work.data_ptr(), size)

    nan, inf = float("nan"), float("inf")
    for bad in (dict(dtype=0), dict(top_dtype=5), dict(ids=None), dict(logits=None), dict(logits=s["top_logits"].data_ptr() + 1), dict(alpha=-0.1),
                dict(alpha=1.1), dict(alpha=nan), dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=nan), dict(temperature=inf),
                dict(temperature=129.0), dict(weight=None), dict(loss_scale=inf), dict(labels=s["labels"].data_ptr() + 1), dict(g_scale=outs[3].data_ptr())):
        assert go(**bad) == cuda.ERR_ARG, bad
    for bad in (dict(top=0), dict(top=257), dict(time=3), dict(time=0), dict(size=need.value - 1)):
        assert go(**bad) == cuda.ERR_SHAPE, bad
    torch.cuda.synchronize()
    assert all((o == 77).all() for o in outs)
    assert go() == cuda.OK
    torch.cuda.synchronize()
    assert all(not (o == 77).all() for o in outs)


@pytest.mark.parametrize("labels", [True, False])
def test_small_shares(cuda_rt, labels):
    """A small alpha without labels, a low temperature: FP16 keeps as many bits of small gradients as of large ones."""
    s = student(300, 100, 64, 700, "f16", True, 12, labels=labels, alpha=1.0 if labels else 0.01, temperature=1 / 64, seed=9)
    got, want = call(cuda_rt, s), formulas(s)
    check(got, want)
    value, _ = want["hidden"]
    # the operand's rounding, half a step of each term; what leaves is 6e-6, where FP16 has steps of 2^-24: half of one more
    assert ((got.hidden.double() - value).abs() <= 2.0 ** -9 * value.abs().max() + 2.0 ** -25).all()
    # the same gradients lifted by the loss scale to where FP16 has all its bits
    got, (value, _) = call(cuda_rt, s, loss_scale=8192.0), formulas(s, loss_scale=8192.0)["hidden"]
    assert ((got.hidden.double() - value).abs() <= 2.0 ** -9 * value.abs().max() + 2.0 ** -25).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("packed", [True, False], ids=["packed", "dense"])
@pytest.mark.parametrize("rows,time,d,vocab,k,more", [
    (32, 32, 256, 8192, 16, dict()), (1, 1, 64, 300, 1, dict(labels=False)), (128, 16, 100, 513, 40, dict(ignored=0.4, temperature=3.0)),
    (127, 127, 72, 1000, 5, dict(labels=False, absent=0.5, temperature=1.0)), (100, 50, 64, 77, 30, dict(hot=True)), (16, 4, 8, 70_000, 3, dict())])
def test_few_rows_keep_more_of_their_gradients(cuda_rt, rows, time, d, vocab, k, more, packed, dtype):
    """Up to 128 rows g * scale is the sum of two 16-bit numbers: off by half a step of half a step."""
    s = student(rows, time, d, vocab, dtype, packed, k, seed=rows, **more)
    half = torch.finfo(TYPES[dtype]).eps / 2
    check(call(cuda_rt, s), formulas(s, operand=half * half))


def test_few_rows_by_pieces_of_the_vocabulary(cuda_rt):
    """So few rows that their logits reach 2^28 only beyond 2^20 columns."""
    s = student(4, 4, 8, (1 << 20) + 300, "f16", False, 6, seed=2)
    s["top_ids"][:, 1] = (1 << 20) + 17
    half = torch.finfo(torch.float16).eps / 2
    check(call(cuda_rt, s), formulas(s, operand=half * half))


@pytest.mark.parametrize("temperature", [1.0, 2.0, 3.0])
def test_columns_that_a_bias_masks(cuda_rt, temperature):
    """A bias of -infinity takes columns out: the others' results are those of the smaller vocabulary, the masked ones' gradients are zero."""
    s = student(400, 100, 64, 1100, "bf16", False, 9, temperature=temperature, seed=14)
    s["labels"] = s["labels"] % 800
    s["top_ids"] = s["top_ids"] % 800
    s["bias"][800:] = -math.inf
    small = dict(s, weight=s["weight"][:800].contiguous(), bias=s["bias"][:800].contiguous())
    got, want = call(cuda_rt, s), formulas(small)
    assert (got.weight[800:] == 0).all() and (got.bias[800:] == 0).all()
    check(got._replace(weight=got.weight[:800], bias=got.bias[:800]), want)
    # a masked column that the teacher has: its row's loss is infinite, as the formula's, and no number is lost
    s["top_ids"][5, 0] = 900
    got = call(cuda_rt, s)
    assert got.row_loss[5] == math.inf and int(got.row_loss.isinf().sum()) == 1 and got.hidden.isfinite().all() and got.weight.isfinite().all()


@pytest.mark.parametrize("labels,alpha,temperature", [(True, 0.5, 2.0), (True, 0.3, 3.0), (True, 0.6, 1.0), (False, 1.0, 1.0), (False, 1.0, 2.5)])
@pytest.mark.parametrize("rows", [64, 1300])
def test_a_target_of_one_sign(cuda_rt, rows, labels, alpha, temperature):
    """The target's logit (the label's, or the teacher's likeliest) is a sum of 4096 positive terms, every other logit zero.  The target is added
    with rounding: a lane's 128 terms one after the other and five steps between lanes, 133 * 2^-24 of the sum at most, of which the tensor
    cores would cut off 2.7e-5.  The loss moves by (1 - alpha) * (1 - q) + alpha * T * (1 - q_T) of that, the bias's gradient by
    (1 - alpha) * q * (1 - q) + alpha * q_T * (1 - q_T), at most a quarter a row."""
    d, vocab = 4096, 400
    g = torch.Generator("cuda").manual_seed(rows)
    hidden = (0.5 + torch.rand(rows, d, generator=g, device="cuda")).half()
    weight = torch.zeros(vocab, d, dtype=torch.float16, device="cuda")
    weight[7] = ((0.5 + torch.rand(d, generator=g, device="cuda")) * (math.log(vocab) * temperature / d)).half()
    ids = torch.tensor([300, 7, -1], dtype=torch.int32, device="cuda").repeat(rows, 1)
    said = torch.tensor([-40.0 * temperature, 2.0, 90.0], device="cuda").repeat(rows, 1)
    token = torch.full((rows,), 7, dtype=torch.int32, device="cuda") if labels else None
    s = dict(hidden=hidden, weight=weight, scale=None, bias=torch.zeros(vocab, dtype=torch.float16, device="cuda"), labels=token, time=rows,
             top_ids=ids, top_logits=said, alpha=alpha, temperature=temperature)
    got, want = call(cuda_rt, s), formulas(s)
    z = (hidden.double() @ weight[7].double())
    hard = (1.0 - alpha) if labels else 0.0
    off = 133 * U * z
    q, q_t = torch.sigmoid(z - math.log(vocab - 1)), torch.sigmoid(z / temperature - math.log(vocab - 1))
    steps = 2.0 ** -20 * (1.0 + temperature ** 2)   # exp, log and the sums of the loss's terms, of sizes up to 1 and T^2 times a few
    bound = (hard * (1 - q) + alpha * temperature * (1 - q_t)) * off + 8 * steps
    assert ((got.row_loss.double() - want["row_loss"][0]).abs() <= bound).all()
    bias = want["bias"][0][7]
    moves = ((hard * q * (1 - q) + alpha * q_t * (1 - q_t)) * off).sum() + (hard + alpha * temperature) * rows * 2.0 ** -20
    assert abs(got.bias[7].double() - bias) <= moves
