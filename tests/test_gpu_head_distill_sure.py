"""CudaRuntime.head_distill_grad on rows that the student is sure of: gradients of 1e-12 to 1e-4, to relative bounds.

As in test_gpu_head_grad.py hidden states are multiples of 1/8 and weights +-1, so the products are exact in any order, and a logit in
units of ln 2, below 64, is off by the roundings of its scale, its bias and itself, 3 * 2^-24 * 64.  A probability takes two logits, a sum
of 400 terms and the logarithm of a softmax's share beside that sum's: off by less than
2 * 1.2e-5 * ln 2 + 80 * 2^-24 + 2^-21 + 3 * 2^-24 * 64 * ln 2 < 2^-14 relatively; a weight of the teacher's by far less."""
import math

import pytest
import torch

from test_gpu_head_distill import call
from test_gpu_head_grad import TYPES, U, inputs, signs

pytestmark = pytest.mark.gpu

OFF = 2.0 ** -14
VOCAB, D = 400, 1000


def sure(rows, dtype, seed, extra=0, labels=True, alpha=0.5, temperature=1.0):
    """A student that leans to the next token, a teacher that says the same; `extra` entries more, 12 * temperature below it."""
    g = torch.Generator("cuda").manual_seed(seed)
    s = inputs(rows, rows, D, VOCAB, dtype, True, lean=2.0, seed=seed)
    after = torch.roll(s["labels"], -1).long()
    h = ((torch.randn(rows, D, generator=g, device="cuda") * 8).round() / 8).clamp(-6, 6) + 2.0 * signs(s["weight"], VOCAB, D)[after].float()
    s["hidden"] = h.to(TYPES[dtype])
    assert torch.equal(s["hidden"].float(), h)
    s["scale"].clamp_(max=0.0155)
    others = (after[:, None] + 1 + torch.arange(extra, device="cuda") * 37) % VOCAB
    s["top_ids"] = torch.cat([others, after[:, None]], 1).to(torch.int32)
    s["top_logits"] = torch.zeros(rows, extra + 1, device="cuda")
    s["top_logits"][:, :extra] -= 12.0 * temperature
    s.update(alpha=alpha, temperature=temperature)
    if not labels:
        s["labels"] = None
    return s, after


def gradient(s, after):
    """(products, g, what g is made of) in 64 bits; of the target's column the sums over the others."""
    rows = len(after)
    at = torch.arange(rows, device="cuda")
    a = s["hidden"].double() @ signs(s["weight"], VOCAB, D).t()
    z = a * s["scale"].double() + s["bias"].double()
    assert z.abs().max() / math.log(2.0) < 64
    hard = 0.0 if s["labels"] is None else 1.0 - s["alpha"]
    soft = s["alpha"] * s["temperature"]
    x = s["top_logits"].double() / s["temperature"]
    said = torch.zeros_like(z).scatter_(1, s["top_ids"].long(), soft * torch.softmax(x, 1))
    g, sizes = -said, said.clone()
    g[at, after] = said.sum(1) - said[at, after]
    sizes[at, after] = g[at, after]
    for share, times in ((hard, 1.0), (soft, 1.0 / s["temperature"])):
        rest = torch.exp(z * times).scatter(1, after[:, None], 0.0)
        hit = torch.exp(z[at, after] * times)
        q = rest / (rest.sum(1) + hit)[:, None]
        g += share * q
        sizes += share * q
        g[at, after] -= share * rest.sum(1) / (rest.sum(1) + hit)
        sizes[at, after] += share * rest.sum(1) / (rest.sum(1) + hit)
    if s["labels"] is not None:
        g[-1] = sizes[-1] = 0.0
    return a, g, sizes


CASES = {"cross-entropy alone": dict(alpha=0.0), "one entry": dict(), "teacher alone": dict(labels=False, alpha=1.0),
         "teacher alone, T = 2": dict(labels=False, alpha=1.0, temperature=2.0), "T = 2": dict(temperature=2.0), "T = 3": dict(temperature=3.0),
         "T = 4": dict(alpha=0.9, temperature=4.0), "three entries": dict(extra=2), "three entries, T = 2": dict(extra=2, temperature=2.0)}


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [100, 128, 129, 600])
def test_gradients_of_sure_rows(cuda_rt, rows, dtype, case):
    s, after = sure(rows, dtype, 5, **CASES[case])
    loss_scale = 65536.0 if dtype == "f16" else 1.0   # FP16 gradients of this size need one
    got = call(cuda_rt, s, loss_scale=loss_scale)
    a, g, sizes = gradient(s, after)
    at = torch.arange(rows - 1, device="cuda")
    if case == "cross-entropy alone":
        assert g[at, after[:-1]].abs().median() < 1e-4
    # the operand g * scale in 16 bits, of few rows the sum of two such numbers; FP16's smallest steps beside the largest scale at 2^14
    t = TYPES[dtype]
    half = torch.finfo(t).eps / 2
    hard = 0.0 if s["labels"] is None else 1.0 - s["alpha"]
    scale = s["scale"].double()
    gs_off = (OFF * sizes + (half * half if rows <= 128 else half) * g.abs()) * scale
    if dtype == "f16":
        room = max(0, math.ceil(math.log2(hard + s["alpha"] * s["temperature"])))
        gs_off = gs_off + 2.0 ** -25 / 2.0 ** (14 - room - math.floor(math.log2(scale.max().item())))
    lowest = torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2
    w, h, gs = signs(s["weight"], VOCAB, D), s["hidden"].double(), g * scale
    for x, value, off, size, terms in ((got.hidden, gs @ w, gs_off @ w.abs(), gs.abs() @ w.abs(), VOCAB),
                                       (got.weight, gs.t() @ h, gs_off.t() @ h.abs(), gs.abs().t() @ h.abs(), rows)):
        value = value * loss_scale
        off = (off + 2 * U * terms * size) * loss_scale + half * value.abs() + lowest + 4 * U * value.abs()
        assert ((x.double() - value).abs() <= off).all()


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [100, 128, 129, 600])
def test_sums_over_sure_rows(cuda_rt, rows, dtype, case):
    s, after = sure(rows, dtype, 5, **CASES[case])
    loss_scale = 65536.0 if dtype == "f16" else 1.0   # FP16 gradients of this size need one
    got = call(cuda_rt, s, loss_scale=loss_scale)
    a, g, sizes = gradient(s, after)
    # what is summed over the rows: U a row, and the sums' own additions
    for x, times in ((got.bias, torch.ones_like(a)), (got.scale, a)):
        value = (g * times).sum(0) * loss_scale
        off = (OFF + U * (32 + rows)) * (sizes * times.abs()).sum(0) * loss_scale
        assert ((x.double() - value).abs() <= off).all()


@pytest.mark.parametrize("rows", [4, 260])
def test_by_pieces_of_the_vocabulary(cuda_rt, rows):
    """Sure of a token in the last piece of a vocabulary of more than 2^20 columns: its bias is 30 above the others'.  The sums of the others'
    exp are off by (80 + 2^20 / 256) * 2^-24 and their logits, below 50 in units of ln 2, by 4 * 2^-24 * 50 each: below 2^-11 in all."""
    vocab, token, d = (1 << 20) + 300, (1 << 20) + 17, 8
    g = torch.Generator("cuda").manual_seed(rows)
    hidden = torch.randn(rows, d, generator=g, device="cuda").half()
    weight = (0.1 * torch.randn(vocab, d, generator=g, device="cuda")).half()
    bias = torch.zeros(vocab, device="cuda").half()
    bias[token] = 30.0
    z = hidden.double() @ weight.double().t() + bias.double()
    for alpha, temperature in ((0.0, 1.0), (0.5, 1.0), (1.0, 1.0)):
        s = dict(hidden=hidden, weight=weight, scale=None, bias=bias, labels=torch.full((rows,), token, dtype=torch.int32, device="cuda"), time=rows,
                 top_ids=torch.tensor([[token, 5]], dtype=torch.int32, device="cuda").repeat(rows, 1), alpha=alpha, temperature=temperature,
                 top_logits=torch.tensor([[0.0, -math.inf]], device="cuda").repeat(rows, 1))
        got = call(cuda_rt, s)
        rest = torch.exp(z - z[:, token:token + 1])
        rest[:, token] = 0.0
        value = -(rest.sum(1) / (1.0 + rest.sum(1)))[:-1].sum()
        assert abs(got.bias[token].double() - value) <= 2.0 ** -11 * -value and value > -1e-6 * rows
        del rest
