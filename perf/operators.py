"""The operators of a training step that keeps little: the head's cross-entropy with its gradient and without logits, and
activations kept in 8 bits with what the backward pass takes from them.

A case names an operator (`op`) and its sizes.  Everything is on the device: torch tensors go in and come out, as a
program that holds its activations there calls `CudaRuntime`.

The 8-bit tape of x [rows, channels]: blocks of 32 consecutive channels of a row (the last one may be shorter) with one
exponent e each, the smallest one >= -126 with 127 * 2^e >= max |x| of the block; codes round(x * 2^-e), ties to even,
int8; the exponent is stored as the byte e + 127.  A code stands for code * 2^e.
"""
from __future__ import annotations

import functools
import math

import torch

own = False

EPS = 1e-5
BLOCK = 32
IGNORED = -1
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # one short window of the small model: what a first training step or a test runs; launches and latency
        {"name": "head one window", "op": "head", "rows": 32, "time": 32, "d": 256, "vocab": 8192, "packed": True,
         "dtype": "f16", "ignored": 0.0},
        # the training batch of the default model: 8 contexts
        {"name": "head default batch", "op": "head", "rows": 16384, "time": 2048, "d": 512, "vocab": 8192, "packed": True,
         "dtype": "f16", "ignored": 0.0},
        # conversations cut to an odd length, the user's half of the tokens unsupervised, a vocabulary of no round size
        {"name": "head ragged chat", "op": "head", "rows": 7655, "time": 1531, "d": 256, "vocab": 10007, "packed": True,
         "dtype": "bf16", "ignored": 0.5},
        # a dense 16-bit head over a large vocabulary: the largest call
        {"name": "head large vocabulary", "op": "head", "rows": 4096, "time": 2048, "d": 512, "vocab": 131072, "packed": False,
         "dtype": "bf16", "ignored": 0.0},
        # LayerNorm of one window, forward with the tape and backward from it
        {"name": "norm one window", "op": "norm", "rows": 512, "channels": 256, "dtype": "f32"},
        # the residual stream of the default model's training batch
        {"name": "norm default batch", "op": "norm", "rows": 16384, "channels": 512, "dtype": "f32"},
        # the headline workload's 64 contexts in 16 bits
        {"name": "norm 64 contexts", "op": "norm", "rows": 131072, "channels": 512, "dtype": "bf16"},
        # weight gradient of the feed-forward key for one context
        {"name": "weight gradient one context", "op": "weight", "rows": 2048, "in": 512, "out": 2048, "dtype": "f16"},
        # ... for the default batch
        {"name": "weight gradient batch", "op": "weight", "rows": 16384, "in": 512, "out": 2048, "dtype": "bf16"},
        # weight gradient of the feed-forward value, ragged contexts
        {"name": "weight gradient ragged", "op": "weight", "rows": 7655, "in": 2048, "out": 512, "dtype": "f16"},
        # activations to 8 bits and back: the default batch
        {"name": "tape default batch", "op": "tape", "rows": 16384, "channels": 512, "dtype": "f32"},
        # ... and a width that ends inside a block
        {"name": "tape ragged", "op": "tape", "rows": 7655, "channels": 1000, "dtype": "bf16"},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["head", "head", "head", "norm", "norm", "weight", "weight", "tape"])
    if op == "head":
        d = rng.choice([64, 200, 256, 512, 512, 768, 1000, 1024])
        vocab = _log(rng, 300, 131072)
        most = 4096 * 131072 * 512 // (max(d, 512) * vocab)
        time = _log(rng, 2, min(2048, most))
        rows = time * max(1, min(most, _log(rng, 1, 16384)) // time)
        return {"op": op, "rows": rows, "time": time, "d": d, "vocab": vocab, "packed": rng.random() < 0.6,
                "dtype": rng.choice(["f16", "bf16"]), "ignored": rng.choice([0.0, 0.0, 0.3, 0.7])}
    if op == "weight":
        return {"op": op, "rows": _log(rng, 1, 16384), "in": rng.choice([64, 250, 256, 512, 1024, 2048]),
                "out": rng.choice([64, 200, 512, 1000, 2048]), "dtype": rng.choice(["f16", "bf16"])}
    channels = rng.choice([64, 256, 500, 512, 768, 1000, 1024, 2048])
    return {"op": op, "rows": _log(rng, 1, 131072 * 512 // channels), "channels": channels,
            "dtype": rng.choice(["f32", "f16", "bf16"])}


# ------------------------------------------------------------------------------------------------ inputs
def _activations(rows, channels, g):
    """Residual stream: channels of different size, a few of them far above the others."""
    size = torch.exp(0.5 * torch.randn(channels, generator=g, device="cuda"))
    size = torch.where(torch.rand(channels, generator=g, device="cuda") < 0.01, 20.0 * size, size)
    return torch.randn(rows, channels, generator=g, device="cuda") * size


def prepare(case, seed):
    g = torch.Generator("cuda")
    g.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    randn = functools.partial(torch.randn, generator=g, device="cuda")
    rand = functools.partial(torch.rand, generator=g, device="cuda")
    s = {"op": case["op"], "dtype": dtype}
    if case["op"] == "head":
        rows, d, vocab = case["rows"], case["d"], case["vocab"]
        # token ids fall off like words do
        labels = torch.clamp(torch.exp(rand(rows) * math.log(vocab)) - 1.0, 0, vocab - 1).to(torch.int32)
        target = torch.cat([labels[1:], labels[:1]]).long()
        hidden = randn(rows, d)
        # a model in training leans towards the target, at some positions hardly and at some by much
        lean = 2.0 * rand(rows, 1)
        if case["packed"]:
            words = (vocab * d + 31) // 32
            bits = torch.randint(-(1 << 31), 1 << 31, (words,), generator=g, device="cuda", dtype=torch.int64).to(torch.int32)
            s["weight"] = bits
            s["scale"] = (0.005 + 0.015 * rand(vocab)).to(torch.float16)
            # signs of the targets' rows
            at = target[:, None] * d + torch.arange(d, device="cuda")
            hidden += lean * (2.0 * ((bits[at >> 5] >> (at & 31)) & 1).float() - 1.0)
        else:
            s["weight"] = (randn(vocab, d) * 0.0125).to(dtype)
            s["scale"] = None
            hidden += lean * torch.sign(s["weight"][target].float())
        s["hidden"] = hidden.to(dtype)
        s["bias"] = (0.01 * randn(vocab)).to(torch.float16)
        s["labels"] = torch.where(rand(rows) < case["ignored"], torch.full_like(labels, IGNORED), labels)
        s["time"] = case["time"]
        # the mean over a sequence, times the power of two that keeps 16-bit gradients clear of the smallest numbers
        steps = max(1, case["time"] - 1)
        s["loss_scale"] = 2.0 ** math.ceil(math.log2(steps)) / steps
    elif case["op"] == "norm":
        rows, c = case["rows"], case["channels"]
        s["x"] = _activations(rows, c, g).to(dtype)
        s["gy"] = (1e-2 * randn(rows, c)).to(dtype)
        s["residual"] = (1e-2 * randn(rows, c)).to(dtype)   # the gradient that comes past the norm
        s["weight"] = (1.0 + 0.02 * randn(c)).to(torch.float16)
        s["bias"] = (0.02 * randn(c)).to(torch.float16)
    elif case["op"] == "weight":
        # the tape lies in memory since the forward pass
        s["codes"], s["exponents"] = _pack(_activations(case["rows"], case["in"], g))
        s["gy"] = (1e-2 * randn(case["rows"], case["out"])).to(dtype)
    else:
        s["x"] = _activations(case["rows"], case["channels"], g).to(dtype)
    return s


# ------------------------------------------------------------------------------------------------ plain form
def _blocks(x):
    c = x.shape[1]
    more = -c % BLOCK
    if more:
        x = torch.cat([x, x.new_zeros(x.shape[0], more)], 1)
    return x.reshape(x.shape[0], -1, BLOCK)


def _pack(x):
    b = _blocks(x.float())
    m, e = torch.frexp(b.abs().amax(2))                       # amax = m * 2^e, 0.5 <= m < 1
    e = torch.where(m <= 127.0 / 128.0, e - 7, e - 6).clamp(min=-126)
    codes = torch.round(torch.ldexp(b, -e[:, :, None])).to(torch.int8)
    return codes.reshape(x.shape[0], -1)[:, : x.shape[1]].contiguous(), (e + 127).to(torch.uint8)


def _unpack(codes, exponents):
    e = exponents.to(torch.int32) - 127
    return torch.ldexp(_blocks(codes.float()), e[:, :, None]).reshape(codes.shape[0], -1)[:, : codes.shape[1]]


def _signs(bits, vocab, d):
    at = torch.arange(vocab * d, device=bits.device).reshape(vocab, d)
    return 2.0 * ((bits[at >> 5] >> (at & 31)) & 1).float() - 1.0


def _targets(labels, time):
    """The token after each row, and whether there is one that counts."""
    rows = labels.numel()
    at = torch.arange(rows, device=labels.device)
    after = torch.cat([labels[1:], labels.new_full((1,), IGNORED)])
    valid = ((at % time) + 1 < time) & (after != IGNORED)
    return torch.where(valid, after, torch.zeros_like(after)).long(), valid


def _head(s):
    h, dtype = s["hidden"].float(), s["dtype"]
    vocab, d = s["bias"].numel(), h.shape[1]
    w = s["weight"].float() if s["scale"] is None else _signs(s["weight"], vocab, d)
    target, valid = _targets(s["labels"], s["time"])
    plain = h @ w.t()
    z = (plain if s["scale"] is None else plain * s["scale"].float()) + s["bias"].float()
    top = z.amax(1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(1, keepdim=True)
    loss = top[:, 0] + torch.log(total[:, 0]) - z.gather(1, target[:, None])[:, 0]
    gz = e / total
    gz.scatter_add_(1, target[:, None], gz.new_full((h.shape[0], 1), -1.0))
    gz = torch.where(valid[:, None], gz, torch.zeros_like(gz)) * s["loss_scale"]
    gs = gz if s["scale"] is None else gz * s["scale"].float()
    return {"row_loss": torch.where(valid, loss, torch.zeros_like(loss)),
            "hidden": (gs @ w).to(dtype), "weight": (gs.t() @ h).to(dtype),
            "scale": None if s["scale"] is None else (gz * plain).sum(0), "bias": gz.sum(0)}


def _norm(s):
    def statistics(x):
        mean = x.mean(1, keepdim=True)
        return x - mean, 1.0 / torch.sqrt((x - mean).square().mean(1, keepdim=True) + EPS)

    w, b, dtype = s["weight"].float(), s["bias"].float(), s["dtype"]
    centred, inv = statistics(s["x"].float())
    y = centred * inv * w + b
    centred, inv = statistics(_unpack(*_pack(s["x"])))        # the backward pass has the tape alone
    xh, gy = centred * inv, s["gy"].float()
    dx = gy * w
    gx = s["residual"].float() + inv * (dx - dx.mean(1, keepdim=True) - xh * (dx * xh).mean(1, keepdim=True))
    return {"y": y.to(dtype), "gx": gx.to(dtype), "weight": (gy * xh).sum(0), "bias": gy.sum(0)}


# ------------------------------------------------------------------------------------------------ one pass
@functools.lru_cache(None)
def _runtime():
    from ullis_b200.cuda import CudaRuntime

    return CudaRuntime(torch.cuda.current_device())


def run(state):
    s = state
    if s["op"] == "head":
        if own:
            r = _runtime().head_ce_grad(s["hidden"], s["weight"], s["labels"], scale=s["scale"], bias=s["bias"],
                                        ignore_id=IGNORED, time=s["time"], loss_scale=s["loss_scale"])
            return {"row_loss": r.row_loss, "hidden": r.hidden, "weight": r.weight, "scale": r.scale, "bias": r.bias}
        return _head(s)
    if s["op"] == "norm":
        if own:
            y, tape = _runtime().tape_layer_norm(s["x"], s["weight"], s["bias"])
            gx, gw, gb = _runtime().tape_layer_norm_backward(tape, s["gy"], s["weight"], residual=s["residual"])
            return {"y": y, "gx": gx, "weight": gw, "bias": gb}
        return _norm(s)
    if s["op"] == "weight":
        if own:
            return _runtime().tape_weight_grad((s["codes"], s["exponents"]), s["gy"])
        return s["gy"].float().t() @ _unpack(s["codes"], s["exponents"])
    if own:
        return _runtime().tape_unpack(_runtime().tape_pack(s["x"]), s["dtype"])
    return _unpack(*_pack(s["x"])).to(s["dtype"])


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "head":
        rows, d, vocab = case["rows"], case["d"], case["vocab"]
        # hidden, weights, scales, biases and labels in; losses and the gradients of all of them out
        weights = vocab * d / 8 + 2 * vocab if case["packed"] else vocab * d * size
        vectors = 4 * vocab * (2 if case["packed"] else 1) + 2 * vocab
        counted = rows * (1.0 - case["ignored"]) * (1.0 - 1.0 / case["time"])
        # the logits and the two gradient products, over the rows that count
        return {"bytes": 2 * rows * d * size + 8 * rows + weights + vocab * d * size + vectors, "flops": 6.0 * counted * vocab * d}
    if case["op"] == "weight":
        rows, i, o = case["rows"], case["in"], case["out"]
        return {"bytes": rows * (i + -(-i // BLOCK)) + rows * o * size + 4 * i * o, "flops": 2.0 * rows * i * o}
    rows, c = case["rows"], case["channels"]
    tape = rows * (c + -(-c // BLOCK))
    if case["op"] == "tape":
        return {"bytes": 2 * tape + 2 * rows * c * size, "flops": 4.0 * rows * c}
    # forward: x in, y and tape out; backward: tape, gy and the other gradient in, gx out
    return {"bytes": 2 * tape + 5 * rows * c * size + 12 * c, "flops": 20.0 * rows * c}


# ------------------------------------------------------------------------------------------------ 64 bits
def _exact_tape(x):
    """What the 8-bit tape of x stands for."""
    x = x.double()
    out = torch.empty_like(x)
    for c in range(0, x.shape[1], BLOCK):
        b = x[:, c : c + BLOCK]
        top = b.abs().amax(1, keepdim=True)
        e = torch.ceil(torch.log2(torch.clamp(top, min=1e-300) / 127.0))
        e = torch.where(127.0 * torch.exp2(e) < top, e + 1.0, torch.where(127.0 * torch.exp2(e - 1.0) >= top, e - 1.0, e))
        step = torch.exp2(torch.clamp(e, min=-126.0))
        out[:, c : c + BLOCK] = torch.round(b / step) * step
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "tape":
        return _exact_tape(s["x"])
    if case["op"] == "weight":
        i = case["in"]
        step = torch.exp2(s["exponents"].double() - 127.0).repeat_interleave(BLOCK, 1)[:, :i]
        return torch.einsum("ro,ri->oi", s["gy"].double(), s["codes"].double() * step)
    if case["op"] == "norm":
        w, gy = s["weight"].double(), s["gy"].double()

        def normed(x):
            var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
            inv = (var + EPS).rsqrt()
            return (x - mean) * inv, inv

        y = normed(s["x"].double())[0] * w + s["bias"].double()
        xh, inv = normed(_exact_tape(s["x"]))
        dx = gy * w
        gx = s["residual"].double() + inv * (dx - dx.mean(1, keepdim=True) - xh * (dx * xh).mean(1, keepdim=True))
        return {"y": y, "gx": gx, "weight": torch.einsum("rc,rc->c", gy, xh), "bias": gy.sum(0)}
    h, vocab, d, packed = s["hidden"].double(), case["vocab"], case["d"], case["packed"]
    rows, time, labels = case["rows"], case["time"], s["labels"].long()
    counts = torch.zeros(rows, dtype=torch.bool, device=h.device)
    counts[:-1] = labels[1:] != IGNORED
    counts[time - 1 :: time] = False
    if packed:   # bit (v * d + c) of the words, the lowest bit of a word first
        words = s["weight"].view(torch.uint8)
        w = torch.stack([(words >> k) & 1 for k in range(8)], 1).reshape(-1)[: vocab * d].reshape(vocab, d)
        w = 2.0 * w.double() - 1.0
        scale = s["scale"].double()
    else:
        w = s["weight"].double()
        scale = torch.ones(vocab, dtype=torch.float64, device=h.device)
    products = h @ w.t()
    logits = torch.addcmul(s["bias"].double(), products, scale)
    log_total = torch.logsumexp(logits, 1)
    row = torch.nonzero(counts)[:, 0]
    target = labels[row + 1]
    loss = torch.zeros(rows, dtype=torch.float64, device=h.device)
    loss[row] = log_total[row] - logits[row, target]
    g = logits.sub_(log_total[:, None]).exp_()
    g[row, target] -= 1.0
    g *= (counts * s["loss_scale"])[:, None]
    g_scale = torch.einsum("rv,rv->v", g, products) if packed else None
    g_bias = g.sum(0)
    g *= scale
    return {"row_loss": loss, "hidden": g @ w, "weight": g.t() @ h, "scale": g_scale, "bias": g_bias}
