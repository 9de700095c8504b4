"""The operators of a student that learns from a teacher, on device memory: the embedding lookup it starts with and the gradient
of its table, the teacher's largest logits, and the head's distillation from them with its gradient and without logits.

A case names an operator (`op`) and its sizes.  Everything is on the device: torch tensors go in and come out, as a program
that holds its activations there calls `CudaRuntime`.

Distillation: with z the student's logits, T the temperature, p = softmax(top_logits / T) over the entries of a row (a negative
id is no entry), y the next token and alpha the teacher's share,
  row_loss = (1 - alpha) * (log sum exp z - z[y]) + alpha * T^2 * sum p * (log p - log softmax(z / T)).
With labels a row counts as in next-token cross-entropy, without them where it has an entry; a row that counts and has no
entry has the first part alone.
"""
from __future__ import annotations

import functools
import math

import torch

own = False

IGNORED = -1
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # the tokens of one window of the small model
        {"name": "embed one window", "op": "embed", "tokens": 512, "d": 256, "vocab": 8192, "table": "f16", "dtype": "f16"},
        # the default model's training batch, into its residual stream
        {"name": "embed default batch", "op": "embed", "tokens": 16384, "d": 512, "vocab": 8192, "table": "f16", "dtype": "f32"},
        # what comes back to the table from one window: launches and latency
        {"name": "embed gradient one window", "op": "embed_grad", "tokens": 512, "d": 256, "vocab": 8192, "dtype": "f16"},
        # ... from the residual stream of the training batch; a seventh of the tokens are the most frequent one
        {"name": "embed gradient default batch", "op": "embed_grad", "tokens": 16384, "d": 512, "vocab": 8192, "dtype": "f32"},
        # ... from conversations of an odd length in a large vocabulary, most of whose rows no token names
        {"name": "embed gradient ragged", "op": "embed_grad", "tokens": 76550, "d": 500, "vocab": 50021, "dtype": "bf16"},
        # what a teacher says at one window
        {"name": "top one window", "op": "top", "rows": 32, "vocab": 8192, "k": 16, "dtype": "f32"},
        # ... at every position of a training batch
        {"name": "top default batch", "op": "top", "rows": 16384, "vocab": 8192, "k": 64, "dtype": "f32"},
        # ... a teacher with a large vocabulary
        {"name": "top large vocabulary", "op": "top", "rows": 4096, "vocab": 131072, "k": 64, "dtype": "bf16"},
        # one window of the small model: a first step or a test
        {"name": "distill one window", "op": "distill", "rows": 32, "time": 32, "d": 256, "vocab": 8192, "packed": True, "k": 16,
         "dtype": "f16", "labels": True, "alpha": 0.5, "temperature": 2.0, "absent": 0.0},
        # the training batch of the default model, teacher and text in equal parts
        {"name": "distill default batch", "op": "distill", "rows": 16384, "time": 2048, "d": 512, "vocab": 8192, "packed": True,
         "k": 64, "dtype": "f16", "labels": True, "alpha": 0.5, "temperature": 2.0, "absent": 0.0},
        # conversations of an odd length from the teacher alone, which answered at half of the positions
        {"name": "distill ragged chat", "op": "distill", "rows": 7655, "time": 1531, "d": 256, "vocab": 10007, "packed": True,
         "k": 20, "dtype": "bf16", "labels": False, "alpha": 1.0, "temperature": 1.0, "absent": 0.5},
        # a dense 16-bit head over a large vocabulary: the largest call
        {"name": "distill large vocabulary", "op": "distill", "rows": 4096, "time": 2048, "d": 512, "vocab": 131072,
         "packed": False, "k": 64, "dtype": "bf16", "labels": True, "alpha": 0.75, "temperature": 1.0, "absent": 0.0},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["embed", "embed_grad", "embed_grad", "top", "top", "distill", "distill", "distill"])
    if op in ("embed", "embed_grad"):
        d = rng.choice([64, 200, 256, 500, 512, 768, 1000, 1024])
        case = {"op": op, "tokens": _log(rng, 1, 76550 * 500 // max(d, 500)), "d": d,
                "vocab": _log(rng, 300, 50021 * 500 // max(d, 500)), "dtype": rng.choice(["f32", "f16", "bf16"])}
        if op == "embed":
            case["table"] = rng.choice(["f16", "f16", "bf16", "f32"])
        return case
    if op == "top":
        vocab, k = _log(rng, 300, 131072), _log(rng, 1, 256)
        return {"op": op, "rows": _log(rng, 1, min(16384, 4096 * 131072 // vocab)), "vocab": vocab, "k": k,
                "dtype": rng.choice(["f32", "f16", "bf16"])}
    d = rng.choice([64, 200, 256, 512, 512, 768, 1000, 1024])
    vocab = _log(rng, 300, 131072)
    most = 4096 * 131072 * 512 // (max(d, 512) * vocab)
    time = _log(rng, 2, min(2048, most))
    rows = time * max(1, min(most, _log(rng, 1, 16384)) // time)
    labels = rng.random() < 0.6
    return {"op": op, "rows": rows, "time": time, "d": d, "vocab": vocab, "packed": rng.random() < 0.6, "k": _log(rng, 1, 128),
            "dtype": rng.choice(["f16", "bf16"]), "labels": labels, "alpha": rng.choice([0.3, 0.5, 0.9]) if labels else 1.0,
            "temperature": rng.choice([1.0, 1.0, 1.5, 2.0, 4.0]), "absent": rng.choice([0.0, 0.0, 0.4])}


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator("cuda")
    g.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    randn = functools.partial(torch.randn, generator=g, device="cuda")
    rand = functools.partial(torch.rand, generator=g, device="cuda")
    s = {"op": case["op"], "dtype": dtype}

    def words(n, vocab):   # token ids fall off like words do
        return torch.clamp(torch.exp(rand(n) * math.log(vocab)) - 1.0, 0, vocab - 1).to(torch.int32)

    if case["op"] in ("embed", "embed_grad"):
        n, d, vocab = case["tokens"], case["d"], case["vocab"]
        s["tokens"], s["vocab"], s["scale"] = words(n, vocab), vocab, math.sqrt(d)
        if case["op"] == "embed":
            s["table"] = (0.02 * randn(vocab, d)).to(DTYPES[case["table"]])
        else:
            s["gy"] = (1e-2 * randn(n, d)).to(dtype)
        return s
    if case["op"] == "top":
        rows, vocab = case["rows"], case["vocab"]
        # frequent tokens are likely everywhere, others where they fit
        z = randn(rows, vocab).mul_(2.5).sub_(torch.log1p(torch.arange(vocab, device="cuda", dtype=torch.float32)).mul_(0.5))
        z[torch.arange(rows, device="cuda"), words(rows, vocab).long()] += 8.0
        s["logits"], s["k"] = z.to(dtype), case["k"]
        return s
    rows, d, vocab, k = case["rows"], case["d"], case["vocab"], case["k"]
    labels = words(rows, vocab)
    target = torch.cat([labels[1:], labels[:1]]).long()
    hidden = randn(rows, d)
    lean = 2.0 * rand(rows, 1)   # a model in training leans towards the target, at some positions hardly and at some by much
    if case["packed"]:
        n = (vocab * d + 31) // 32
        bits = torch.randint(-(1 << 31), 1 << 31, (n,), generator=g, device="cuda", dtype=torch.int64).to(torch.int32)
        s["weight"] = bits
        s["scale"] = (0.005 + 0.015 * rand(vocab)).to(torch.float16)
        at = target[:, None] * d + torch.arange(d, device="cuda")
        hidden += lean * (2.0 * ((bits[at >> 5] >> (at & 31)) & 1).float() - 1.0)
    else:
        s["weight"] = (randn(vocab, d) * 0.0125).to(dtype)
        s["scale"] = None
        hidden += lean * torch.sign(s["weight"][target].float())
    s["hidden"] = hidden.to(dtype)
    s["bias"] = (0.01 * randn(vocab)).to(torch.float16)
    # the teacher's entries: distinct ids, the more frequent the token the likelier, the target first, logits that fall off
    j = torch.arange(k, device="cuda")
    ids = (j + ((j + rand(rows, k)) / k) ** 3 * (vocab - k)).long().clamp_(max=vocab - 1)
    ids = ids.gather(1, torch.argsort(rand(rows, k), 1))
    ids = torch.where(ids == target[:, None], ids[:, :1], ids)
    ids[:, 0] = target
    top = 14.0 - 1.5 * torch.log1p(j.float()) - torch.cumsum(0.2 * rand(rows, k), 1) - 3.0 * rand(rows, 1) * (j > 0)
    absent = rand(rows, 1) < case["absent"]   # the teacher was not asked there
    s["top_ids"] = torch.where(absent, IGNORED, ids).to(torch.int32)
    s["top_logits"] = top.to(dtype)
    s["labels"] = labels if case["labels"] else None
    s["time"], s["alpha"], s["temperature"] = case["time"], case["alpha"], case["temperature"]
    # the mean over a sequence, times the power of two that keeps 16-bit gradients clear of the smallest numbers
    steps = max(1, case["time"] - 1)
    s["loss_scale"] = 2.0 ** math.ceil(math.log2(steps)) / steps
    return s


# ------------------------------------------------------------------------------------------------ plain form
def _embed(s):
    return (s["table"][s["tokens"].long()].float() * s["scale"]).to(s["dtype"])


def _embed_grad(s):
    g = torch.zeros(s["vocab"], s["gy"].shape[1], dtype=torch.float32, device=s["gy"].device)
    return g.index_add_(0, s["tokens"].long(), s["gy"].float()).mul_(s["scale"])


def _top(s):
    """The largest k of every row, in falling order, equal ones by rising index."""
    z = s["logits"]
    vocab = z.shape[1]
    bits = (z.float() + 0.0).view(torch.int32)                      # -0 is 0
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)          # as integers they stand in the order of the values
    key = (order.long() << 32) + (vocab - 1 - torch.arange(vocab, device=z.device))
    ids = vocab - 1 - (torch.topk(key, s["k"], 1).values & 0xFFFFFFFF)
    return {"ids": ids.to(torch.int32), "logits": z.gather(1, ids)}


def _signs(bits, vocab, d):
    at = torch.arange(vocab * d, device=bits.device).reshape(vocab, d)
    return 2.0 * ((bits[at >> 5] >> (at & 31)) & 1).float() - 1.0


def _distill(s):
    h, dtype, t, alpha = s["hidden"].float(), s["dtype"], s["temperature"], s["alpha"]
    rows, d = h.shape
    vocab = s["bias"].numel()
    w = s["weight"].float() if s["scale"] is None else _signs(s["weight"], vocab, d)
    entry = s["top_ids"] >= 0
    ids = torch.where(entry, s["top_ids"], 0).long()
    has = entry.any(1)
    if s["labels"] is None:
        counts, target = has, torch.zeros_like(ids[:, 0])
    else:
        after = torch.cat([s["labels"][1:], s["labels"].new_full((1,), IGNORED)])
        counts = (torch.arange(rows, device=h.device) % s["time"] + 1 < s["time"]) & (after != IGNORED)
        target = torch.where(counts, after, 0).long()
    # the teacher's probabilities and their logarithms
    said = torch.where(entry, s["top_logits"].float() / t, -torch.inf)
    said = said - torch.where(has, said.amax(1), 0.0)[:, None]
    log_p = said - torch.where(has, torch.exp(said).sum(1), 1.0).log()[:, None]
    p = torch.exp(log_p)
    log_p = torch.where(p > 0, log_p, 0.0)
    soft = (alpha * t * (counts & has))[:, None]
    hard = ((1.0 - alpha) * counts)[:, None]
    plain = h @ w.t()
    z = (plain if s["scale"] is None else plain * s["scale"].float()) + s["bias"].float()
    top = z.amax(1, keepdim=True)

    def softmax(times):
        e = torch.exp((z - top) * times)
        total = e.sum(1, keepdim=True)
        return e.div_(total), top * times + torch.log(total)

    q, lse = softmax(1.0 / t)
    loss = soft[:, 0] * t * (p * (log_p - z.gather(1, ids) / t + lse)).sum(1)
    gz = q.mul_(soft)
    gz.scatter_add_(1, ids, -soft * p)
    if alpha < 1.0:
        q, lse = softmax(1.0)
        loss += hard[:, 0] * (lse - z.gather(1, target[:, None]))[:, 0]
        gz += q.mul_(hard)
        gz.scatter_add_(1, target[:, None], -hard)
    gz *= s["loss_scale"]
    gs = gz if s["scale"] is None else gz * s["scale"].float()
    return {"row_loss": torch.where(counts, loss, 0.0), "hidden": (gs @ w).to(dtype), "weight": (gs.t() @ h).to(dtype),
            "scale": None if s["scale"] is None else (gz * plain).sum(0), "bias": gz.sum(0)}


# ------------------------------------------------------------------------------------------------ one pass
@functools.lru_cache(None)
def _runtime():
    from ullis_b200.cuda import CudaRuntime

    return CudaRuntime(torch.cuda.current_device())


def run(state):
    s = state
    if s["op"] == "embed":
        return _runtime().embed(s["table"], s["tokens"], scale=s["scale"], dtype=s["dtype"]) if own else _embed(s)
    if s["op"] == "embed_grad":
        return _runtime().embed_grad(s["tokens"], s["gy"], s["vocab"], scale=s["scale"]) if own else _embed_grad(s)
    if s["op"] == "top":
        if own:
            r = _runtime().top_logits(s["logits"], s["k"])
            return {"ids": r.ids, "logits": r.logits}
        return _top(s)
    if own:
        r = _runtime().head_distill_grad(s["hidden"], s["weight"], s["top_ids"], s["top_logits"], scale=s["scale"], bias=s["bias"],
                                         labels=s["labels"], alpha=s["alpha"], temperature=s["temperature"], ignore_id=IGNORED,
                                         time=s["time"], loss_scale=s["loss_scale"])
        return {"row_loss": r.row_loss, "hidden": r.hidden, "weight": r.weight, "scale": r.scale, "bias": r.bias}
    return _distill(s)


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "embed":
        n, d = case["tokens"], case["d"]
        rows = min(n, case["vocab"])   # of the table
        return {"bytes": 4 * n + n * d * size + rows * d * (4 if case["table"] == "f32" else 2), "flops": 1.0 * n * d}
    if case["op"] == "embed_grad":
        n, d = case["tokens"], case["d"]
        return {"bytes": 4 * n + n * d * size + 4 * case["vocab"] * d, "flops": 1.0 * n * d}
    if case["op"] == "top":
        rows, k = case["rows"], case["k"]
        return {"bytes": rows * case["vocab"] * size + rows * k * (4 + size), "flops": 1.0 * rows * case["vocab"]}
    rows, d, vocab, k = case["rows"], case["d"], case["vocab"], case["k"]
    weights = vocab * d / 8 + 2 * vocab if case["packed"] else vocab * d * size
    vectors = 4 * vocab * (2 if case["packed"] else 1) + 2 * vocab
    counted = rows * (1.0 - 1.0 / case["time"]) if case["labels"] else rows * (1.0 - case["absent"])
    # hidden, weights, scales, biases, labels and the teacher's entries in; losses and all gradients out
    return {"bytes": 2 * rows * d * size + 8 * rows + rows * k * (4 + size) + weights + vocab * d * size + vectors,
            "flops": 6.0 * counted * vocab * d}


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "embed":
        return torch.nn.functional.embedding(s["tokens"], s["table"].double()) * s["scale"]
    if case["op"] == "embed_grad":
        # rows sorted by token, running sums, differences at the ends of the tokens' runs
        order = torch.argsort(s["tokens"], stable=True)
        counts = torch.bincount(s["tokens"], minlength=case["vocab"])
        sums = torch.zeros(case["tokens"] + 1, case["d"], dtype=torch.float64, device="cuda")
        torch.cumsum(s["gy"][order].double(), 0, out=sums[1:])
        ends = torch.cumsum(counts, 0)
        return (sums[ends] - sums[ends - counts]) * s["scale"]
    if case["op"] == "top":
        found = {"ids": [], "logits": []}
        for part in s["logits"].split(max(1, (1 << 27) // case["vocab"])):
            values, ids = torch.sort(part.double(), dim=1, descending=True, stable=True)
            found["ids"].append(ids[:, : case["k"]].to(torch.int32))
            found["logits"].append(values[:, : case["k"]].clone())
        return {name: torch.cat(parts) for name, parts in found.items()}
    rows, time, vocab, d = case["rows"], case["time"], case["vocab"], case["d"]
    t, alpha = case["temperature"], case["alpha"]
    h = s["hidden"].double()
    if case["packed"]:   # bit (v * d + c) of the words, the lowest bit of a word first
        octets = s["weight"].view(torch.uint8)
        w = torch.stack([(octets >> b) & 1 for b in range(8)], 1).reshape(-1)[: vocab * d].reshape(vocab, d)
        w = 2.0 * w.double() - 1.0
        scale = s["scale"].double()
    else:
        w, scale = s["weight"].double(), torch.ones(vocab, dtype=torch.float64, device="cuda")
    products = h @ w.t()
    logits = torch.addcmul(s["bias"].double(), products, scale)
    asked = s["top_ids"][:, 0] != IGNORED          # a row has all of its entries or none
    if case["labels"]:
        counted = torch.ones(rows, dtype=torch.bool, device="cuda")
        counted[time - 1 :: time] = False
    else:
        counted = asked
    loss = torch.zeros(rows, dtype=torch.float64, device="cuda")
    g = torch.zeros_like(logits)
    row = torch.nonzero(counted & asked)[:, 0]
    if row.numel() and alpha > 0:
        log_p = torch.log_softmax(s["top_logits"][row].double() / t, 1)
        log_q = torch.log_softmax(logits[row] / t, 1)
        ids = s["top_ids"][row].long()
        loss[row] += alpha * t * t * torch.nn.functional.kl_div(log_q.gather(1, ids), log_p, reduction="none", log_target=True).sum(1)
        q = log_q.exp_()
        q[torch.arange(row.numel(), device="cuda")[:, None], ids] -= log_p.exp()
        g[row] += alpha * t * q
        del q, log_q
    row = torch.nonzero(counted)[:, 0]
    if row.numel() and alpha < 1:
        target = s["labels"].long()[row + 1]
        loss[row] += (1 - alpha) * torch.nn.functional.cross_entropy(logits[row], target, reduction="none")
        q = torch.softmax(logits[row], 1)
        q[torch.arange(row.numel(), device="cuda"), target] -= 1.0
        g[row] += (1 - alpha) * q
        del q
    del logits
    g *= s["loss_scale"]
    g_scale = torch.einsum("rv,rv->v", g, products) if case["packed"] else None
    g_bias = g.sum(0)
    g *= scale
    return {"row_loss": loss, "hidden": g @ w, "weight": g.t() @ h, "scale": g_scale, "bias": g_bias}
