"""What the Python layer of embedding, top logits and distillation refuses before it calls the library; no device needed."""
import numpy as np
import pytest
import torch

from test_device_ops_host import Fake

from ullis_b200 import cuda

H, F, I32 = torch.float16, torch.float32, torch.int32


def ids(*shape):
    return torch.zeros(*shape, dtype=I32)


def distill(rt, **more):
    a = dict(hidden=torch.zeros(4, 64, dtype=H), weight=torch.zeros(9, 64, dtype=H), top_ids=ids(4, 3), top_logits=torch.zeros(4, 3))
    a.update(more)
    return rt.head_distill_grad(a.pop("hidden"), a.pop("weight"), a.pop("top_ids"), a.pop("top_logits"), **a)


REFUSED = {
    "embed: an array": (lambda rt: rt.embed(np.zeros((4, 64), np.float32), ids(3)), cuda.ERR_ARG),
    "embed: table's type": (lambda rt: rt.embed(torch.zeros(4, 64, dtype=torch.float64), ids(3)), cuda.ERR_ARG),
    "embed: table's dimensions": (lambda rt: rt.embed(torch.zeros(2, 4, 64), ids(3)), cuda.ERR_SHAPE),
    "embed: a transposed table": (lambda rt: rt.embed(torch.zeros(64, 4).t(), ids(3)), cuda.ERR_SHAPE),
    "embed: 64-bit tokens": (lambda rt: rt.embed(torch.zeros(4, 64), ids(3).long()), cuda.ERR_ARG),
    "embed: tokens on another device": (lambda rt: rt.embed(torch.zeros(4, 64), torch.zeros(3, dtype=I32, device="meta")), cuda.ERR_ARG),
    "embed: tokens with gaps": (lambda rt: rt.embed(torch.zeros(4, 64), ids(6)[::2]), cuda.ERR_SHAPE),
    "embed: to integers": (lambda rt: rt.embed(torch.zeros(4, 64), ids(3), dtype=I32), cuda.ERR_ARG),
    "embed: ignore_id": (lambda rt: rt.embed(torch.zeros(4, 64), ids(3), ignore_id=1 << 32), cuda.ERR_ARG),
    "embed gradient: tokens": (lambda rt: rt.embed_grad(ids(5), torch.zeros(4, 64), 9), cuda.ERR_SHAPE),
    "embed gradient: 64-bit tokens": (lambda rt: rt.embed_grad(ids(4).long(), torch.zeros(4, 64), 9), cuda.ERR_ARG),
    "embed gradient: gy's type": (lambda rt: rt.embed_grad(ids(4), torch.zeros(4, 64, dtype=torch.float64), 9), cuda.ERR_ARG),
    "embed gradient: one dimension": (lambda rt: rt.embed_grad(ids(4), torch.zeros(4), 9), cuda.ERR_SHAPE),
    "embed gradient: no vocabulary": (lambda rt: rt.embed_grad(ids(4), torch.zeros(4, 64), 0), cuda.ERR_SHAPE),
    "embed gradient: ignore_id": (lambda rt: rt.embed_grad(ids(4), torch.zeros(4, 64), 9, ignore_id=-(1 << 31) - 1), cuda.ERR_ARG),
    "top: integers": (lambda rt: rt.top_logits(ids(4, 64), 3), cuda.ERR_ARG),
    "top: one dimension": (lambda rt: rt.top_logits(torch.zeros(64), 3), cuda.ERR_SHAPE),
    "top: none": (lambda rt: rt.top_logits(torch.zeros(4, 64), 0), cuda.ERR_SHAPE),
    "top: more than there are": (lambda rt: rt.top_logits(torch.zeros(4, 64), 65), cuda.ERR_SHAPE),
    "top: more than 256": (lambda rt: rt.top_logits(torch.zeros(4, 640), 257), cuda.ERR_SHAPE),
    "top: rows on top of each other": (lambda rt: rt.top_logits(torch.zeros(1, 64).expand(4, 64), 3), cuda.ERR_SHAPE),
    "top: transposed": (lambda rt: rt.top_logits(torch.zeros(64, 4).t(), 3), cuda.ERR_SHAPE),
    "distill: f32": (lambda rt: distill(rt, hidden=torch.zeros(4, 64)), cuda.ERR_ARG),
    "distill: weight's type": (lambda rt: distill(rt, weight=torch.zeros(9, 64)), cuda.ERR_ARG),
    "distill: channels": (lambda rt: distill(rt, weight=torch.zeros(9, 32, dtype=H)), cuda.ERR_SHAPE),
    "distill: 64-bit ids": (lambda rt: distill(rt, top_ids=ids(4, 3).long()), cuda.ERR_ARG),
    "distill: integer logits": (lambda rt: distill(rt, top_logits=ids(4, 3)), cuda.ERR_ARG),
    "distill: ids and logits": (lambda rt: distill(rt, top_logits=torch.zeros(4, 2)), cuda.ERR_SHAPE),
    "distill: rows": (lambda rt: distill(rt, top_ids=ids(5, 3), top_logits=torch.zeros(5, 3)), cuda.ERR_SHAPE),
    "distill: no entries": (lambda rt: distill(rt, top_ids=ids(4, 0), top_logits=torch.zeros(4, 0)), cuda.ERR_SHAPE),
    "distill: more than 256": (lambda rt: distill(rt, top_ids=ids(4, 257), top_logits=torch.zeros(4, 257)), cuda.ERR_SHAPE),
    "distill: gaps": (lambda rt: distill(rt, top_ids=ids(4, 6)[:, ::2]), cuda.ERR_SHAPE),
    "distill: transposed logits": (lambda rt: distill(rt, top_logits=torch.zeros(3, 4).t()), cuda.ERR_SHAPE),
    "distill: labels": (lambda rt: distill(rt, labels=ids(5)), cuda.ERR_SHAPE),
    "distill: 64-bit labels": (lambda rt: distill(rt, labels=ids(4).long()), cuda.ERR_ARG),
    "distill: time": (lambda rt: distill(rt, labels=ids(4), time=3), cuda.ERR_SHAPE),
    "distill: alpha": (lambda rt: distill(rt, alpha=1.5), cuda.ERR_ARG),
    "distill: alpha is NaN": (lambda rt: distill(rt, alpha=float("nan")), cuda.ERR_ARG),
    "distill: temperature": (lambda rt: distill(rt, temperature=0.0), cuda.ERR_ARG),
    "distill: temperature is infinite": (lambda rt: distill(rt, temperature=float("inf")), cuda.ERR_ARG),
    "distill: bias": (lambda rt: distill(rt, bias=torch.zeros(8, dtype=H)), cuda.ERR_SHAPE),
    "distill: packed without words": (lambda rt: distill(rt, scale=torch.zeros(9, dtype=H)), cuda.ERR_ARG),
    "distill: ignore_id": (lambda rt: distill(rt, labels=ids(4), ignore_id=1 << 32), cuda.ERR_ARG),
}


@pytest.mark.parametrize("call,code", REFUSED.values(), ids=REFUSED.keys())
def test_refused_before_the_library_is_called(call, code):
    with pytest.raises(cuda.UllisCudaError) as e:
        call(Fake())
    assert e.value.code == code
