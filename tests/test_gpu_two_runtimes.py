"""Two runtimes of one device, each with a thread and a stream of its own, as the header allows: a function's limit of dynamic shared
memory belongs to the device, so what one thread's calls ask of it must not come in between the other's."""
import threading

import pytest
import torch

from ullis_b200.cuda import CudaRuntime

pytestmark = pytest.mark.gpu

CALLS = 20_000


class Recorded(CudaRuntime):
    """A runtime whose last call can be made again as it was, without the steps in Python that lie between two calls."""

    def _workspace(self, *args):
        self.kept = super()._workspace(*args)
        return self.kept

    def record(self, entry, call):
        plain, runtime = self._lib, self

        class Lib:
            def __getattr__(self, name):
                function = getattr(plain, name)
                if name != entry:
                    return function

                def go(*args):
                    runtime.again = lambda: function(*args)
                    return function(*args)
                return go

        self._lib = Lib()
        try:
            return call(self)
        finally:
            self._lib = plain


def top(rows):
    x = torch.randn(rows, 16384, device="cuda")
    return lambda rt: rt.top_logits(x, 200)


def distill(rows, k):
    g = torch.Generator("cuda").manual_seed(k)
    hidden, weight = torch.randn(rows, 64, generator=g, device="cuda").half(), torch.randn(600, 64, generator=g, device="cuda").half()
    ids = torch.argsort(torch.rand(rows, 600, generator=g, device="cuda"), 1)[:, :k].to(torch.int32).contiguous()
    said = torch.randn(rows, k, generator=g, device="cuda")
    return lambda rt: rt.head_distill_grad(hidden, weight, ids, said)


def embed(rows):
    tokens, gy = (torch.arange(rows, device="cuda") * 7919 % 503).to(torch.int32), torch.ones(rows, 1, device="cuda")
    return lambda rt: rt.embed_grad(tokens, gy, 503)


PAIRS = {   # two calls of one kernel that need different sizes of shared memory
    "top_logits": lambda: (top(1), top(300)),
    "head_distill_grad": lambda: (distill(8, 256), distill(8, 130)),
    "embed_grad": lambda: (embed(11 * 16384), embed(7 * 16384)),
}


@pytest.mark.parametrize("entry", PAIRS)
def test_two_threads(entry):
    calls = PAIRS[entry]()
    runtimes, streams = [Recorded(0), Recorded(0)], [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    found, wanted = [], []
    for rt, stream, call in zip(runtimes, streams, calls):
        with torch.cuda.stream(stream):
            out = rt.record("ullis_cuda_" + entry, call)
            found.append([t for t in (out if isinstance(out, tuple) else (out,)) if t is not None])
            wanted.append([t.clone() for t in found[-1]])
    torch.cuda.synchronize()
    start, refused = threading.Barrier(2), [0, 0]

    def work(i):
        start.wait(60)
        for k in range(CALLS):
            refused[i] += runtimes[i].again() != 0
            if k % 200 == 199:
                streams[i].synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert refused == [0, 0]
    for got, want in zip(found, wanted):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    for rt in runtimes:
        rt.close()
