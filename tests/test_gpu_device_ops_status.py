"""Operators on a caller's stream: a kernel whose bounded wait runs out is reported to the next call of the runtime, whatever call that
is, and to no other one."""
import numpy as np
import pytest
import torch

from ullis_b200 import cuda, synth

pytestmark = pytest.mark.gpu


def give_up(rt):
    """Nothing ever arrives on the barrier of the self-test's kernel: it gives up after some milliseconds and returns."""
    stream = torch.cuda.Stream()
    rt.wait_selftest_on(stream.cuda_stream)
    stream.synchronize()


X = np.arange(8, dtype=np.float32)
CALLS = {
    "synchronize": lambda rt: rt.synchronize(),
    "host arrays": lambda rt: rt.residual_add(X, X),
    "device memory": lambda rt: rt.tape_pack(torch.ones(4, 64, device="cuda")),
    "zero rows": lambda rt: rt.tape_pack(torch.ones(0, 64, device="cuda")),
    "a setting": lambda rt: rt.set_mode(cuda.MODE_FAST),
}


@pytest.mark.parametrize("call", CALLS.values(), ids=CALLS.keys())
def test_the_next_call_is_told_and_the_one_after_is_not(cuda_rt, call):
    for _ in range(2):
        give_up(cuda_rt)
        with pytest.raises(cuda.UllisCudaError) as e:
            call(cuda_rt)
        assert e.value.code == cuda.ERR_TIMEOUT and "earlier call" in e.value.message and "99" in e.value.message
        call(cuda_rt)
    cuda_rt.synchronize()


def test_models_and_states_are_told(cuda_rt, oracle):
    m = cuda.CudaHeron(cuda_rt, synth.heron_checkpoint("tiny", batch_size=2))
    tokens = synth.zipf_tokens(11, 128, 512)
    want = m.forward_ce(tokens, tokens, cuda.CE_NO_IGNORE, 2, 64)
    state = m.train_state()
    for call in (lambda: m.forward_ce(tokens, tokens, cuda.CE_NO_IGNORE, 2, 64),
                 lambda: state.train_step(tokens, tokens, cuda.CE_NO_IGNORE, 2, 64, 0.05)):
        give_up(cuda_rt)
        with pytest.raises(cuda.UllisCudaError) as e:
            call()
        assert e.value.code == cuda.ERR_TIMEOUT
    assert m.forward_ce(tokens, tokens, cuda.CE_NO_IGNORE, 2, 64) == want      # neither call did anything


def test_refusals(cuda_rt):
    for polls in (0, (1 << 20) + 1):
        with pytest.raises(cuda.UllisCudaError) as e:
            cuda_rt.wait_selftest_on(0, polls)
        assert e.value.code == cuda.ERR_ARG
    cuda_rt.synchronize()
