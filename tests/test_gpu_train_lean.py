"""Training steps that keep little (CudaTrainState.set_lean) against the CPU restatement of the step: the head in pieces within
the same tolerances as the ordinary step, the 8-bit tape within them of a step whose residual streams are what the tape stands for."""
import numpy as np
import pytest

import test_gpu_train as base
from oracle import train as T
from ullis_b200 import cuda, synth

pytestmark = pytest.mark.gpu


def tape_values(x, rows, c):
    """What the 8-bit tape of x stands for (numpy, by the definition)."""
    out = np.empty((rows, c), np.float64)
    x = np.asarray(x, np.float64).reshape(rows, c)
    for c0 in range(0, c, 32):
        b = x[:, c0:c0 + 32]
        m, e = np.frexp(np.abs(b).max(1, keepdims=True))
        step = np.exp2(np.maximum(np.where(m <= 127 / 128, e - 7, e - 6), -126).astype(np.float64))
        out[:, c0:c0 + 32] = np.round(b / step) * step
    return out.astype(np.float32).ravel()


def keep_on_tape(ref, oracle):
    """The restatement's backward pass takes its residual streams from here: let them be what the tape stands for."""
    plain = ref.m.forward_ce

    def forward_ce(tokens, labels, ignore_id, batch, time, taps=None, **more):
        out = plain(tokens, labels, ignore_id, batch, time, taps, **more)
        if taps is not None:
            rows, d, t = batch * time, ref.m.d, ref.m.t
            for l in range(ref.m.layers):
                x = tape_values(taps[f"{l}.after_rosa"], rows, d)
                taps[f"{l}.after_rosa"] = x
                taps[f"{l}.ln2_out"] = oracle.layer_norm(x, t[f"blocks.{l}.ln2.weight"], t[f"blocks.{l}.ln2.bias"], rows, d)
        return out

    ref.m.forward_ce = forward_ce


def compare(ref, st, oracle, lr):
    for name in ref.fp16_names():
        w = ref.m.t[name]
        a = oracle.fp16_to_f32(w) + ref.residual[name]
        b = oracle.fp16_to_f32(st.read(name, np.uint16, w.size)) + st.read(name + ".residual", np.float32, w.size)
        assert np.abs(a - b).max() <= lr * base.GRAD_TOL, name
    for prefix in ref.packed_names():
        lat = ref.latent[prefix]
        a = oracle.fp16_to_f32(lat) + ref.residual[prefix + ".latent"]
        b = oracle.fp16_to_f32(st.read(prefix + ".latent", np.uint16, lat.size)) + \
            st.read(prefix + ".latent.residual", np.float32, lat.size)
        assert np.abs(a - b).max() <= lr * base.GRAD_TOL, prefix


FORMS = {"head": (False, True), "tape": (True, False), "both": (True, True)}


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("case", base.CASES)
def test_steps_match_the_cpu_restatement(cuda_rt, oracle, case, form):
    shape, B, Tn, lr, steps = base.CASES[case]
    tape8, head_pieces = FORMS[form]
    data = synth.heron_checkpoint(shape, batch_size=B, seed=11, ln_gain_one=not case.startswith("benchmark"))
    ref = T.HeronTrainer(data)
    if tape8:
        keep_on_tape(ref, oracle)
    m = cuda.CudaHeron(cuda_rt, data)
    st = m.train_state()
    st.set_lean(tape8=tape8, head_pieces=head_pieces)
    tokens = synth.zipf_tokens(5, B * Tn, ref.m.vocab)
    for s in range(steps):
        want = ref.train_step(tokens, tokens, oracle.CE_NO_IGNORE, B, Tn, lr)
        got = st.train_step(tokens, tokens, oracle.CE_NO_IGNORE, B, Tn, lr)
        assert got["n_valid"] == want["n_valid"] == B * (Tn - 1)
        assert abs(got["loss"] - want["loss"]) <= base.LOSS_TOL, (s, got, want)
        for k in ("flips_head", "flips_cmix", "flips_rosa_o"):
            assert abs(got[k] - want[k]) <= max(2, 0.02 * want[k]), (s, k, got, want)
    compare(ref, st, oracle, lr)


def test_ignored_labels(cuda_rt, oracle):
    shape, B, Tn = (64, 1, 260, 40, 96), 2, 40
    data = synth.heron_checkpoint(shape, batch_size=B, seed=2, ln_gain_one=True)
    ref = T.HeronTrainer(data)
    keep_on_tape(ref, oracle)
    st = cuda.CudaHeron(cuda_rt, data).train_state()
    st.set_lean()
    tokens = synth.zipf_tokens(9, B * Tn, 260)
    labels = tokens.copy()
    labels.reshape(B, Tn)[:, 25:] = 3
    want = ref.train_step(tokens, labels, 3, B, Tn, 0.05)
    got = st.train_step(tokens, labels, 3, B, Tn, 0.05)
    assert got["n_valid"] == want["n_valid"] and abs(got["loss"] - want["loss"]) <= base.LOSS_TOL
    compare(ref, st, oracle, 0.05)
    emb = st.read("embedding", np.uint16, 260 * 64)
    r = st.train_step(tokens, np.full_like(tokens, 3), 3, B, Tn, 0.05)
    assert r["n_valid"] == 0 and r["loss"] == 0.0 and r["flips_head"] == 0
    assert np.array_equal(st.read("embedding", np.uint16, 260 * 64), emb)


def test_to_and_fro(cuda_rt, oracle):
    """Off again, a step gives what it gave before; two states of one model may keep differently."""
    data = synth.heron_checkpoint(synth.CONFIGS["tiny"], batch_size=2, seed=4, ln_gain_one=True)
    tokens = synth.zipf_tokens(5, 128, 512)

    def embedding_after(*forms):
        st = cuda.CudaHeron(cuda_rt, data).train_state()
        for f in forms:
            st.set_lean(*f)
        st.train_step(tokens, tokens, oracle.CE_NO_IGNORE, 2, 64, 0.05)
        return st.read("embedding", np.uint16, 512 * 64)

    plain = embedding_after()
    assert np.array_equal(embedding_after((True, True), (False, False)), plain)
    lean = embedding_after((True, True))
    m = cuda.CudaHeron(cuda_rt, data)
    a, b = m.train_state(), m.train_state()
    a.set_lean(True, True)
    a.train_step(tokens, tokens, oracle.CE_NO_IGNORE, 2, 64, 0.05)
    assert np.array_equal(a.read("embedding", np.uint16, 512 * 64), lean)
    b.train_step(tokens, tokens, oracle.CE_NO_IGNORE, 2, 64, 0.05)
    a.train_step(tokens, tokens, oracle.CE_NO_IGNORE, 2, 64, 0.05)
    assert np.isfinite(b.train_step(tokens, tokens, oracle.CE_NO_IGNORE, 2, 64, 0.05)["loss"])


def test_refusals(cuda_rt, oracle):
    data = synth.heron_checkpoint((64, 1, 260, 40, 96), batch_size=2, seed=2, ln_gain_one=True)
    tokens = synth.zipf_tokens(9, 80, 260)
    st = cuda.CudaHeron(cuda_rt, data).train_state()
    st.set_lean(tape8=True, head_pieces=True)
    cuda_rt.set_mode(cuda.MODE_EXACT)
    try:
        with pytest.raises(cuda.UllisCudaError) as e:
            st.train_step(tokens, tokens, oracle.CE_NO_IGNORE, 2, 40, 0.05)
        assert e.value.code == cuda.ERR_ARG and "MODE_FAST" in e.value.message
        st.set_lean(tape8=True, head_pieces=False)            # the tape alone goes in either mode
        assert np.isfinite(st.train_step(tokens, tokens, oracle.CE_NO_IGNORE, 2, 40, 0.05)["loss"])
    finally:
        cuda_rt.set_mode(cuda.MODE_FAST)
    assert st._lib.ullis_cuda_train_state_set_lean(None, 1, 1) == cuda.ERR_ARG
