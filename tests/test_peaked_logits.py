"""Peaked logit rows: the running maximum of a row moves far past the lazy
threshold in the middle of the vocabulary, in some rows of a warp and not in
others, which makes the tensor-core rank sums rescale their accumulator in
TMEM.  Tolerances as the step's other parity tests (loss 1e-4, gradients 1e-3
relative L2)."""
import os

import numpy as np
import pytest

import lora_ce
import workload as wl

pytestmark = pytest.mark.gpu

NTHREADS = os.cpu_count() or 8


def rel(a, b):
    return float(np.linalg.norm(np.asarray(a, np.float64) - b) / max(np.linalg.norm(b), 1e-30))


@pytest.mark.parametrize("V,d,r,T", [
    (4099, 128, 16, 150),
    (4099, 128, 32, 300),    # in place probabilities, two rank groups
    (3000, 192, 64, 260),    # separate probability tile
    (49152, 576, 16, 129),
    (2048, 576, 4, 300),     # the per-logit epilogue, for comparison
])
def test_step_on_peaked_rows(oracle, V, d, r, T):
    rng = np.random.default_rng(V + r + T)
    W = (rng.standard_normal((V, d)) / np.sqrt(d)).astype(np.float16)
    _, tgt, A, B = wl.make_step_inputs(5, T, V, d, r)
    h = rng.standard_normal((T, d))
    # two of three rows point at a token of their own, anywhere in the vocabulary
    ids = rng.integers(0, V, T)
    boost = np.where(np.arange(T) % 3 == 0, 0.0, rng.uniform(12.0, 24.0, T))
    h += boost[:, None] * W[ids].astype(np.float64)
    tgt = np.where(np.arange(T) % 2 == 0, ids, tgt).astype(np.int32)
    H = wl.f32_to_bf16_bits(h.astype(np.float32))
    Wb = W.view(np.uint16)
    m = lora_ce.LoraCE(lora_ce.default_config(d, V, r, T, scale=2.0, lr=1e-3))
    m.set_weight(Wb)
    m.set_adapter(A, B, 0)
    loss = m.step(H, tgt)
    gA, gB, _, _ = m.get_grads()
    m.close()
    ref = oracle.step(Wb, A, B, wl.oracle_hidden(H), tgt, 2.0, 1e-3, nthreads=NTHREADS)
    assert abs(loss - ref["loss"]) <= 1e-4 * abs(ref["loss"])
    assert rel(gA, ref["gA"]) <= 1e-3
    assert rel(gB, ref["gB"]) <= 1e-3
