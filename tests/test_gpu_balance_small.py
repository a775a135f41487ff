"""Mean probabilities far below one: the router balance's sums are whole
numbers of 2^-80, so an expert that is hardly ever likely keeps the relative
precision of f32, in the form of small calls (one block) and of large ones."""
import numpy as np
import pytest

from fp8_util import F32
from test_gpu_balance import balance, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,E,S", [(80, 64, 1), (300, 130, 3), (3000, 64, 1), (5000, 128, 7), (2500, 300, 2)])
def test_small_probabilities(cuda_lib, T, E, S):
    rng = np.random.default_rng(T + E)
    z = rng.standard_normal((T, E)).astype(np.float32)
    for e, low in enumerate((9.0, 11.0, 16.0, 21.0, 25.0, 27.0, 29.0, 33.0, 37.0)):  # p from 1e-6 to 1e-18
        z[:, e] -= low
    idx = np.argsort(-z, 1, kind="stable")[:, :4].astype(np.int32)
    mask = (rng.random(T) < 0.9).astype(np.uint8)
    seq = np.concatenate([[0], np.sort(rng.integers(1, T, S - 1)), [T]])
    got, zv = balance(cuda_lib, z, F32, idx, mask, seq)
    counts, prob, loss, _ = reference(zv, idx, mask, seq, 0.01, 1.0)
    assert np.array_equal(got[0], counts)
    # a softmax in f32 (exponential, E terms, division) and its exponent's rounding, 2^-24 of x log2 e for x down to the
    # lowest logit's distance, 50 at most; then sums over tokens in pieces of any order; then units of 2^-80
    rel = (E + 16 + min(T, 1024) + 50 * 1.4427) * 2.0 ** -24
    assert prob.min() < 1e-15
    assert (np.abs(got[1] - prob) <= rel * prob + 2.0 ** -81).all(), (np.abs(got[1] / prob - 1).max(), rel)
    assert abs(got[2] - loss) <= (rel + 4 * 2.0 ** -24) * loss
