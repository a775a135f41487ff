"""The router balance as large calls run it, against the formulas: runs of
several tokens a lane group with documents that end inside them, padding in
between, more documents than fit shared memory, and many documents in the
one-block form."""
import numpy as np
import pytest

from fp8_util import BF16, F16, F32
from test_gpu_balance import balance, compare, term_sizes

pytestmark = pytest.mark.gpu


def documents(rng, T, longest):
    """Offsets of documents of 1 to `longest` tokens, every tenth of them empty."""
    lengths = []
    while sum(lengths) < T:
        lengths.append(0 if rng.random() < 0.1 else int(rng.integers(1, longest + 1)))
    seq = np.minimum(np.concatenate([[0], np.cumsum(lengths)]), T)
    return seq.astype(np.int64)


# a lane group's tokens in a row on 148 SMs: 3, 3, 3, 5, 5, 16
@pytest.mark.parametrize("T,E,k,longest,code", [(20000, 128, 4, 40, F32), (20000, 128, 4, 40, BF16), (40000, 60, 2, 90, F16),
                                                (20001, 256, 8, 300, F32), (5003, 300, 4, 7, F32), (150000, 128, 4, 5000, F32)])
def test_runs_of_tokens(cuda_lib, T, E, k, longest, code):
    rng = np.random.default_rng(T + E)
    z = (rng.standard_normal((T, E)) * 1.5 + rng.standard_normal(E) * 0.7).astype(np.float32)
    idx = np.argsort(-z, 1, kind="stable")[:, :k].astype(np.int32)
    mask = (rng.random(T) < 0.9).astype(np.uint8)
    seq = documents(rng, T, longest)
    scale = 2.0 ** 20 if code == F16 else 1.0
    got, zv = balance(cuda_lib, z, code, idx, mask, seq, scale=scale)
    compare(got, term_sizes(zv, idx, mask, seq, 0.01, scale), code, E, T)


@pytest.mark.parametrize("T,E,S", [(9000, 64, 1500), (20000, 130, 3001), (900, 2, 1200), (1000, 1, 4000)])
def test_many_documents(cuda_lib, T, E, S):
    rng = np.random.default_rng(S)
    z = (rng.standard_normal((T, E)) * 1.5).astype(np.float32)
    idx = np.argsort(-z, 1, kind="stable")[:, :1].astype(np.int32)
    mask = (rng.random(T) < 0.9).astype(np.uint8)
    seq = np.concatenate([[0], np.sort(rng.integers(0, T + 1, S - 1)), [T]])
    got, zv = balance(cuda_lib, z, F32, idx, mask, seq)
    compare(got, term_sizes(zv, idx, mask, seq, 0.01, 1.0), F32, E, T)
