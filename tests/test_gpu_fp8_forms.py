"""Every form of the 8-bit product with every output type, bias and
accumulation, at sizes whose rows leave by TMA and at odd ones; grouped
products of many experts; the column quantiser past its first turn."""
import numpy as np
import pytest

import fp8_util as f8
from fp8_util import BF16, F16, F32
from test_fp8_forms import SIZES
from test_gpu_fp8 import activations, check, matmul, quant

pytestmark = pytest.mark.gpu


def operands(rng, w_block, M, N, K):
    """Codes and scales of a and w, their values, and the bias."""
    a, asc = f8.quant_rows(activations(rng, M, K))
    w = (rng.standard_normal((N, K)) / np.sqrt(K)).astype(np.float32)
    if w_block == 1:
        wc, ws = f8.quant_rows(w)
        wv = f8.rows_value(wc, ws)
    else:
        wc, ws = f8.quant_weight(w[None])
        wv = f8.weight_value(wc[0], ws[0])
    return a, asc, wc, ws, f8.rows_value(a, asc), wv, (rng.standard_normal(N) * 0.1).astype(np.float16)


@pytest.mark.parametrize("which", [0, 1], ids=["whole", "odd"])
@pytest.mark.parametrize("key", SIZES, ids=str)
def test_every_form(cuda_lib, key, which):
    M, N, K = SIZES[key][which]
    assert cuda_lib.ts_cuda_selftest_matmul_fp8_form(M, N, K, key[0], 0, 1, 0) == key[1]
    rng = np.random.default_rng(M + N + K)
    a, asc, w, ws, av, wv, bias = operands(rng, key[0], M, N, K)
    y, b = av @ wv.T, bias.astype(np.float64)
    held = rng.standard_normal((M, N)).astype(np.float32)
    for out in (F16, BF16, F32):
        check(matmul(cuda_lib, a, asc, w, ws, M, N, K, out, w_block=key[0]), av, wv, y, out)
        check(matmul(cuda_lib, a, asc, w, ws, M, N, K, out, w_block=key[0], bias=bias), av, wv, y + b, out, np.abs(b))
    check(matmul(cuda_lib, a, asc, w, ws, M, N, K, F32, w_block=key[0], acc=held), av, wv, y + held, F32, np.abs(held))
    check(matmul(cuda_lib, a, asc, w, ws, M, N, K, F32, w_block=key[0], bias=bias, acc=held), av, wv, y + b + held, F32,
          np.abs(b) + np.abs(held))


@pytest.mark.parametrize("E,most,N,K,out", [(200, 60, 130, 257, F32), (200, 900, 264, 128, F16), (1024, 3, 24, 48, BF16),
                                            (1024, 40, 64, 128, F32), (77, 4, 128, 4096, F16)])
def test_many_experts(cuda_lib, E, most, N, K, out):
    """The prefix over segments past one warp's first pass, empty experts among them."""
    rng = np.random.default_rng(E + N)
    sizes = rng.integers(0, most + 1, E) * (rng.random(E) < 0.8)
    seg = np.concatenate([[0], np.cumsum(sizes)])
    M = int(seg[-1])
    a, asc = f8.quant_rows(activations(rng, M, K))
    w, ws = f8.quant_weight((rng.standard_normal((E, N, K)) / np.sqrt(K)).astype(np.float32))
    bias = (rng.standard_normal((E, N)) * 0.1).astype(np.float16)
    o = matmul(cuda_lib, a, asc, w, ws, M, N, K, out, bias=bias, seg=seg, E=E)
    av = f8.rows_value(a, asc)
    got = o.float().cpu().numpy().astype(np.float64)
    assert np.isfinite(got).all()
    for e in range(E):
        r = slice(seg[e], seg[e + 1])
        if not sizes[e]:
            continue
        wv, b = f8.weight_value(w[e], ws[e]), bias[e].astype(np.float64)
        y = av[r] @ wv.T + b
        assert (np.abs(got[r] - y) <= f8.product_bound(av[r], wv, y, out, np.abs(b))).all(), e


@pytest.mark.parametrize("code", [F16, BF16, F32])
@pytest.mark.parametrize("rows,cols,ldx", [(9000, 1300, None), (9000, 1300, 1303), (16391, 1280, None)])
def test_quantise_columns_over_several_turns(cuda_lib, code, rows, cols, ldx):
    """More tiles than blocks that fit the GPU: each block takes several, the next on its way while one is quantised."""
    rng = np.random.default_rng(rows + cols)
    _, _, codes, scales, xv = quant(cuda_lib, activations(rng, rows, cols), code, True, ldx)
    ec, es = f8.quant_rows(xv.T)
    assert np.array_equal(scales, es)
    assert np.array_equal(codes, ec)
