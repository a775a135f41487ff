"""Which form of the 8-bit product a call's sizes choose, on the CPU: the
sizes that the GPU tests use for each form have to reach it on 148 SMs."""
import pytest

SMS = 148  # of a B200
EMPTY, MATVEC, PAIRS, WIDE, NARROW, SPLIT2, SPLIT4, SPLIT8 = range(8)

# (w_block, form): sizes (M, N, K) whose output rows can leave by TMA, then sizes that fit no tile
SIZES = {
    (128, PAIRS): [(4000, 640, 129), (3001, 1003, 130)],
    (128, WIDE): [(1000, 1280, 129), (1501, 1001, 131)],
    (128, NARROW): [(300, 640, 384), (41, 1001, 301)],
    (128, SPLIT2): [(520, 1000, 4096), (519, 1003, 4001)],
    (128, SPLIT4): [(520, 640, 2048), (301, 1001, 2050)],
    (128, SPLIT8): [(40, 1000, 2048), (41, 257, 2047)],
    (1, PAIRS): [(2000, 1280, 129), (1501, 2047, 130)],
    (1, WIDE): [(300, 640, 129), (41, 1001, 300)],
    (1, SPLIT2): [(520, 1000, 2048), (301, 2047, 2050)],
    (1, SPLIT4): [(520, 640, 1024), (301, 1001, 1025)],
    (1, SPLIT8): [(40, 1000, 1024), (41, 641, 1030)],
}


@pytest.mark.parametrize("key", SIZES, ids=str)
def test_sizes_reach_their_form(cuda_lib, key):
    for M, N, K in SIZES[key]:
        assert cuda_lib.ts_cuda_selftest_matmul_fp8_form(M, N, K, key[0], 0, 1, SMS) == key[1], (M, N, K)


def test_forms_by_rule(cuda_lib):
    form = cuda_lib.ts_cuda_selftest_matmul_fp8_form
    assert form(5, 64, 0, 128, 0, 1, SMS) == EMPTY
    assert form(16, 64, 128, 128, 0, 1, SMS) == MATVEC
    assert form(16, 64, 128, 128, 1, 1, SMS) != MATVEC and form(16, 64, 128, 1, 0, 1, SMS) == WIDE
    assert form(17, 64, 128, 128, 0, 1, SMS) == NARROW


@pytest.mark.parametrize("args", [(0, 1, 1, 128, 0, 1, SMS), (1, 0, 1, 128, 0, 1, SMS), (1, 1, 1, 64, 0, 1, SMS),
                                  (1, 1, 1, 128, 0, 0, SMS), (1, 1, 1, 128, 0, 1, 7)])
def test_refusals(cuda_lib, args):
    assert cuda_lib.ts_cuda_selftest_matmul_fp8_form(*args) == -1
