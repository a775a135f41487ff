"""The 8-bit operators at the ends of their sizes, where 32-bit index
arithmetic would wrap: nothing is read or written past a row's end."""
import pytest

from fp8_util import F16
from gpu_util import ptr, stream

pytestmark = pytest.mark.gpu

MOST = 0x7fffff00  # the largest M, N or K that the products take


def test_empty_sum_of_most_rows(cuda_lib):
    """K = 0 on the largest number of rows: a step past the last row must not come round to negative rows, which lie
    before the output (guarded here on both sides)."""
    import torch
    guard = 1 << 16
    room = torch.full((guard + MOST + guard,), 5.0, dtype=torch.float16, device="cuda")
    bias = torch.tensor([0.25], dtype=torch.float16, device="cuda")
    assert cuda_lib.ts_cuda_op_matmul_fp8(None, 0, None, MOST, None, 0, None, 0, 128, ptr(bias), None, 1,
                                          ptr(room) + 2 * guard, F16, 1, 0, MOST, 1, 0, stream()) == 0, \
        cuda_lib.ts_cuda_last_error()
    torch.cuda.synchronize()
    assert bool((room[guard:guard + MOST] == 0.25).all())
    assert bool((room[:guard] == 5.0).all()) and bool((room[guard + MOST:] == 5.0).all())
