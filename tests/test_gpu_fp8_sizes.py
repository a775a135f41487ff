"""The 8-bit operators at the ends of their sizes, where 32-bit index
arithmetic would wrap: nothing is read or written past a row's end."""
import numpy as np
import pytest

import fp8_util as f8
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


@pytest.mark.parametrize("transpose", [False, True])
def test_quantise_longest_row(cuda_lib, transpose):
    """A row (or column) of 2^32 - 1 values: the last piece of 16 holds 15 of them, and what lies behind the row (a value
    that would raise the last block's scale) is no part of it."""
    import torch
    C = (1 << 32) - 1
    x = torch.full((C + 1,), 1.0, dtype=torch.float16, device="cuda")
    tail = np.random.default_rng(1).standard_normal(1000).astype(np.float16)
    x[C - 1000:C] = torch.from_numpy(tail).cuda()
    x[C] = 60000.0
    rows, cols, ldx = (C, 1, 1) if transpose else (1, C, C + 1)
    codes = torch.full((C + 1,), 0xAB, dtype=torch.uint8, device="cuda")
    scales = torch.full((f8.up(C, 128) // 128, 1), -1.0, device="cuda")
    assert cuda_lib.ts_cuda_op_quant_fp8(ptr(x), F16, ldx, rows, cols, int(transpose), ptr(codes), C + 1, ptr(scales), 1,
                                         stream()) == 0, cuda_lib.ts_cuda_last_error()
    torch.cuda.synchronize()
    first = C // 128 * 128 - 6 * 128  # the tail's blocks but the one that its start shares with the ones
    ec, es = f8.quant_rows(tail[first - (C - 1000):].astype(np.float32)[None])
    assert np.array_equal(codes[first:C].cpu().numpy(), ec[0])
    assert np.array_equal(scales[first // 128:].cpu().numpy(), es)
    oc, os_ = f8.quant_rows(np.ones((1, 128), np.float32))
    ones = (C - 1000) // 128 * 128
    assert bool((codes[:ones] == int(oc[0, 0])).all()) and bool((scales[:ones // 128] == float(os_[0, 0])).all())
