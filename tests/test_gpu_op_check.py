"""The error flag of the operators that take no handle: a wait that runs out
on one stream reaches that stream's check, whichever stream checks first.

The wait is the self-test's: one CTA on a barrier that nothing arrives at,
with a limit of 2 ms, after which it gives up and frees what it holds.
"""
import numpy as np
import pytest

import fp8_util as f8
from fp8_util import F32
from gpu_util import ptr, stream

pytestmark = pytest.mark.gpu

DEVICE, ARG = -5, -1


@pytest.fixture
def told(cuda_lib):
    """Both checks before and after: the default stream has heard of every error, so other tests' checks report none."""
    cuda_lib.ts_cuda_op_check(stream())
    yield
    cuda_lib.ts_cuda_op_check(stream())
    assert cuda_lib.ts_cuda_op_check(stream()) == 0


def test_an_error_reaches_every_streams_check(cuda_lib, told):
    import torch
    L = cuda_lib
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for s in (a, b):
        L.ts_cuda_op_check(s.cuda_stream)
        assert L.ts_cuda_op_check(s.cuda_stream) == 0
    res = torch.full((2,), 7, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    assert L.ts_cuda_selftest_op_wait_timeout(2000, ptr(res), a.cuda_stream) == 0, L.ts_cuda_last_error()
    a.synchronize()
    assert res.tolist() == [0, 0]  # both waits gave up
    assert L.ts_cuda_op_check(b.cuda_stream) == DEVICE  # found by another stream's check ...
    assert L.ts_cuda_op_check(a.cuda_stream) == DEVICE  # ... and still there for its own
    assert b"bounded wait timed out" in L.ts_cuda_last_error()
    for s in (a, b):
        assert L.ts_cuda_op_check(s.cuda_stream) == 0
    # a second error is a new one for both
    assert L.ts_cuda_selftest_op_wait_timeout(2000, None, b.cuda_stream) == 0
    assert L.ts_cuda_op_check(b.cuda_stream) == DEVICE
    assert L.ts_cuda_op_check(a.cuda_stream) == DEVICE
    assert L.ts_cuda_op_check(a.cuda_stream) == 0 and L.ts_cuda_op_check(b.cuda_stream) == 0


def test_operators_work_after_an_error(cuda_lib, told):
    import torch
    L = cuda_lib
    x = torch.ones(4, 128, device="cuda")
    codes, scales = torch.zeros(4, 128, dtype=torch.uint8, device="cuda"), torch.zeros(1, 4, device="cuda")
    assert L.ts_cuda_selftest_op_wait_timeout(2000, None, stream()) == 0
    assert L.ts_cuda_op_check(stream()) == DEVICE
    assert L.ts_cuda_op_quant_fp8(ptr(x), F32, 128, 4, 128, 0, ptr(codes), 128, ptr(scales), 4, stream()) == 0
    assert L.ts_cuda_op_check(stream()) == 0
    ec, es = f8.quant_rows(np.ones((4, 128), np.float32))
    assert np.array_equal(codes.cpu().numpy(), ec) and np.array_equal(scales.cpu().numpy(), es)


def test_bad_limits(cuda_lib):
    assert cuda_lib.ts_cuda_selftest_op_wait_timeout(0, None, None) == ARG
    assert cuda_lib.ts_cuda_selftest_op_wait_timeout(1000001, None, None) == ARG
    assert cuda_lib.ts_cuda_selftest_op_wait_timeout(10, 2, None) == ARG
