"""The 8-bit expert layer's example makes weights in the format that the
operators document: the largest magnitude times f32(1/448), codes of the
values times the scale's f32 reciprocal."""
import os
import sys

import numpy as np
import pytest

import fp8_util as f8
from conftest import ROOT

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("E,N,K", [(1, 16, 16), (3, 130, 257), (4, 640, 512)])
def test_weights_are_in_the_format(cuda_lib, E, N, K):
    import torch
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    import fp8_expert_layer as ex
    w = np.random.default_rng(N).standard_normal((E, N, K)).astype(np.float32) / np.float32(np.sqrt(K))
    got = ex.Weight(torch.from_numpy(w).cuda())
    torch.cuda.synchronize()
    codes, scales = f8.quant_weight(w)
    assert np.array_equal(got.scales.cpu().numpy(), scales)
    assert np.array_equal(got.codes[:, :, :K].cpu().numpy(), codes)
    assert np.array_equal(got.codes_t[:, :, :N].cpu().numpy(), codes.transpose(0, 2, 1))
