"""The 8-bit expert layer's example end to end: its errors are those of 8-bit
operands, and its segments are the balance's counts."""
import os
import sys

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("args", [["--tokens", "700", "--experts", "16", "--hidden", "256", "--k", "2"],
                                  ["--tokens", "33", "--experts", "8", "--hidden", "128", "--documents", "1"]])
def test_example(cuda_lib, args):
    import torch
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    import fp8_expert_layer as ex
    out = ex.main(args)
    # a code is off by at most 2^-4 of its value, by 2^-4 / sqrt(3) or so in the mean; the forward is two such operands
    # (the weight's codes are exact here) through the gate, the weight gradient a product of two
    for name, v in out["errors"].items():
        assert v <= 2.0 ** -4 * (2 if name == "weight gradient" else 1) * 1.5, (name, v)
    counts = out["counts"].sum(0)
    assert torch.equal(out["seg"][1:], counts.cumsum(0).int())
    assert out["seg"][-1] == out["order"].numel()
