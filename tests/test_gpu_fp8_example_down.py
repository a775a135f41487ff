"""The 8-bit expert layer's example checks its down product and the layer's
output too, and both are as near f32 as 8-bit operands are."""
import os
import sys

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("args", [["--tokens", "500", "--experts", "16", "--hidden", "256", "--k", "2"],
                                  ["--tokens", "33", "--experts", "8", "--hidden", "128", "--documents", "1"]])
def test_down_product_and_output(cuda_lib, args):
    import torch
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    import fp8_expert_layer as ex
    out = ex.main(args)
    # the input's codes are off by at most 2^-4 of their value each (the weight's codes are exact here), and so, in the
    # mean, is what they are multiplied to; the output adds such products with weights of one sign
    for name in ("down product", "output"):
        assert 0.0 < out["errors"][name] <= 2.0 ** -4 * 1.5, (name, out["errors"])
    assert out["y"].shape[0] == int(args[1]) and bool(torch.isfinite(out["y"]).all())
