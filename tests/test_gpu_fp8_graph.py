"""The 8-bit operators and the router balance inside a CUDA graph: they
allocate nothing and do not synchronize, so a captured chain of them replays
on new inputs with the results of separate calls."""
import numpy as np
import pytest

import fp8_util as f8
from fp8_util import F16, F32
from gpu_util import ptr, stream

pytestmark = pytest.mark.gpu


def test_chain_in_a_graph(cuda_lib):
    import torch
    L = cuda_lib
    M, N, K, E, k = 300, 640, 512, 640, 4
    rng = np.random.default_rng(0)
    w, ws = f8.quant_weight(rng.standard_normal((1, N, K)).astype(np.float32) / np.sqrt(K))
    dw, dws = torch.from_numpy(f8.pitched(w)).cuda(), torch.from_numpy(ws).cuda()
    x = torch.randn(M, K, device="cuda").half()
    codes, scales = torch.empty(M, K, dtype=torch.uint8, device="cuda"), torch.empty(K // 128, M, device="cuda")
    y = torch.empty(M, N, device="cuda")
    idx = torch.from_numpy(rng.integers(0, E, (M, k)).astype(np.int32)).cuda()
    counts, prob = torch.empty(1, E, dtype=torch.int32, device="cuda"), torch.empty(1, E, device="cuda")
    loss, grad = torch.empty(1, device="cuda"), torch.empty(M, E, device="cuda")
    work = torch.empty(L.ts_cuda_router_balance_work(1, E), dtype=torch.uint8, device="cuda")

    def chain():
        """Quantise x, multiply, and take the products as router logits."""
        assert L.ts_cuda_op_quant_fp8(ptr(x), F16, K, M, K, 0, ptr(codes), K, ptr(scales), M, stream()) == 0
        assert L.ts_cuda_op_matmul_fp8(ptr(codes), K, ptr(scales), M, ptr(dw), dw.stride(1), ptr(dws), 0, 128, None, None, 1,
                                       ptr(y), F32, N, 0, M, N, K, stream()) == 0
        assert L.ts_cuda_op_router_balance(ptr(y), F32, N, ptr(idx), None, None, 1, M, E, k, 0.01, 1.0, ptr(counts), ptr(prob),
                                           ptr(loss), ptr(grad), E, ptr(work), work.numel(), stream()) == 0

    chain()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        chain()
    for seed in range(3):
        x.copy_(torch.from_numpy(np.random.default_rng(seed).standard_normal((M, K)).astype(np.float16)))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (codes, scales, y, counts, prob, loss, grad)]
        chain()
        torch.cuda.synchronize()
        for a, b in zip(got, (codes, scales, y, counts, prob, loss, grad)):
            assert torch.equal(a, b)
        ec, es = f8.quant_rows(x.float().cpu().numpy())
        assert np.array_equal(codes.cpu().numpy(), ec) and np.array_equal(scales.cpu().numpy(), es)
        ref = f8.rows_value(ec, es) @ f8.weight_value(w[0], ws[0]).T
        bound = f8.product_bound(f8.rows_value(ec, es), f8.weight_value(w[0], ws[0]), ref, F32)
        assert (np.abs(y.cpu().numpy() - ref) <= bound).all()
    del graph
