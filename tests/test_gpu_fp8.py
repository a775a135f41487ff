"""The 8-bit floating point operators against their definition in numpy
(tests/fp8_util.py): codes and scales bit for bit, products within the bound
that f32 sums of any order keep."""
import numpy as np
import pytest

import fp8_util as f8
from fp8_util import BF16, F16, F32
from gpu_util import ptr, stream

pytestmark = pytest.mark.gpu

TORCH = {F16: "float16", BF16: "bfloat16", F32: "float32"}


def tdt(code):
    import torch
    return getattr(torch, TORCH[code])


def cuda(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def activations(rng, rows, cols):
    x = rng.standard_normal((rows, cols)) * np.exp(0.5 * rng.standard_normal((rows, 1)))
    return (x * np.where(rng.random((1, cols)) < 0.02, 12.0, 1.0)).astype(np.float32)


def device_x(x, code, ld=None):
    """x as a device tensor of the given type in rows of ld elements, and the f32 values it holds."""
    import torch
    rows, cols = x.shape
    full = torch.full((rows, ld or cols), float("nan"), dtype=tdt(code), device="cuda")
    full[:, :cols] = cuda(x).to(tdt(code))
    return full, full[:, :cols].float().cpu().numpy()


def quant(L, x, code, transpose=False, ldx=None, pad=0):
    """Runs the operator; returns (device codes, device scales, host codes, host scales, f32 input)."""
    import torch
    rows, cols = x.shape
    dx, xv = device_x(x, code, ldx)
    R, C = (cols, rows) if transpose else (rows, cols)
    codes = torch.full((R, f8.up(C, 16) + 16 * pad), 0xAB, dtype=torch.uint8, device="cuda")
    scales = torch.full((f8.up(C, 128) // 128, f8.up(R, 4) + pad), -1.0, device="cuda")
    assert L.ts_cuda_op_quant_fp8(ptr(dx), code, dx.stride(0), rows, cols, int(transpose), ptr(codes), codes.stride(0),
                                  ptr(scales), scales.stride(0), stream()) == 0, L.ts_cuda_last_error()
    torch.cuda.synchronize()
    return codes, scales, codes[:, :C].cpu().numpy(), scales[:, :R].cpu().numpy(), xv


@pytest.mark.parametrize("code", [F16, BF16, F32])
@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("rows,cols,ldx", [(1, 1, None), (1, 640, None), (3, 127, None), (5, 128, 131), (129, 129, None),
                                           (128, 256, None), (257, 1000, 1003), (131, 2050, 2056), (1025, 72, 80),
                                           (70, 16400, None), (4099, 32, None)])
def test_quant_bit_exact(cuda_lib, code, transpose, rows, cols, ldx):
    rng = np.random.default_rng(rows * 31 + cols)
    _, _, codes, scales, xv = quant(cuda_lib, activations(rng, rows, cols), code, transpose, ldx, pad=rows % 3)
    ec, es = f8.quant_rows(xv.T if transpose else xv)
    assert np.array_equal(scales, es)
    assert np.array_equal(codes, ec)


@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("code", [F16, BF16, F32])
def test_quant_awkward_values(cuda_lib, code, transpose):
    """Zeros of both signs, infinities, NaN, a block of zeros, subnormals, the largest finite value."""
    rng = np.random.default_rng(7)
    x = activations(rng, 256, 384)
    x[0] = 0.0
    x[1, ::2] = -0.0
    x[2, 5], x[2, 6], x[2, 200] = np.inf, -np.inf, np.nan
    x[3] = np.inf
    x[4] = np.nan
    x[5] = 2.0 ** -24 * rng.integers(0, 3, 384)
    x[6, 0] = {F16: 65504.0, BF16: 3.3895e38, F32: 3.4028235e38}[code]
    x[7] = 1e-37 * rng.standard_normal(384)
    x[8] *= 1e-30 if code != F16 else 1e-3
    x[128:, 3] = 0.0
    _, _, codes, scales, xv = quant(cuda_lib, x, code, transpose)
    ec, es = f8.quant_rows(xv.T if transpose else xv)
    assert np.array_equal(scales, es)
    assert np.array_equal(codes, ec)


def test_quant_leaves_the_rest_alone(cuda_lib):
    """Nothing past the codes' rows and blocks of scales is written, but for the padding of a row to 16 bytes."""
    import torch
    rng = np.random.default_rng(3)
    for transpose in (0, 1):
        x, _ = device_x(activations(rng, 37, 70), F16)
        R, C = (70, 37) if transpose else (37, 70)
        codes = torch.full((R + 2, 160), 0xAB, dtype=torch.uint8, device="cuda")
        scales = torch.full((2, 75), -1.0, device="cuda")
        assert cuda_lib.ts_cuda_op_quant_fp8(ptr(x), F16, 70, 37, 70, transpose, ptr(codes), 160, ptr(scales), 75,
                                             stream()) == 0
        torch.cuda.synchronize()
        assert (codes[R:] == 0xAB).all() and (codes[:, f8.up(C, 16):] == 0xAB).all()
        assert (scales[:, R:] == -1.0).all() and (scales[1:] == -1.0).all()


@pytest.mark.parametrize("E,N,K", [(1, 16, 16), (3, 130, 257), (2, 64, 128), (1, 1000, 640), (5, 127, 1)])
def test_transpose_exact(cuda_lib, E, N, K):
    import torch
    rng = np.random.default_rng(N)
    codes, scales = rng.integers(0, 256, (E, N, K), np.uint8), rng.random((E, f8.up(N, 128) // 128, f8.up(K, 128) // 128),
                                                                        np.float32)
    dc, ds = cuda(f8.pitched(codes)), cuda(scales)
    t = torch.zeros(E, K, f8.up(N, 16), dtype=torch.uint8, device="cuda")
    ts = torch.zeros(E, scales.shape[2], scales.shape[1], device="cuda")
    assert cuda_lib.ts_cuda_op_transpose_fp8(ptr(dc), dc.stride(1), ptr(ds), E, N, K, ptr(t), t.stride(1), ptr(ts),
                                             stream()) == 0, cuda_lib.ts_cuda_last_error()
    torch.cuda.synchronize()
    assert np.array_equal(t[:, :, :N].cpu().numpy(), codes.transpose(0, 2, 1))
    assert np.array_equal(ts.cpu().numpy(), scales.transpose(0, 2, 1))


def matmul(L, a, asc, w, ws, M, N, K, out, w_block=128, bias=None, seg=None, E=1, acc=None, ldo=None, st=None):
    """a, w: host codes; asc, ws: host scales.  Returns the device result [M, ldo]."""
    import torch
    da, dw = cuda(f8.pitched(a, f8.up(K, 16) + 32)), cuda(f8.pitched(w))
    das = torch.full((asc.shape[0], M + 3), float("nan"), device="cuda")
    das[:, :M] = cuda(asc)
    dws = cuda(ws)
    db = None if bias is None else cuda(bias.view(np.int16))
    dseg = None if seg is None else cuda(np.asarray(seg, np.int32))
    if acc is not None:
        o = cuda(acc)
    else:
        o = torch.full((M, ldo or N), -7.0, dtype=tdt(out), device="cuda")
    torch.cuda.synchronize()
    rc = L.ts_cuda_op_matmul_fp8(ptr(da), da.stride(0), ptr(das), das.stride(0), ptr(dw), dw.stride(-2), ptr(dws),
                                 dws.stride(0) if w_block == 1 else 0, w_block, None if db is None else ptr(db),
                                 None if dseg is None else ptr(dseg), E, ptr(o), out, o.stride(0), int(acc is not None),
                                 M, N, K, stream() if st is None else st)
    assert rc == 0, L.ts_cuda_last_error()
    torch.cuda.synchronize()
    assert L.ts_cuda_op_check(stream()) == 0, L.ts_cuda_last_error()
    return o


def check(o, a, w, y, out, extra=0.0):
    got = o.float().cpu().numpy().astype(np.float64)
    bound = f8.product_bound(a, w, y, out, extra)
    off = np.abs(got - y)
    assert np.isfinite(got).all()
    assert (off <= bound).all(), (np.unravel_index((off - bound).argmax(), off.shape), (off - bound).max())


SHAPES = [(1, 1, 1), (1, 16, 128), (2, 17, 130), (16, 640, 640), (17, 33, 129), (33, 128, 384), (64, 200, 2048),
          (127, 256, 640), (128, 129, 128), (129, 640, 256), (257, 1152, 640), (300, 77, 1000), (517, 1001, 1500),
          (1000, 513, 100), (2050, 384, 512)]


@pytest.mark.parametrize("out", [F16, BF16, F32])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_matmul(cuda_lib, M, N, K, out):
    rng = np.random.default_rng(M * 7 + N * 3 + K)
    a, asc = f8.quant_rows(activations(rng, M, K))
    w, ws = f8.quant_weight(rng.standard_normal((1, N, K)).astype(np.float32) / np.sqrt(K))
    bias = (rng.standard_normal(N) * 0.1).astype(np.float16) if (M + N) % 2 else None
    av, wv = f8.rows_value(a, asc), f8.weight_value(w[0], ws[0])
    y = av @ wv.T + (0 if bias is None else bias.astype(np.float64))
    o = matmul(cuda_lib, a, asc, w, ws, M, N, K, out, bias=bias, ldo=N + (M % 5))
    check(o[:, :N], av, wv, y, out, 0 if bias is None else np.abs(bias.astype(np.float64)))
    assert (o[:, N:].float() == -7.0).all()  # what lies between the rows stays


# sizes that reach the CTA pairs (many tiles, their edges odd) and the clusters that split k (few tiles, k long)
@pytest.mark.parametrize("M,N,K,out", [(9001, 2310, 385, F16), (9001, 2311, 385, BF16), (20000, 1152, 640, F16),
                                       (6000, 3080, 129, F32), (100, 520, 4100, F16), (33, 64, 8192, F32),
                                       (130, 127, 6001, BF16), (257, 1000, 2048, F32)])
def test_matmul_large_and_long(cuda_lib, M, N, K, out):
    rng = np.random.default_rng(M + N + K)
    a, asc = f8.quant_rows(activations(rng, M, K))
    w, ws = f8.quant_weight(rng.standard_normal((1, N, K)).astype(np.float32) / np.sqrt(K))
    bias = (rng.standard_normal(N) * 0.1).astype(np.float16)
    av, wv = f8.rows_value(a, asc), f8.weight_value(w[0], ws[0])
    y = av @ wv.T + bias.astype(np.float64)
    check(matmul(cuda_lib, a, asc, w, ws, M, N, K, out, bias=bias), av, wv, y, out, np.abs(bias.astype(np.float64)))


@pytest.mark.parametrize("sizes,N,K", [([3000, 0, 5001, 17, 4100, 9000], 1032, 260), ([5, 0, 40, 1], 130, 4100),
                                       ([0, 0, 0], 64, 4096)])
def test_matmul_experts_large_and_long(cuda_lib, sizes, N, K):
    E, M = len(sizes), max(1, sum(sizes))
    rng = np.random.default_rng(M)
    seg = np.concatenate([[0], np.cumsum(sizes)])
    a, asc = f8.quant_rows(activations(rng, M, K))
    w, ws = f8.quant_weight(rng.standard_normal((E, N, K)).astype(np.float32) / np.sqrt(K))
    o = matmul(cuda_lib, a, asc, w, ws, M, N, K, F16, seg=seg, E=E)
    av = f8.rows_value(a, asc)
    for e in range(E):
        r = slice(seg[e], seg[e + 1])
        if sizes[e]:
            wv = f8.weight_value(w[e], ws[e])
            check(o[r], av[r], wv, av[r] @ wv.T, F16)
    assert (o[seg[-1]:].float() == -7.0).all()


@pytest.mark.parametrize("M,N,K", [(256, 256, 256), (1025, 1280, 640), (40, 640, 384), (8192, 2304, 256), (64, 128, 4096)])
def test_matmul_exact_integers(cuda_lib, M, N, K):
    """Small whole numbers and power-of-two scales leave nothing to round: every tile and block has to be exact."""
    rng = np.random.default_rng(K)
    a = f8.e4m3(rng.integers(-8, 9, (M, K)))
    w = f8.e4m3(rng.integers(-8, 9, (1, N, K)))
    asc = np.exp2(rng.integers(-2, 3, (f8.up(K, 128) // 128, M))).astype(np.float32)
    ws = np.exp2(rng.integers(-2, 3, (1, f8.up(N, 128) // 128, f8.up(K, 128) // 128))).astype(np.float32)
    o = matmul(cuda_lib, a, asc, w, ws, M, N, K, F32)
    y = f8.rows_value(a, asc) @ f8.weight_value(w[0], ws[0]).T
    assert np.array_equal(o.cpu().numpy().astype(np.float64), y)


@pytest.mark.parametrize("sizes", [[0, 5, 0, 130, 1, 64], [300], [0, 0, 0, 7], [128, 128, 129, 127], [1] * 40,
                                   [16, 0, 517, 3, 256, 0, 0, 1]])
@pytest.mark.parametrize("N,K,out", [(1280, 640, F16), (130, 257, F32), (64, 128, BF16)])
def test_matmul_experts(cuda_lib, sizes, N, K, out):
    E, M = len(sizes), sum(sizes)
    rng = np.random.default_rng(E * 100 + N)
    seg = np.concatenate([[0], np.cumsum(sizes)])
    a, asc = f8.quant_rows(activations(rng, M, K))
    w, ws = f8.quant_weight(rng.standard_normal((E, N, K)).astype(np.float32) / np.sqrt(K))
    bias = (rng.standard_normal((E, N)) * 0.1).astype(np.float16)
    o = matmul(cuda_lib, a, asc, w, ws, M, N, K, out, bias=bias, seg=seg, E=E)
    av = f8.rows_value(a, asc)
    for e in range(E):
        r = slice(seg[e], seg[e + 1])
        if sizes[e]:
            wv = f8.weight_value(w[e], ws[e])
            check(o[r], av[r], wv, av[r] @ wv.T + bias[e].astype(np.float64), out, np.abs(bias[e].astype(np.float64)))


def test_matmul_rows_outside_segments_stay(cuda_lib):
    """Rows that no segment covers are not written, and bounds past M are clamped."""
    rng = np.random.default_rng(1)
    M, N, K = 200, 96, 256
    a, asc = f8.quant_rows(activations(rng, M, K))
    w, ws = f8.quant_weight(rng.standard_normal((3, N, K)).astype(np.float32))
    o = matmul(cuda_lib, a, asc, w, ws, M, N, K, F32, seg=[10, 40, 40, 1000], E=3).cpu().numpy()
    assert (o[:10] == -7.0).all() and (o[10:] != -7.0).all()
    av = f8.rows_value(a, asc)
    for e, r in ((0, slice(10, 40)), (2, slice(40, 200))):
        wv = f8.weight_value(w[e], ws[e])
        assert (np.abs(o[r] - av[r] @ wv.T) <= f8.product_bound(av[r], wv, o[r], F32)).all()
    o = matmul(cuda_lib, a, asc, w, ws, M, N, K, F32, seg=[-5, -1, 0, 0], E=3).cpu().numpy()
    assert (o == -7.0).all()


@pytest.mark.parametrize("T,N,K", [(1, 16, 16), (100, 130, 70), (129, 256, 128), (1000, 640, 1280), (4097, 64, 200),
                                   (260, 3001, 2050), (2050, 640, 1281)])
def test_weight_gradient(cuda_lib, T, N, K):
    """dW = dY^T X from operands quantised along the tokens, written and accumulated."""
    rng = np.random.default_rng(T)
    dy, x = activations(rng, T, N), activations(rng, T, K)
    _, _, cy, sy, dyv = quant(cuda_lib, dy, BF16, transpose=True)
    _, _, cx, sx, xv = quant(cuda_lib, x, F16, transpose=True)
    av, wv = f8.rows_value(cy, sy), f8.rows_value(cx, sx)
    y = av @ wv.T
    o = matmul(cuda_lib, cy, sy, cx, sx, N, K, T, F32, w_block=1)
    check(o, av, wv, y, F32)
    held = rng.standard_normal((N, K)).astype(np.float32)
    o = matmul(cuda_lib, cy, sy, cx, sx, N, K, T, F32, w_block=1, acc=held)
    check(o, av, wv, y + held, F32, np.abs(held))
    # and the gradient of the unquantised product, to the format's own precision: a code is off by at most 2^-4 of its
    # value, or half the smallest step, 2^-10, times its scale
    dyt, xt = np.abs(dyv.T.astype(np.float64)), np.abs(xv.T.astype(np.float64))
    spread = [2.0 ** -4 * v + 2.0 ** -10 * np.repeat(s.T.astype(np.float64), 128, 1)[:, :T] for v, s in ((dyt, sy), (xt, sx))]
    far = (dyt + spread[0]) @ (xt + spread[1]).T - dyt @ xt.T
    assert (np.abs(y - dyv.T.astype(np.float64) @ xv) <= 1.0001 * far).all()


@pytest.mark.parametrize("M,N,K", [(5, 130, 300), (16, 64, 128), (300, 257, 384), (300, 256, 129), (40, 64, 8192),
                                   (9000, 2304, 130)])
def test_accumulate(cuda_lib, M, N, K):
    """Added to what the output holds, in every form of the product."""
    rng = np.random.default_rng(M + K)
    a, asc = f8.quant_rows(activations(rng, M, K))
    w, ws = f8.quant_weight(rng.standard_normal((1, N, K)).astype(np.float32) / np.sqrt(K))
    held = rng.standard_normal((M, N)).astype(np.float32)
    av, wv = f8.rows_value(a, asc), f8.weight_value(w[0], ws[0])
    check(matmul(cuda_lib, a, asc, w, ws, M, N, K, F32, acc=held), av, wv, av @ wv.T + held, F32, np.abs(held))


@pytest.mark.parametrize("M,N,K", [(1, 64, 128), (50, 300, 260), (300, 640, 1280)])
def test_input_gradient(cuda_lib, M, N, K):
    """dX = dY W through the weight laid out by columns, against differences of the forward product: the product is
    linear, so f(x + h) - f(x) along a direction of the input equals the gradient's product with it."""
    import torch
    rng = np.random.default_rng(N)
    w, ws = f8.quant_weight(rng.standard_normal((1, N, K)).astype(np.float32) / np.sqrt(K))
    dw, dws = cuda(f8.pitched(w)), cuda(ws)
    wt = torch.full((1, K, f8.up(N, 16)), 0xFF, dtype=torch.uint8, device="cuda")
    wts = torch.zeros(1, ws.shape[2], ws.shape[1], device="cuda")
    assert cuda_lib.ts_cuda_op_transpose_fp8(ptr(dw), dw.stride(1), ptr(dws), 1, N, K, ptr(wt), wt.stride(1), ptr(wts),
                                             stream()) == 0
    dy = activations(rng, M, N)
    _, _, cy, sy, _ = quant(cuda_lib, dy, F16)
    torch.cuda.synchronize()
    o = matmul(cuda_lib, cy, sy, wt[:, :, :N].cpu().numpy(), wts.cpu().numpy(), M, K, N, F32)
    dyv, wv = f8.rows_value(cy, sy), f8.weight_value(w[0], ws[0])
    check(o, dyv, wv.T, dyv @ wv, F32)
    # differences: the forward at x and at x + h d, both quantised exactly (whole numbers, one scale)
    x = rng.integers(-4, 5, (M, K)).astype(np.float64)
    d = rng.integers(-2, 3, (M, K)).astype(np.float64)
    one = np.ones((f8.up(K, 128) // 128, M), np.float32)
    fwd = [matmul(cuda_lib, f8.e4m3(v), one, w, ws, M, N, K, F32).cpu().numpy().astype(np.float64) for v in (x, x + d)]
    slope = ((fwd[1] - fwd[0]) * dyv).sum()
    grad = (o.cpu().numpy().astype(np.float64) * d).sum()
    far = (f8.product_bound(x, wv, fwd[0], F32) + f8.product_bound(x + d, wv, fwd[1], F32)) * np.abs(dyv)
    far = far.sum() + (f8.product_bound(dyv, wv.T, dyv @ wv, F32) * np.abs(d)).sum()
    assert abs(slope - grad) <= far


@pytest.mark.parametrize("out", [F16, BF16, F32])
@pytest.mark.parametrize("code", [F16, BF16, F32])
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 640, 640), (1, 1000, 1500), (2, 33, 127), (3, 4096, 129), (5, 640, 2049),
                                   (8, 256, 4096), (9, 130, 384), (16, 1152, 640)])
def test_matvec(cuda_lib, M, N, K, code, out):
    import torch
    rng = np.random.default_rng(M + N + K)
    x, xv = device_x(activations(rng, M, K), code, K + 1 + M % 7)
    w, ws = f8.quant_weight(rng.standard_normal((1, N, K)).astype(np.float32) / np.sqrt(K))
    bias = (rng.standard_normal(N) * 0.1).astype(np.float16) if N % 2 == 0 else None
    dw, dws, db = cuda(f8.pitched(w)), cuda(ws), None if bias is None else cuda(bias.view(np.int16))
    o = torch.full((M, N + 3), -7.0, dtype=tdt(out), device="cuda")
    assert cuda_lib.ts_cuda_op_matvec_fp8(ptr(x), code, x.stride(0), ptr(dw), dw.stride(1), ptr(dws),
                                          None if db is None else ptr(db), ptr(o), out, N + 3, M, N, K,
                                          stream()) == 0, cuda_lib.ts_cuda_last_error()
    torch.cuda.synchronize()
    a, asc = f8.quant_rows(xv)
    av, wv = f8.rows_value(a, asc), f8.weight_value(w[0], ws[0])
    b = 0 if bias is None else bias.astype(np.float64)
    check(o[:, :N], av, wv, av @ wv.T + b, out, np.abs(b))
    assert (o[:, N:].float() == -7.0).all()


def test_empty_sums(cuda_lib):
    """K = 0: the bias or zero; accumulation keeps what is there.  M = 0 or N = 0: nothing."""
    import torch
    bias = torch.arange(8, dtype=torch.float16, device="cuda")
    o = torch.full((3, 8), 5.0, device="cuda")
    call = cuda_lib.ts_cuda_op_matmul_fp8
    assert call(None, 0, None, 3, None, 0, None, 0, 128, ptr(bias), None, 1, ptr(o), F32, 8, 1, 3, 8, 0, stream()) == 0
    torch.cuda.synchronize()
    assert (o == 5.0 + bias.float()).all()
    assert call(None, 0, None, 3, None, 0, None, 0, 128, None, None, 1, ptr(o), F32, 8, 0, 3, 8, 0, stream()) == 0
    torch.cuda.synchronize()
    assert (o == 0).all()
    assert call(None, 0, None, 0, None, 0, None, 0, 128, None, None, 1, None, F32, 8, 0, 0, 8, 16, stream()) == 0
    assert cuda_lib.ts_cuda_op_matvec_fp8(None, F16, 0, None, 0, None, ptr(bias), ptr(o), F32, 8, 3, 8, 0, stream()) == 0
    torch.cuda.synchronize()
    assert (o == bias.float()).all()


def test_nan_codes_reach_their_own_outputs_only(cuda_lib):
    rng = np.random.default_rng(5)
    M, N, K = 150, 300, 256
    a, asc = f8.quant_rows(activations(rng, M, K))
    w, ws = f8.quant_weight(rng.standard_normal((1, N, K)).astype(np.float32))
    a[3, 200], w[0, 130, 7] = 0x7F, 0xFF
    o = matmul(cuda_lib, a, asc, w, ws, M, N, K, F32).cpu().numpy()
    bad = np.isnan(o)
    assert bad[3].all() and bad[:, 130].all()
    bad[3], bad[:, 130] = False, False
    assert not bad.any()


def test_another_stream_and_repeats(cuda_lib):
    """On a stream of its own, beside other work, and bit for bit the same every time."""
    import torch
    rng = np.random.default_rng(11)
    M, N, K = 700, 640, 1280
    a, asc = f8.quant_rows(activations(rng, M, K))
    w, ws = f8.quant_weight(rng.standard_normal((1, N, K)).astype(np.float32))
    s = torch.cuda.Stream()
    first = matmul(cuda_lib, a, asc, w, ws, M, N, K, F32)
    for _ in range(3):
        again = matmul(cuda_lib, a, asc, w, ws, M, N, K, F32, st=s.cuda_stream)
        assert torch.equal(first, again)


def test_row_offsets_past_32_bits(cuda_lib):
    """Operand and output rows that lie beyond 2^32 bytes."""
    import torch
    M, N, K, lda, ldo = 70, 64, 128, 1 << 26, 1 << 25
    rng = np.random.default_rng(2)
    a, asc = f8.quant_rows(activations(rng, M, K))
    w, ws = f8.quant_weight(rng.standard_normal((1, N, K)).astype(np.float32))
    big = torch.empty(M * lda, dtype=torch.uint8, device="cuda")
    big.view(M, lda)[:, :K] = cuda(a)
    o = torch.empty(M * ldo, dtype=torch.float32, device="cuda")
    das, dw, dws = cuda(asc), cuda(f8.pitched(w)), cuda(ws)
    assert cuda_lib.ts_cuda_op_matmul_fp8(ptr(big), lda, ptr(das), M, ptr(dw), dw.stride(1), ptr(dws), 0, 128, None, None, 1,
                                          ptr(o), F32, ldo, 0, M, N, K, stream()) == 0, cuda_lib.ts_cuda_last_error()
    torch.cuda.synchronize()
    av, wv = f8.rows_value(a, asc), f8.weight_value(w[0], ws[0])
    check(o.view(M, ldo)[:, :N], av, wv, av @ wv.T, F32)
    # and the quantiser's
    x = torch.empty(M * (1 << 25), dtype=torch.float32, device="cuda").view(M, -1)
    xs = activations(rng, M, K)
    x[:, :K] = cuda(xs)
    codes, scales = torch.zeros(M, K, dtype=torch.uint8, device="cuda"), torch.zeros(1, M, device="cuda")
    assert cuda_lib.ts_cuda_op_quant_fp8(ptr(x), F32, x.stride(0), M, K, 0, ptr(codes), K, ptr(scales), M, stream()) == 0
    torch.cuda.synchronize()
    ec, es = f8.quant_rows(xs)
    assert np.array_equal(codes.cpu().numpy(), ec) and np.array_equal(scales.cpu().numpy(), es)
